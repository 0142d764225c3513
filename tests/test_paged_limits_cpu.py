"""CPU checks of the sizes that the paged calls and neon_sample_rows take."""
import pytest

import neonengine_amd as ne


@pytest.mark.parametrize("V", [700, 4096, 4097, 32003, 65536, 65537, 201088, 1 << 24])
def test_sampling_workspace_never_falls(V):
    """A buffer for the largest batch serves the smaller ones."""
    sizes = [ne.sample_rows_workspace(B, V) for B in (*range(1, 700), 1000, 1024, 65535)]
    assert sizes == sorted(sizes)


def test_attention_workspace_never_falls():
    sizes = [ne.paged_attn_workspace(n, 64, 64, 8, 64) for n in (*range(1, 100), 4096, 100000)]
    assert sizes == sorted(sizes)


def test_append_refuses_more_threads_than_a_launch_holds():
    """2^23 rows of 512 threads are 2^32, one more than a launch has."""
    import ctypes as C
    P = 4096  # an aligned address, never dereferenced: the call is refused first
    kv = ne.PagedKVStruct(P, P, None, None, ne.KV_BF16, 8, 16, 8, 64)
    status = ne.lib().neon_paged_append(C.addressof(kv), P, 144 * 64, P, 9, P, P, P, 1 << 20, P,
                                        1 << 23, 2, 128, None)
    assert status == ne.NEON_EINVAL


def test_paged_kv_refuses_other_number_types():
    torch = pytest.importorskip("torch")
    shape = (2, 1, 16, 64)
    for dtype in (torch.bfloat16, torch.int16):
        ne.paged_kv(torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype))
    half, whole = (torch.zeros(shape, dtype=t) for t in (torch.float16, torch.bfloat16))
    for k, v in ((half, half), (whole, half), (half, whole)):
        with pytest.raises(ValueError):
            ne.paged_kv(k, v)
