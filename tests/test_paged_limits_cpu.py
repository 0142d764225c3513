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
