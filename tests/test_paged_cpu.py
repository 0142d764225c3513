"""CPU checks of neon_paged_* and neon_sample_rows: every refusal that the host
makes before it touches a device, the workspace queries, and the plain MXFP4
forms that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import neonengine_amd as ne
from tests.paged_util import E2M1, bf16, f32, quantise, values

P = 4096  # an aligned address, never dereferenced: validation fails first


def kv(**k):
    s = ne.PagedKVStruct(P, P, None, None, ne.KV_BF16, 8, 16, 2, 64)
    for n, v in k.items():
        setattr(s, n, v)
    return C.addressof(s), s


def append(k=None, qkv=P, stride=8 * 64, table=P, n_pos=9, q_start=P, kv_len=P, pages=P,
           max_pages=2, q_out=P, n_rows=3, B=2, Hq=4, **fields):
    ref, keep = kv(**fields)
    return ne.lib().neon_paged_append(ref if k is None else k, qkv, stride, table, n_pos, q_start,
                                      kv_len, pages, max_pages, q_out, n_rows, B, Hq, None)


def gather(k_out=P, v_out=P, q_start=P, kv_len=P, pages=P, max_pages=2, n_rows=3, B=2, **fields):
    ref, keep = kv(**fields)
    return ne.lib().neon_paged_gather(ref, q_start, kv_len, pages, max_pages, k_out, v_out, n_rows,
                                      B, None)


def attn(q=P, stride=256, sinks=P, q_start=P, kv_len=P, pages=P, max_pages=2, out=P, n_rows=3, B=2,
         Hq=4, window=0, ws=P, wb=1 << 40, cnt=P, cb=1 << 40, **fields):
    ref, keep = kv(**fields)
    return ne.lib().neon_paged_attn(ref, q, stride, sinks, q_start, kv_len, pages, max_pages, out,
                                    n_rows, B, Hq, window, ws, wb, cnt, cb, None)


CACHE = [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(format=2), dict(format=-1),
         dict(format=ne.KV_MXFP4), dict(format=ne.KV_MXFP4, k_scales=P), dict(k_scales=P, v_scales=P),
         dict(format=ne.KV_MXFP4, k_scales=P + 1, v_scales=P), dict(n_pages=0), dict(page_size=0),
         dict(page_size=8), dict(page_size=24), dict(page_size=1 << 17), dict(page_size=-16),
         dict(n_kv_heads=0), dict(n_kv_heads=-2), dict(head_dim=32), dict(head_dim=96),
         dict(head_dim=256)]
ROWS = [dict(kv_len=None), dict(pages=None), dict(max_pages=0), dict(B=0), dict(B=-1),
        dict(B=65536), dict(n_rows=-1), dict(n_rows=(1 << 23) + 1), dict(q_start=None, n_rows=3, B=2)]


@pytest.mark.parametrize("bad", CACHE + ROWS, ids=str)
@pytest.mark.parametrize("call", [append, gather, attn])
def test_cache_and_rows_are_refused(call, bad):
    if call is append and "k" in bad and bad["k"] is None:
        ref, keep = kv(k=None)
        bad = dict(k=ref)
    elif call is append and "k" in bad:
        ref, keep = kv(**bad)
        bad = dict(k=ref)
    assert call(**bad) == ne.NEON_EINVAL
    assert ne.lib().neon_last_error(None).startswith(b"neon_paged_")


@pytest.mark.parametrize("bad", [
    dict(qkv=None), dict(qkv=P + 4), dict(stride=8 * 64 - 8), dict(stride=8 * 64 + 4),
    dict(stride=-512), dict(table=P + 4), dict(n_pos=0), dict(q_out=None), dict(q_out=P + 2),
    dict(Hq=-1), dict(Hq=65536)], ids=str)
def test_append_refusals(bad):
    assert append(**bad) == ne.NEON_EINVAL


def test_null_struct():
    L = ne.lib()
    assert L.neon_paged_append(None, P, 512, P, 9, P, P, P, 2, P, 3, 2, 4, None) == ne.NEON_EINVAL
    assert L.neon_paged_gather(None, P, P, P, 2, P, P, 3, 2, None) == ne.NEON_EINVAL
    assert L.neon_paged_attn(None, P, 256, P, P, P, P, 2, P, 3, 2, 4, 0, P, 1 << 40, P, 1 << 40,
                             None) == ne.NEON_EINVAL


@pytest.mark.parametrize("bad", [dict(k_out=None), dict(v_out=None), dict(k_out=P + 8)], ids=str)
def test_gather_refusals(bad):
    assert gather(**bad) == ne.NEON_EINVAL


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q=P + 4), dict(out=None), dict(out=P + 8), dict(stride=248),
    dict(stride=260), dict(Hq=3), dict(Hq=1), dict(Hq=0), dict(Hq=130, stride=1 << 20),
    dict(window=-1), dict(n_rows=1 << 17, B=65535, Hq=1024, n_kv_heads=1024, stride=1 << 16)], ids=str)
def test_attn_refusals(bad):
    assert attn(**bad) == ne.NEON_EINVAL


@pytest.mark.parametrize("n_rows,B,Hq,Hkv,D", [(1, 1, 8, 8, 64), (64, 64, 64, 8, 64),
                                               (4096, 3, 64, 8, 64), (70, 64, 24, 8, 128)])
def test_attn_workspace_is_checked(n_rows, B, Hq, Hkv, D):
    wb, cb = ne.paged_attn_workspace(n_rows, B, Hq, Hkv, D)
    same = dict(n_rows=n_rows, B=B, Hq=Hq, n_kv_heads=Hkv, head_dim=D, stride=Hq * D)
    if wb:
        assert attn(**same, wb=wb - 1) == ne.NEON_EINVAL
        assert attn(**same, ws=None) == ne.NEON_EINVAL
        assert attn(**same, ws=P + 8) == ne.NEON_EINVAL
    if cb:
        assert attn(**same, cb=cb - 1) == ne.NEON_EINVAL
        assert attn(**same, cnt=None) == ne.NEON_EINVAL


def test_workspace_queries_of_bad_shapes_are_zero():
    L = ne.lib()
    assert L.neon_paged_attn_workspace(1, 0, 8, 8, 64) == 0
    assert L.neon_paged_attn_counters(1, 1, 9, 8, 64) == 0
    assert L.neon_paged_attn_workspace(1, 1, 8, 8, 80) == 0
    assert L.neon_sample_rows_workspace(0, 10) == 0
    assert L.neon_sample_rows_workspace(1, (1 << 24) + 1) == 0


def test_no_rows_is_no_work():
    assert append(n_rows=0) == ne.NEON_OK
    assert gather(n_rows=0) == ne.NEON_OK
    assert attn(n_rows=0) == ne.NEON_OK


def test_sample_rows_refusals():
    f = ne.lib().neon_sample_rows
    ok = [P, 100, 2, 100, P, P, P, P, P, P, P, 1 << 40, None]
    for at, bad in ((0, None), (8, None), (9, None), (2, 0), (2, 65536), (3, 0), (3, 101),
                    (1, 99), (1, -100)):
        args = list(ok)
        args[at] = bad
        assert f(*args) == ne.NEON_EINVAL, (at, bad)
    assert f(P, 1 << 25, 1, (1 << 24) + 1, P, P, P, P, P, P, P, 1 << 40, None) == ne.NEON_EINVAL
    need = ne.sample_rows_workspace(2, 201088)
    if need:
        assert f(P, 201088, 2, 201088, P, P, P, P, P, P, P, need - 1, None) == ne.NEON_EINVAL
        assert f(P, 201088, 2, 201088, P, P, P, P, P, P, None, need, None) == ne.NEON_EINVAL


def test_plain_quantiser():
    """The rule as neon_paged_append states it, on values worked out by hand."""
    x = np.zeros((1, 64), np.float32)
    x[0, :8] = [6, -6, 5, 5.5, 0.25, 0.75, 2.5, 3.5]
    x[0, 32:36] = [7.5, 1, -1, 3]  # 7.5 > 7: the scale doubles
    c, s = quantise(x)
    assert s.tolist() == [[127, 128]]
    v = values(c, s)
    assert v[0, :8].tolist() == [6, -6, 4, 6, 0, 1, 2, 4]
    assert v[0, 32:36].tolist() == [8, 1, -1, 3]
    assert values(*quantise(np.full((1, 32), np.inf)))[0, 0] != values(
        *quantise(np.full((1, 32), np.inf)))[0, 0]
    c, s = quantise(np.zeros((1, 32), np.float32))
    assert s.tolist() == [[127]] and not c.any()


def test_plain_quantiser_is_nearest():
    rng = np.random.default_rng(0)
    x = (rng.normal(size=(200, 64)) * np.exp(rng.normal(size=(200, 1)) * 9)).astype(np.float32)
    v = values(*quantise(x)).reshape(200, 2, 32)
    b = x.reshape(200, 2, 32).astype(np.float64)
    _, s = quantise(x)
    grid = E2M1 * np.ldexp(1.0, s.astype(int) - 127)[..., None]
    best = np.abs(b[..., None] - grid[:, :, None]).min(-1)
    assert np.array_equal(np.abs(v - b), best)
    # no element is off by more than half a step of the top binade
    top = np.ldexp(1.0, s.astype(int) - 127)[..., None]
    assert (np.abs(v - b) <= top).all()


def test_bf16_rounding_helper():
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -2.5], np.float32)
    assert f32(bf16(x)).tolist() == [1.0, 1.0, 1 + 2.0 ** -6, -2.5]


def test_no_rows_need_no_buffers():
    """A tensor of no rows has no memory."""
    assert append(n_rows=0, qkv=None, q_out=None) == ne.NEON_OK
    assert gather(n_rows=0, k_out=None, v_out=None) == ne.NEON_OK
    assert attn(n_rows=0, q=None, out=None, ws=None, wb=0, cnt=None, cb=0) == ne.NEON_OK
    assert attn(n_rows=0, page_size=24) == ne.NEON_EINVAL
