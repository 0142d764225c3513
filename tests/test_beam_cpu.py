"""CPU checks of neon_beam_* and neon_pages_*: every refusal that the host makes
before it touches a device, the workspace queries, and the plain forms that the
GPU tests compare with, on cases small enough to write down."""
import ctypes as C

import numpy as np
import pytest

import neonengine_amd as ne
from tests import beam_util

P = 4096  # an aligned address, never dereferenced: validation fails first


def select(logits=P, stride=100, B=2, W=4, V=100, score=P, stop=P, n_stop=2, token=P, parent=P, out=P,
           et=P, ep=P, es=P, ws=P, wb=1 << 40):
    return ne.lib().neon_beam_select(logits, stride, B, W, V, score, stop, n_stop, token, parent, out, et,
                                     ep, es, ws, wb, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(score=None), dict(token=None), dict(parent=None), dict(out=None),
    dict(stop=None), dict(stride=99), dict(B=0), dict(B=65536), dict(W=0), dict(W=33), dict(V=0),
    dict(V=(1 << 24) + 1, stride=1 << 30), dict(n_stop=-1), dict(n_stop=17), dict(et=None), dict(ep=None),
    dict(es=None), dict(et=None, ep=None), dict(ws=None), dict(ws=P + 8), dict(wb=100),
    dict(B=65535, W=32, V=1 << 17, stride=1 << 17)], ids=str)
def test_select_refusals(bad):
    assert select(**bad) == ne.NEON_EINVAL
    assert ne.lib().neon_last_error(None).startswith(b"neon_beam_select")


@pytest.mark.parametrize("B,W,V,n_stop", [(1, 1, 1, 0), (1, 4, 201088, 3), (65535, 32, 17, 16),
                                          (3, 32, 1 << 24, 1)])
def test_select_workspace_is_checked(B, W, V, n_stop):
    n = ne.beam_select_workspace(B, W, V, n_stop)
    assert n >= B * W * 8 * (W + n_stop)
    assert select(B=B, W=W, V=V, stride=V, n_stop=n_stop, wb=B * W * 8 * (W + n_stop)) == ne.NEON_EINVAL


@pytest.mark.parametrize("W,V,n_stop", [(1, 201088, 0), (4, 32003, 3), (8, 60000, 1), (32, 5, 16), (5, 1, 0)])
def test_select_workspace_serves_smaller_batches(W, V, n_stop):
    """The query never falls as B grows."""
    last = 0
    for B in list(range(1, 400)) + list(range(400, 65536, 397)):
        n = ne.beam_select_workspace(B, W, V, n_stop)
        assert n >= last
        last = n


def reorder(states=(P, P), n=None, B=2, W=4, slabs=2, T=8, row=128, length=P, parent=P):
    s = None if states is None else (C.c_void_p * len(states))(*states)
    return ne.lib().neon_beam_reorder(s, len(states) if n is None else n, B, W, slabs, T, row, length, parent,
                                      None)


@pytest.mark.parametrize("bad", [
    dict(states=None, n=1), dict(states=(P, None)), dict(states=(P + 4,)), dict(n=-1), dict(B=0),
    dict(B=65536), dict(W=0), dict(W=33), dict(slabs=0), dict(T=0), dict(row=0), dict(row=2), dict(row=6),
    dict(parent=None), dict(T=1 << 30, slabs=1 << 20), dict(T=(1 << 31) - 1, row=(1 << 31) - 4),
    dict(B=65535, slabs=1 << 20)], ids=str)
def test_reorder_refusals(bad):
    assert reorder(**bad) == ne.NEON_EINVAL
    assert ne.lib().neon_last_error(None).startswith(b"neon_beam_reorder")


Q = 1 << 20  # another address


def fork(refs=P, table=P, length=P, B_in=3, parent=P, keep=P, add=P, refs_out=P, table_out=Q, len_out=P,
         src=P, dst=P, rows=P, B=3, n_pages=50, page=16, width=4, ws=P, wb=1 << 40, cnt=P, cb=1 << 40):
    return ne.lib().neon_pages_fork(refs, table, length, B_in, parent, keep, add, refs_out, table_out,
                                    len_out, src, dst, rows, B, n_pages, page, width, ws, wb, cnt, cb, None)


SHAPES = [dict(B=0), dict(B=65536), dict(n_pages=0), dict(n_pages=(1 << 24) + 1), dict(page=8),
          dict(page=48), dict(page=1 << 17), dict(page=-16), dict(width=0), dict(width=-1),
          dict(B=65535, width=1 << 30), dict(B=200, width=1 << 26), dict(B=32, width=1 << 26), dict(ws=None), dict(ws=P + 4), dict(wb=10), dict(refs=None),
          dict(table=None), dict(length=None), dict(refs_out=None), dict(table_out=None), dict(src=None),
          dict(dst=None)]


@pytest.mark.parametrize("bad", SHAPES + [
    dict(B_in=0), dict(B_in=65536), dict(len_out=None), dict(rows=None), dict(cnt=None), dict(cnt=P + 8),
    dict(cb=599), dict(parent=None, B_in=2), dict(table_out=P)], ids=str)
def test_fork_refusals(bad):
    assert fork(**bad) == ne.NEON_EINVAL
    assert ne.lib().neon_last_error(None).startswith(b"neon_pages_fork")


def compact(refs=P, table=P, length=P, refs_out=P, table_out=P, to=P, src=P, dst=P, B=3, n_pages=50, page=16,
            width=4, ws=P, wb=1 << 40):
    return ne.lib().neon_pages_compact(refs, table, length, refs_out, table_out, to, src, dst, B, n_pages,
                                       page, width, ws, wb, None)


@pytest.mark.parametrize("bad", SHAPES + [dict(to=None)], ids=str)
def test_compact_refusals(bad):
    assert compact(**bad) == ne.NEON_EINVAL
    assert ne.lib().neon_last_error(None).startswith(b"neon_pages_compact")


def test_plan_workspaces():
    for n, B in [(1, 1), (1000, 3), (1 << 24, 65535)]:
        wb, cb = ne.pages_workspace(n, B)
        assert wb > 0 and cb >= 8 * n
        assert fork(n_pages=n, B=B, B_in=B, wb=wb - 1) == ne.NEON_EINVAL
        assert fork(n_pages=n, B=B, B_in=B, cb=cb - 1) == ne.NEON_EINVAL
        assert compact(n_pages=n, B=B, wb=wb - 1) == ne.NEON_EINVAL
    assert ne.pages_workspace(0, 1) == (0, 0) and ne.pages_workspace(5, 0)[0] == 0
    assert ne.beam_select_workspace(1, 33, 5, 0) == 0 and ne.beam_select_workspace(1, 1, 5, 17) == 0


def copy(kv=({},), n_kv=None, src=P, dst=P, rows=P, n=3):
    fields = dict(k=P, v=P, k_scales=None, v_scales=None, format=ne.KV_BF16, n_pages=8, page_size=16,
                  n_kv_heads=2, head_dim=64)
    s = None if kv is None else (ne.PagedKVStruct * len(kv))(*(
        ne.PagedKVStruct(*{**fields, **k}.values()) for k in kv))
    return ne.lib().neon_pages_copy(None if s is None else C.addressof(s), len(kv or ()) if n_kv is None
                                    else n_kv, src, dst, rows, n, None)


@pytest.mark.parametrize("bad", [
    dict(kv=None, n_kv=1), dict(n_kv=0), dict(n_kv=-1), dict(src=None), dict(dst=None), dict(n=-1),
    dict(n=(1 << 24) + 1), dict(kv=({}, dict(n_pages=9))), dict(kv=({}, dict(page_size=32))),
    dict(kv=({}, dict(n_kv_heads=3))), dict(kv=({}, dict(head_dim=128))), dict(kv=(dict(k=None),)),
    dict(kv=({}, dict(v=P + 8))), dict(kv=(dict(format=7),)), dict(kv=(dict(page_size=24),)),
    dict(kv=({}, dict(format=ne.KV_MXFP4, k_scales=P, v_scales=P))),
    dict(kv=(dict(page_size=65536, n_kv_heads=1024),), n=1 << 24)], ids=str)
def test_copy_refusals(bad):
    assert copy(**bad) == ne.NEON_EINVAL
    assert ne.lib().neon_last_error(None).startswith(b"neon_pages_copy")


def test_copy_of_nothing():
    assert copy(n=0) == ne.NEON_OK
    assert copy(n=0, src=None, dst=None, rows=None) == ne.NEON_OK


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def test_plain_select():
    l = np.array([[0, 1, 2, 0], [2.5, 0, 0, -np.inf]], np.float32)
    token, parent, out, et, ep, es = beam_util.select(l, np.array([-1.0, -1.0], np.float32), 2)
    # 2.5 of place 1, then 2 of place 0: both go on where they are
    assert token.tolist() == [2, 0] and parent.tolist() == [0, 1]
    assert np.allclose(out, [-1 + 2 - np.log(np.exp([0, 1, 2, 0]).sum()),
                             -1 + 2.5 - np.log(np.exp([2.5, 0, 0]).sum())])
    assert et.tolist() == [-1, -1] and (es == -np.inf).all()
    # token 0 ends: the best candidate of all, so it is listed, and place 0 goes on twice
    token, parent, out, et, ep, es = beam_util.select(l, np.array([-1.0, -1.0], np.float32), 2, [0])
    assert et.tolist() == [0, -1] and ep.tolist() == [1, -1]
    assert token.tolist() == [2, 1] and parent.tolist() == [0, 0]
    # a first step: one beam
    token, parent, _, _, _, _ = beam_util.select(l, np.array([0.0, -np.inf], np.float32), 2)
    assert token.tolist() == [2, 1] and parent.tolist() == [0, 0]
    # equal values: the lower place, the lower token
    token, parent, _, _, _, _ = beam_util.select(np.zeros((3, 2), np.float32), np.zeros(3, np.float32), 3)
    assert token.tolist() == [0, 0, 1] and parent.tolist() == [0, 1, 0]


def test_plain_fork():
    # two beams of 20 tokens on pages of 16: page 5 shared, 2 and 3 their own; both go on from row 0
    table = np.array([[5, 2, -7], [5, 3, -7]], np.int32)
    refs = np.array([0, 0, 1, 1, 0, 2], np.int32)
    out, full = beam_util.fork(refs, table, [20, 20], 16, np.full((2, 3), -9, np.int32), parent=[0, 0])
    refs2, table2, length, src, dst, rows = out
    assert table2.tolist() == [[5, 2, -9], [5, 0, -9]] and not full
    assert refs2.tolist() == [1, 0, 1, 0, 0, 2] and length.tolist() == [21, 21]
    assert src.tolist() == [-1, 2] and dst.tolist() == [-1, 0] and rows.tolist() == [0, 4]
    # at a page's end both take a new one, in order; page 3 is free again and taken last
    out, full = beam_util.fork(refs, table, [32, 32], 16, np.full((2, 3), -9, np.int32), parent=[0, 0])
    assert out[1].tolist() == [[5, 2, 0], [5, 2, 1]] and out[0].tolist() == [1, 1, 2, 0, 0, 2]


def test_plain_compact():
    out = beam_util.compact(np.array([0, 2, 0, 0, 1, 1], np.int32), np.array([[4, 1], [1, -7]], np.int32),
                            [20, 16], 16, np.full((2, 2), -9, np.int32))
    assert [x.tolist() for x in out] == [[1, 2, 1, 0, 0, 0], [[0, 1], [1, -9]], [-1, 1, -1, -1, 0, 2],
                                         [4, 5, -1], [0, 2, -1]]


# ---------------------------------------------------------------------------
# states that overlap would be moved twice at once
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("others", [(Q,), (Q + 16,), (Q + 16384 - 16,), (Q - 16384 + 16,), (1 << 30, Q + 8192),
                                    tuple((1 << 30) + 16384 * i for i in range(70)) + (Q + 16,)])
def test_reorder_refuses_states_that_overlap(others):
    # 2 requests of 4 places, 2 slabs of 8 rows of 128 bytes: 16384 bytes
    assert reorder(states=(Q, *others)) == ne.NEON_EINVAL
    assert b"overlap" in ne.lib().neon_last_error(None)


def test_beam_states_refuse_tensors_that_overlap():
    torch = pytest.importorskip("torch")
    x, y = torch.zeros(8, 2, 6, 4), torch.zeros(8, 2, 6, 4)
    whole = torch.zeros(9, 2, 6, 4)
    for states in ([x, x], [x, y, x], [whole[:8], whole[1:]], [whole[1:], y, whole[:8]]):
        with pytest.raises(ValueError, match="overlap"):
            ne.beam_states(states, 4)
    both = torch.zeros(2, 8, 2, 6, 4)
    assert ne.beam_states([both[1], x, both[0]], 4).rows == 8
