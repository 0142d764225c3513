"""GPU tests of neon_beam_select and neon_beam_reorder against the definitions in
64 bits (numpy).  Ids have to be equal.  A score is the 64-bit value rounded once to
fp32 (half a step, 2^-24 of it); the kernel's 64-bit value is off by a few 2e-14 of the
sum of exponentials (its exponential's polynomial) and by the rounding of 64-bit sums of
up to 2^24 terms, under 1e-11 together."""
import sys

import numpy as np
import pytest

import neonengine_amd as ne
from tests import beam_util
from tests.gpu_util import empty_dev, to_dev, to_host, torch_cuda

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def run(l, score, W, stop=(), stride=None, ended=True, alias=False, workspace=None):
    torch = torch_cuda()
    N, V = l.shape
    x = to_dev(l)
    if stride is not None:
        wide = torch.full((N, stride), float("inf"), device="cuda")
        wide[:, :V] = x
        x = wide[:, :V]
    token, parent = empty_dev(N, np.int32), empty_dev(N, np.int32)
    s = to_dev(score)
    out = s if alias else empty_dev(N, np.float32)
    end = (empty_dev(N, np.int32), empty_dev(N, np.int32), empty_dev(N, np.float32)) if ended else None
    ne.beam_select(x, s, W, token, parent, out, stop=to_dev(np.array(stop, np.int32)) if len(stop) else None,
                   ended=end, workspace=workspace)
    got = [to_host(t) for t in (token, parent, out)]
    return got + ([to_host(t) for t in end] if ended else [])


def check(got, want):
    for i in (0, 1, 3, 4):
        if i < len(got):
            assert np.array_equal(got[i], want[i]), (i, np.nonzero(got[i] != want[i])[0][:8])
    for i in (2, 5):
        if i < len(got):
            fine = np.isfinite(want[i])
            assert np.array_equal(got[i][~fine], want[i][~fine].astype(np.float32))
            g, w = got[i][fine].astype(np.float64), want[i][fine]
            assert (np.abs(g - w) <= 2.0 ** -24 * np.abs(w) + 1e-11).all(), np.abs(g - w).max()


def case(rng, B, W, V, dev=2.5, masked=0.02, dead=0.1):
    l = rng.normal(0, dev, (B * W, V)).astype(np.float32)
    l[rng.random(l.shape) < masked] = -np.inf
    score = (-12 - 2 * rng.random(B * W)).astype(np.float32)
    score[rng.random(B * W) < dead] = -np.inf
    return l, score


@pytest.mark.parametrize("B,W,V,n_stop,stride", [
    (1, 1, 1, 0, None), (1, 1, 2, 1, None), (2, 4, 3, 2, 5), (3, 2, 63, 0, 64), (1, 4, 1023, 3, None),
    (2, 4, 1024, 3, 1025), (1, 4, 4093, 3, 4099), (1, 3, 4096, 2, 4096), (2, 5, 4097, 1, None),
    (5, 32, 700, 16, None), (1, 32, 33000, 16, 33001), (7, 8, 32003, 2, None), (1, 4, 201088, 3, None),
    (16, 4, 50257, 3, 50260), (300, 2, 999, 1, None), (40, 16, 5000, 4, None)])
def test_select(B, W, V, n_stop, stride):
    rng = np.random.default_rng(B * 1000 + V)
    l, score = case(rng, B, W, V)
    stop = rng.choice(V, min(n_stop, V), replace=False)
    for t in stop[:2]:
        l[:, t] = np.where(rng.random(B * W) < 0.4, l.max(-1), l[:, t])
    say(f"select B={B} W={W} V={V} stops={len(stop)} stride={stride}")
    check(run(l, score, W, stop, stride), beam_util.select(l, score, W, stop))
    ne.device_check()


@pytest.mark.parametrize("V", [5, 1030, 9001])
@pytest.mark.parametrize("form", ["all equal", "ascending", "descending", "lowest", "one", "zeros", "huge",
                                  "ties"])
def test_select_orders(form, V):
    W, B = 8, 2
    i = np.arange(V)
    row = {"all equal": np.full(V, 1.5), "ascending": i * 0.01, "descending": -i * 0.01,
           "lowest": np.full(V, np.finfo(np.float32).min), "one": np.where(i == V // 2, 3.0, -np.inf),
           "zeros": np.where(i % 2, 0.0, -0.0), "huge": np.where(i % 3, 3e38, -3e38),
           "ties": (i * 7 % 5).astype(float)}[form]
    l = np.repeat(row[None], B * W, 0).astype(np.float32)
    if form == "lowest":
        l[1::2, V // 3] = -np.inf
    score = np.repeat(np.float32(-3.0) - np.arange(B * W) % 3, 1).astype(np.float32)
    stop = [0, V // 2, V - 1]
    say(f"order {form} V={V}")
    check(run(l, score, W, stop), beam_util.select(l, score, W, stop))
    check(run(l, score, W), beam_util.select(l, score, W))
    ne.device_check()


# Plateaus of 256 tokens (a group of a wave, whose first one the exponentials are relative
# to until another is more than 64 above it), repeated along the row
RISES = {"mask of -1e9": [-1e9, 0.0], "mask of the lowest": [np.finfo(np.float32).min, 0.0],
         "just below": [-63.0, 0.0], "just above": [-66.0, 0.0], "by 100": [-100.0, 0.0],
         "stairs": [-1e30, -1e9, -2e4, -500.0, -100.0, 0.0, -3.0], "fall and rise": [0.0, -1e4, 90.0, -1e9],
         "past the exponent": [0.0, 710.0, 1500.0, 3000.0], "huge": [-1e38, 1e38, 3e38, -3e38],
         "open": [-np.inf, -1e9, 0.0, np.nan, 200.0]}


@pytest.mark.parametrize("V", [300, 1500, 8000, 40000, 600011])
@pytest.mark.parametrize("form", list(RISES))
def test_select_logits_that_rise_by_much(form, V):
    """Tokens far above those before them; one group of a wave, and several (up to 4 and up
    to 8 of them: 12 and 360 rows)."""
    for B in (3, 90) if V < 50000 else (3,):
        W = 4
        rng = np.random.default_rng(V + B)
        steps = np.array(RISES[form])[np.arange(V) // 256 % len(RISES[form])]
        l = (steps + rng.normal(0, 2.0, (B * W, V))).astype(np.float32)
        l[1] = np.roll(l[1], 256)
        l[2] = l[2, ::-1]
        score = (-12 - 2 * rng.random(B * W)).astype(np.float32)
        stop = [int(l[0].argmax()) if form != "open" else int(np.nanargmax(l[0])), V - 1]
        say(f"rises {form} V={V} B={B}")
        check(run(l, score, W, stop), beam_util.select(l, score, W, stop))
        ne.device_check()


def test_select_first_step_and_dead_requests():
    rng = np.random.default_rng(5)
    l, score = case(rng, 6, 4, 3001)
    score[:] = -np.inf
    score[0], score[9], score[20:24] = 0.0, -1.0, -2.0
    l[score == -np.inf] = np.nan  # not read
    l[21] = -np.inf               # nothing to choose
    l[22, :3000] = -np.inf        # one token
    say("first step")
    check(run(l, score, 4, [5, 77]), beam_util.select(l, score, 4, [5, 77]))
    ne.device_check()


def test_select_nan_and_infinite():
    rng = np.random.default_rng(6)
    l, score = case(rng, 4, 4, 2000, dead=0)
    l[rng.random(l.shape) < 0.1] = np.nan
    say("NaN logits")
    check(run(l, score, 4, [9]), beam_util.select(l, score, 4, [9]))
    ne.device_check()
    for where, bad in (("score", np.nan), ("score", np.inf), ("logit", np.inf)):
        l2, s2 = l.copy(), score.copy()
        if where == "score":
            s2[5] = bad
        else:
            l2[5, 1234] = bad
        say(f"{where} {bad}")
        check(run(l2, s2, 4, [9]), beam_util.select(l2, s2, 4, [9]))
        with pytest.raises(ne.NeonError):
            ne.device_check()
        ne.device_check()


def test_select_stop_ids():
    """Ids twice, ids of no token, every token a stop token, no ended list."""
    rng = np.random.default_rng(7)
    l, score = case(rng, 2, 4, 50)
    for stop in ([3, 3, -1, 50, 1 << 30], list(range(16))):
        check(run(l, score, 4, stop), beam_util.select(l, score, 4, stop))
    l, score = case(rng, 2, 4, 9)
    check(run(l, score, 4, list(range(9))), beam_util.select(l, score, 4, list(range(9))))
    l, score = case(rng, 3, 4, 5000)
    check(run(l, score, 4, [17], ended=False), beam_util.select(l, score, 4, [17])[:3])


def test_select_in_place_and_shared_workspace():
    """out_score may be score; a workspace of any contents and of a larger batch serves."""
    torch = torch_cuda()
    rng = np.random.default_rng(8)
    ws = torch.full((ne.beam_select_workspace(40, 8, 60000, 1),), 0xFF, dtype=torch.uint8, device="cuda")
    for B in (40, 9, 1):
        l, score = case(rng, B, 8, 60000)
        check(run(l, score, 8, [0], alias=True, workspace=ws), beam_util.select(l, score, 8, [0]))


def test_select_far_offsets():
    """Rows whose offset passes 2^31 elements."""
    torch = torch_cuda()
    stride, W, V = 1 << 30, 3, 70001
    big = torch.empty(2 * stride + V, dtype=torch.float32, device="cuda")
    rows = big.as_strided((3, V), (stride, 1))
    rng = np.random.default_rng(9)
    l, score = case(rng, 1, W, V, dead=0)
    rows.copy_(to_dev(l))
    token, parent, out = empty_dev(3, np.int32), empty_dev(3, np.int32), empty_dev(3, np.float32)
    say("far offsets")
    ne.beam_select(rows, to_dev(score), W, token, parent, out)
    check([to_host(t) for t in (token, parent, out)], beam_util.select(l, score, W)[:3])


def test_select_refusals_python():
    torch = torch_cuda()
    f = lambda *s: torch.zeros(s, device="cuda")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    l = f(8, 50)
    for args in ((l.half(), f(8), 4, i(8), i(8), f(8)), (l, f(7), 4, i(8), i(8), f(8)),
                 (l, f(8), 3, i(8), i(8), f(8)), (l, f(8), 4, f(8), i(8), f(8)),
                 (l, f(8), 4, i(8), i(7), f(8)), (l, f(8), 4, i(8), i(8), i(8)),
                 (l.t(), f(8), 4, i(8), i(8), f(8)), (l.cpu(), f(8), 4, i(8), i(8), f(8))):
        with pytest.raises(ValueError):
            ne.beam_select(*args)
    with pytest.raises(ne.NeonError):
        ne.beam_select(l, f(8), 4, i(8), i(8), f(8), stop=i(17))
    with pytest.raises(ne.NeonError):
        ne.beam_select(l, f(8), 4, i(8), i(8), f(8), workspace=f(1))


# ---------------------------------------------------------------------------
# states
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("B,W,slabs,T,row,n", [
    (1, 1, 1, 1, 4, 1), (1, 4, 1, 7, 4, 1), (2, 3, 2, 33, 12, 2), (3, 4, 8, 300, 128, 2), (2, 8, 3, 65, 128, 3),
    (1, 16, 2, 50, 256, 2), (2, 32, 1, 41, 20, 1), (5, 2, 1, 1000, 16, 70), (1, 5, 1, 129, 4, 2)])
@pytest.mark.parametrize("kind", ["beams", "permutation", "any"])
def test_reorder(B, W, slabs, T, row, n, kind):
    rng = np.random.default_rng(W * T + row)
    N = B * W
    first = np.repeat(np.arange(B) * W, W)
    if kind == "permutation":
        parent = np.concatenate([b * W + rng.permutation(W) for b in range(B)])
    else:
        parent = first + rng.integers(0, W, N)
        if kind == "beams":
            parent = np.where(rng.random(N) < 0.6, np.arange(N), parent)
            parent = np.where(parent[parent] == parent, parent, np.arange(N))
        parent[rng.random(N) < 0.1] = -1
    length = rng.integers(0, T + 3, N).astype(np.int32)
    length[0] = -2 if kind == "any" else T
    for lens in (length, None):
        x = [rng.integers(-2 ** 31, 2 ** 31, (N, slabs, T, row // 4)).astype(np.int32) for _ in range(n)]
        d = [to_dev(v) for v in x]
        say(f"reorder {kind} B={B} W={W} slabs={slabs} T={T} row={row}")
        ne.beam_reorder(ne.beam_states(d, W), to_dev(parent.astype(np.int32)), None if lens is None else to_dev(lens))
        for v, t in zip(x, d):
            assert np.array_equal(to_host(t), beam_util.reorder(v, parent, lens, W))
    ne.device_check()


def test_reorder_shapes_and_bad_parents():
    torch = torch_cuda()
    # token histories [B W][T], caches in bf16 [B W][Hkv][T][D]
    h = torch.arange(8 * 5, dtype=torch.int32, device="cuda").view(8, 5)
    want = h[[1, 1, 0, 3, 4, 4, 4, 7]].clone()
    ne.beam_reorder(ne.beam_states([h], 4), to_dev(np.array([1, 1, 0, 3, 4, 4, 4, 7], np.int32)))
    assert torch.equal(h, want)
    x = torch.randn(4, 2, 6, 64, device="cuda").bfloat16()
    old = x.clone()
    bad = to_dev(np.array([2, 1, 1, 5], np.int32))  # of another request, and of no row
    ne.beam_reorder(ne.beam_states([x], 2), bad)
    assert torch.equal(x[[0, 1, 3]], old[[0, 1, 3]]) and torch.equal(x[2], old[2])
    with pytest.raises(ne.NeonError):
        ne.device_check()
    for states, W in (([], 2), ([x], 3), ([x, h], 2), ([x, x.cpu()], 2), ([torch.zeros(4, device="cuda")], 2)):
        with pytest.raises(ValueError):
            ne.beam_states(states, W)
    with pytest.raises(ValueError):
        ne.beam_reorder(ne.beam_states([x], 2), bad[:3])
    with pytest.raises(ValueError):
        ne.beam_reorder(ne.beam_states([x], 2), bad, bad.float())
    with pytest.raises(ne.NeonError):
        ne.beam_reorder(ne.beam_states([torch.zeros(4, 3, 1, dtype=torch.uint8, device="cuda")], 2), bad)


class Guarded:
    """A device buffer with a sentinel on both sides."""

    def __init__(self, n, fill=0x5A):
        torch = torch_cuda()
        self.all = torch.full((n + 512,), fill, dtype=torch.uint8, device="cuda")
        self.fill, self.n = fill, n
        self.mid = self.all[256:256 + n]

    def as_type(self, dtype, *shape):
        return self.mid.view(dtype).view(*shape)

    def intact(self):
        a = to_host(self.all)
        return (a[:256] == self.fill).all() and (a[256 + self.n:] == self.fill).all()


@pytest.mark.parametrize("B,W,V,n_stop", [(1, 1, 1, 0), (2, 3, 5000, 2), (3, 32, 2049, 16), (60, 4, 33000, 3)])
def test_select_stays_inside_its_buffers(B, W, V, n_stop):
    torch = torch_cuda()
    rng = np.random.default_rng(V)
    l, score = case(rng, B, W, V)
    stop = rng.choice(V, min(V, n_stop), replace=False)
    N = B * W
    need = ne.beam_select_workspace(B, W, V, len(stop))
    ws = Guarded(need)
    outs = [Guarded(4 * N) for _ in range(6)]
    t = [g.as_type(torch.float32 if i in (2, 5) else torch.int32, N) for i, g in enumerate(outs)]
    # rows from an odd place of wider ones
    wide = torch.full((N, V + 9), float("inf"), device="cuda")
    wide[:, 3:3 + V] = to_dev(l)
    say(f"guards B={B} W={W} V={V}")
    ne.beam_select(wide[:, 3:3 + V], to_dev(score), W, *t[:3], stop=to_dev(stop.astype(np.int32)) if len(stop) else None,
                   ended=tuple(t[3:]), workspace=ws.mid)
    check([to_host(x) for x in t], beam_util.select(l, score, W, stop))
    assert ws.intact() and all(g.intact() for g in outs)


@pytest.mark.parametrize("W", [1, 32])
def test_select_largest_vocabulary(W):
    torch = torch_cuda()
    V = 1 << 24
    g = torch.Generator(device="cuda")
    g.manual_seed(W)
    l = torch.randn((W, V), generator=g, device="cuda")
    score = (-10 - torch.rand(W, generator=g, device="cuda"))
    token, parent, out = empty_dev(W, np.int32), empty_dev(W, np.int32), empty_dev(W, np.float32)
    say(f"2^24 tokens, {W} beams")
    ne.beam_select(l, score, W, token, parent, out)
    # the candidates that count: the best of each row
    v = torch.empty(W, W, dtype=torch.float64, device="cuda")
    at = torch.empty(W, W, dtype=torch.int64, device="cuda")
    for w in range(W):
        x = l[w].double()
        lse = x.max() + (x - x.max()).exp().sum().log()
        top, at[w] = torch.topk(x, W)
        v[w] = score[w].double() + (top - lse)
    v, at = to_host(v).reshape(-1), to_host(at).reshape(-1)
    best = np.argsort(-v, kind="stable")[:W]
    place, rest = {}, []
    for i in best:
        (rest.append(i) if i // W in place else place.__setitem__(i // W, i))
    for w in range(W):
        if w not in place:
            place[w] = rest.pop(0)
    for w, i in place.items():
        assert to_host(token)[w] == at[i] and to_host(parent)[w] == i // W
        assert abs(to_host(out)[w] - v[i]) <= 2.0 ** -24 * abs(v[i]) + 1e-10


def test_select_equal_beams_wherever_their_rows_begin():
    """Equal rows and scores are ordered by their places, then tokens, whatever the
    alignment of the rows: their 64-bit values are bit-equal."""
    rng = np.random.default_rng(12)
    for V in (1001, 4099, 20003):
        one = rng.normal(0, 2, V).astype(np.float32)
        l = np.repeat(one[None], 8, 0)
        token, parent, out = run(l, np.full(8, -1.5, np.float32), 8, ended=False)
        assert np.array_equal(token, np.full(8, one.argmax())) and np.array_equal(parent, np.arange(8))
        assert (out == out[0]).all()


@pytest.mark.parametrize("row", [4, 16, 48])
def test_reorder_stays_inside_its_states(row):
    torch = torch_cuda()
    rng = np.random.default_rng(row)
    N, slabs, T = 6, 3, 37
    x = rng.integers(-2 ** 31, 2 ** 31, (N, slabs, T, row // 4)).astype(np.int32)
    g = Guarded(x.nbytes)
    d = g.as_type(torch.int32, *x.shape)
    d.copy_(to_dev(x))
    parent = np.array([1, 2, 0, 3, 3, 4], np.int32)
    length = np.array([37, 5, 0, 37, 36, 1], np.int32)
    ne.beam_reorder(ne.beam_states([d], 3), to_dev(parent), to_dev(length))
    assert np.array_equal(to_host(d), beam_util.reorder(x, parent, length, 3)) and g.intact()
