"""GPU tests of neon_sample_rows against the definition in 64 bits (numpy): the
ids have to be equal.  The kernel's masses are round(w 2^44), off by at most
2^-45 of the largest weight each, so two computations can differ only where
u x mass (or top_p x mass, or min_p) falls within V 2^-45 of a token's border.
Rows whose reference lies within twice that are left out and counted."""
import sys

import numpy as np
import pytest

import neonengine_amd as ne
from tests.gpu_util import to_dev, to_host, torch_cuda

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def reference(l, t, k, p, mp, u):
    """(id, distance from the nearest border relative to the mass) of one row."""
    V = len(l)
    x = np.where(np.isnan(l), -np.inf, l).astype(np.float64)
    m = x.max()
    if m == -np.inf:
        return -1, 1.0
    if t == 0:
        return int(x.argmax()), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / np.float64(t)))
    order = np.lexsort((np.arange(V), -x))
    ws = w[order]
    if 0 < k < V:
        ws = np.where(np.arange(V) < k, ws, 0)
    far = 1.0
    if p < 1:
        run = np.cumsum(ws)
        goal = np.float64(p) * run[-1]
        n = int(np.searchsorted(run, goal))  # first with run >= goal
        if not (ws[:n + 1] == 1).all():  # whole weights sum exactly
            far = min(far, np.abs(run - goal).min() / run[-1])
        ws = np.where(np.arange(V) <= n, ws, 0)
    if mp > 0:
        d = np.abs(ws - np.float64(mp))
        far = min(far, d[ws != 1].min() if (ws != 1).any() else 1.0)
        ws = np.where(ws >= np.float64(mp), ws, 0)
    kept = np.zeros(V)
    kept[order] = ws
    run = np.cumsum(kept)
    target = np.float64(u) * run[-1]
    i = int(np.searchsorted(run, target, side="right"))
    if not (np.unique(kept[kept > 0]) == 1).all():
        # a border lies at a kept token (before the first one the sum is 0 exactly)
        far = min(far, np.abs(run - target)[kept > 0].min() / run[-1])
    return i, far


def draw(l, t=None, k=None, p=None, mp=None, u=None, stride=None):
    torch = torch_cuda()
    B, V = l.shape
    wide = np.full((B, stride or V), 1e30, np.float32)
    wide[:, :V] = l
    dl = to_dev(wide)[:, :V]
    out = torch.full((B,), -5, dtype=torch.int32, device="cuda")

    def dev(a, dt):
        return None if a is None else to_dev(np.broadcast_to(np.asarray(a, dt), (B,)).copy())

    ne.sample_rows(dl, dev(u, np.float32), out, dev(t, np.float32), dev(k, np.int32),
                   dev(p, np.float32), dev(mp, np.float32))
    return to_host(out)


def compare(l, t, k, p, mp, u, most_left_out=0.02, **kw):
    B = l.shape[0]
    got = draw(l, t, k, p, mp, u, **kw)
    full = [np.broadcast_to(np.asarray(d if a is None else a, dt), (B,)) for a, d, dt in
            ((t, 1, np.float32), (k, 0, np.int32), (p, 1, np.float32), (mp, 0, np.float32),
             (u, 0, np.float32))]
    left = 0
    for b in range(B):
        want, far = reference(l[b], *(a[b] for a in full))
        if far < l.shape[1] * 2.0 ** -44:
            left += 1
            continue
        assert got[b] == want, (b, got[b], want, far, [a[b] for a in full])
    assert left <= max(1, most_left_out * B), left
    return got


SIZES = [1, 2, 63, 64, 65, 255, 256, 257, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8192, 8193,
         16385, 32003, 50000, 65537]


@pytest.mark.parametrize("V", SIZES)
def test_every_setting(V):
    say("sample_rows V", V)
    rng = np.random.default_rng(V)
    B = 40
    l = (rng.normal(size=(B, V)) * rng.uniform(0.3, 5, (B, 1))).astype(np.float32)
    l[:, rng.integers(0, V, V // 7)] = -np.inf
    l[:, V // 2] = 1.0
    t = rng.uniform(0.2, 2.0, B).astype(np.float32)
    t[:3] = 0
    k = rng.integers(-1, V + 2, B).astype(np.int32)
    k[5:9] = [1, 2, V, V + 100]
    p = rng.uniform(0.02, 1.0, B).astype(np.float32)
    p[rng.random(B) < 0.3] = 1
    mp = (rng.random(B) * 0.2 * (rng.random(B) < 0.5)).astype(np.float32)
    u = rng.random(B).astype(np.float32)
    u[10], u[11] = 0, np.float32(1 - 2.0 ** -24)
    compare(l, t, k, p, mp, u, stride=V + V % 5)
    compare(l, t, None, None, None, u)
    compare(l, t, k, None, None, u)
    compare(l, t, None, p, None, u)
    compare(l, t, None, None, mp, u)
    compare(l, None, k, p, None, u)


@pytest.mark.parametrize("B", [1, 5, 130])
def test_the_presets_vocabulary(B):
    V = 201088
    rng = np.random.default_rng(B)
    l = (rng.normal(size=(B, V)) * rng.uniform(0.5, 3.5, (B, 1))).astype(np.float32)
    t = rng.uniform(0.3, 1.7, B).astype(np.float32)
    p = rng.uniform(0.3, 1.0, B).astype(np.float32)
    k = rng.integers(0, 3000, B).astype(np.int32)
    u = rng.random(B).astype(np.float32)
    compare(l, t, k, p, None, u)
    compare(l, t, None, p, None, u)
    compare(l, t, k * 50, p, np.float32(0.001), u)


@pytest.mark.parametrize("V", [5, 1000, 4097, 50001, 201088])
def test_equal_logits(V):
    """Flat rows, and rows with large groups of equal values: ties go to the
    lowest index.  Equal weights of 1 sum exactly, so nothing is left out."""
    rng = np.random.default_rng(V)
    B = 12
    flat = np.full((B, V), -3.25, np.float32)
    u = rng.random(B).astype(np.float32)
    u[0], u[1] = 0, np.float32(1 - 2.0 ** -24)
    k = np.array([0, 1, 2, V // 2, V - 1, V, 3, 7, 64, 100, 1000, 5000], np.int32)
    p = np.array([1, 1, .5, .5, .25, .75, 1, .125, .5, 1, .5, 1], np.float32)
    compare(flat, None, k, p, None, u, 0)
    compare(flat, 0.5, None, p, 1.0, u, 0)
    some = flat.copy()
    some[:, rng.integers(0, V, V // 3 + 1)] = 1.5  # the kept ones are whole weights
    compare(some, 1.0, k, np.minimum(p, np.float32(.5)), np.float32(0.5), u, 0)
    three = np.floor(rng.normal(size=(B, V)) * 1.2).astype(np.float32)
    compare(three, 0.9, k, p, None, u, 0.5)
    compare(three, 0.9, k, None, None, u, 0.5)


def test_extreme_logits():
    lo = np.finfo(np.float32).min
    hi = np.finfo(np.float32).max
    V = 3000
    rng = np.random.default_rng(3)
    base = rng.normal(size=V).astype(np.float32)
    rows = []
    r = base.copy(); r[1:] = lo; rows.append(r)                       # masked by the lowest value
    rows.append(np.full(V, lo, np.float32))                            # all of them
    rows.append(np.full(V, -np.inf, np.float32))                       # nothing left
    rows.append(np.full(V, np.nan, np.float32))
    r = base.copy(); r[::2] = np.nan; rows.append(r)
    r = base.copy(); r[[7, 2000]] = np.inf; rows.append(r)             # two of infinite weight
    r = base.copy(); r[5] = hi; r[9] = lo; rows.append(r)
    r = base.copy(); r[:] = -np.inf; r[2999] = -40; rows.append(r)
    r = np.where(base > 0, np.float32(0.0), np.float32(-0.0)); rows.append(r)  # equal zeros
    r = base * 1e-42; rows.append(r.astype(np.float32))                # denormals
    l = np.stack(rows).astype(np.float32)
    u = np.full(len(rows), 0.625, np.float32)
    for t in (0.0, 1.0, 1e-30, 1e30):
        for k, p in ((0, 1.0), (3, 1.0), (0, 0.5), (2, 0.5)):
            got = compare(l, t, k, p, None, u, 0.2)
            assert got[2] == -1 and got[3] == -1
    ne.device_check()


def test_parameters_out_of_range():
    rng = np.random.default_rng(4)
    B, V = 10, 700
    l = rng.normal(size=(B, V)).astype(np.float32)
    t, p = np.ones(B, np.float32), np.full(B, 0.9, np.float32)
    mp, u = np.zeros(B, np.float32), np.full(B, 0.4, np.float32)
    t[0], t[1], t[2] = -1, np.inf, np.nan
    p[3], p[4] = 0, 1.5
    mp[5], mp[6] = -0.1, np.nan
    u[7], u[8] = 1.0, np.nan
    got = draw(l, t, None, p, mp, u)
    assert (got[:9] == -1).all()
    assert got[9] == reference(l[9], 1.0, 0, np.float32(0.9), 0.0, np.float32(0.4))[0]
    with pytest.raises(ne.NeonError) as e:
        ne.device_check()
    assert e.value.status == ne.NEON_EINVAL and "parameter" in str(e.value)
    ne.device_check()


def test_frequencies():
    """Evenly spread random numbers give each token its share of the draws."""
    V, n = 40, 4096
    rng = np.random.default_rng(6)
    row = rng.normal(size=V).astype(np.float32) * 2
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = draw(np.tile(row, (n, 1)), 0.8, 12, 0.9, None, u)
    w = np.exp((row.astype(np.float64) - row.max()) / np.float64(np.float32(0.8)))
    order = np.argsort(-w)
    w[order[12:]] = 0
    run = np.cumsum(w[order])
    w[order[int(np.searchsorted(run, np.float64(np.float32(0.9)) * run[-1])) + 1:]] = 0
    share = w / w.sum() * n
    counts = np.bincount(got, minlength=V)
    # an interval of length share holds its share of evenly spaced points, to one
    assert np.abs(counts - share).max() <= 1 + 1e-3


def test_agrees_with_the_engine_s_sampler_at_its_limits():
    """top_k 1, temperature 0 and a tiny top_p all give neon_sample's greedy
    limit."""
    torch = torch_cuda()
    rng = np.random.default_rng(7)
    l = rng.normal(size=(6, 5000)).astype(np.float32)
    u = rng.random(6).astype(np.float32)
    want = l.argmax(1)
    for kw in ({"k": 1}, {"t": 0}, {"p": np.float32(1e-7)}, {"mp": 1.0}):
        assert np.array_equal(draw(l, u=u, **kw), want), kw
    out = torch.empty(6, dtype=torch.int32, device="cuda")
    ne.sample_logits(to_dev(l), 6, 5000, 1.0, 1e-7, 3, to_dev(np.zeros(6, np.int32)), out)
    assert np.array_equal(to_host(out), want)


def test_same_draws_again_and_through_a_graph():
    torch = torch_cuda()
    B, V = 9, 201088
    g = torch.Generator(device="cuda").manual_seed(1)
    l = torch.randn((B, V), device="cuda", generator=g) * 2
    u = torch.rand(B, device="cuda", generator=g)
    p = torch.full((B,), 0.95, device="cuda")
    out = torch.empty(B, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(ne.sample_rows_workspace(B, V), 1), dtype=torch.uint8, device="cuda")
    ne.sample_rows(l, u, out, top_p=p, workspace=ws)
    first = to_host(out).copy()
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ne.sample_rows(l, u, out, top_p=p, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        ne.sample_rows(l, u, out, top_p=p, workspace=ws)
    for i in range(4):
        ws.fill_(0xA5 + i)  # any contents
        out.zero_()
        graph.replay()
        assert np.array_equal(to_host(out), first)
        l.mul_(1.0)
        ne.sample_rows(l, u, out, top_p=p)
        assert np.array_equal(to_host(out), first)
