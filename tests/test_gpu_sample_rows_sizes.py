"""GPU tests of neon_sample_rows at the sizes of its documented range: workspaces
shared by batches of different sizes, vocabularies past 2^18 tokens."""
import numpy as np
import pytest

import neonengine_amd as ne
from tests.gpu_util import to_dev, to_host, torch_cuda
from tests.test_gpu_sample_rows import draw, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [32003, 4097])
def test_one_workspace_for_all_batches(V):
    """Sized for 300 rows, used by fewer; flat rows, whose draw is floor(u V)."""
    torch = torch_cuda()
    ws = torch.empty(max(ne.sample_rows_workspace(300, V), 1), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(V)
    for B in (300, 257, 256, 100, 17, 1):
        u = rng.random(B).astype(np.float32)
        out = torch.full((B,), -5, dtype=torch.int32, device="cuda")
        ws.fill_(0xA5)
        ne.sample_rows(torch.full((B, V), 1.5, device="cuda"), to_dev(u), out, workspace=ws)
        # u V is a multiple of 2^-24: exact in 64 bits
        assert np.array_equal(to_host(out), np.floor(u.astype(np.float64) * V).astype(np.int32)), B
    ne.device_check()


def small_kept(V, k, p, u):
    """The draw from V equal logits: kept are the first ceil(p min(k, V)) tokens; every
    product here is exact in 64 bits."""
    k = np.where((k > 0) & (k < V), k, V).astype(np.float64)
    n = np.ceil(p.astype(np.float64) * k)
    return np.floor(u.astype(np.float64) * n).astype(np.int32)


# past 2^18 tokens a mass has fewer bits; past 2^21 there are more than 512 parts
@pytest.mark.parametrize("V", [1 << 18, (1 << 18) + 1, (1 << 21) + 5, 3_000_001, 1 << 24])
def test_equal_logits_of_large_vocabularies(V):
    torch = torch_cuda()
    print("V", V, flush=True)
    last = np.float32(1 - 2.0 ** -24)
    k = np.array([0, 0, 0, 0, V // 2, V - 1, 5000, 0], np.int32)
    p = np.array([1, 1, .5, .5, 1, .75, 1, .25], np.float32)
    u = np.array([0, last, last, .375, last, last, .5, 0], np.float32)
    out = torch.full((8,), -5, dtype=torch.int32, device="cuda")
    ne.sample_rows(torch.full((8, V), -2.25, device="cuda"), to_dev(u), out, top_k=to_dev(k),
                   top_p=to_dev(p))
    got = to_host(out)
    assert np.array_equal(got, small_kept(V, k, p, u)), (got, small_kept(V, k, p, u))
    ne.device_check()


def kept_mass(l, t, k, p, mp):
    """Of one row, in units of the largest weight."""
    x = np.sort(l.astype(np.float64))[::-1]
    w = np.exp((x - x[0]) / np.float64(t))[:k if 0 < k < len(l) else None]
    run = np.cumsum(w)
    w = w[:int(np.searchsorted(run, np.float64(p) * run[-1])) + 1]
    return w[w >= np.float64(mp)].sum()


@pytest.mark.parametrize("V", [(1 << 18) + 1, (1 << 21) + 5])
def test_settings_of_large_vocabularies(V):
    """Rows are compared where u or top_p lies further than twice the masses' rounding
    from a border: V tokens, each off by at most half of 2^-(62 - ceil(log2 V)) of the
    largest weight.  reference() gives the distance relative to the mass, which is M
    largest weights (the kept mass, the smallest of those it divides by): so the
    rounding is V 2^-(63 - ceil(log2 V)) / M there."""
    print("V", V, flush=True)
    rng = np.random.default_rng(V)
    B = 4
    l = (rng.normal(size=(B, V)) * np.array([[3], [2], [4], [2.5]])).astype(np.float32)
    l[:, 11::50] = -np.inf
    t = np.array([1, 0.8, 1.5, 0.7], np.float32)
    k = np.array([0, 4000, 100000, 0], np.int32)
    p = np.array([0.9, 0.95, 0.8, 1], np.float32)
    mp = np.array([0, 0, 1e-4, 1e-3], np.float32)
    u = np.array([0.3, 0.9, 0.01, 0.999], np.float32)
    got = draw(l, t, k, p, mp, u)
    ne.device_check()
    near = V * 2.0 ** -(62 - (V - 1).bit_length())
    left = 0
    for b in range(B):
        want, far = reference(l[b], t[b], k[b], p[b], mp[b], u[b])
        if far < near / kept_mass(l[b], t[b], k[b], p[b], mp[b]):
            left += 1
            continue
        assert got[b] == want, (b, got[b], want, far)
    assert left <= 1
