"""GPU tests of the paged KV cache: neon_paged_append, neon_paged_gather and
neon_paged_attn against plain forms, at the sizes, masks and layouts where
they can go wrong.

The append's results are compared bit for bit: the rotation is two rounded
products and a rounded sum in fp32, which numpy states the same way, and every
rounding after it is to the nearest, ties to even.

Attention is held to |got - ref| <= 2^-8 |ref| + (2^-8 + 2^-12) A with A =
sum_j p_j |v_j| in 64 bits: 2^-8 is half a bf16 step of the output, and the
same again for each p_j, if a kernel rounds it to bf16 for the product (at
most half a step, whatever it rounds).  2^-12 covers what is in fp32: a score
is off by at most (D + 2) 2^-24 sum_d |q_d k_d| / sqrt(D), under 2^-13.4 for
the inputs here (D <= 128; sum |q_d k_d| / sqrt(D) < 90), its exponential by
as much relative to itself, half of it again from the normalising sum, and
sums of n terms in runs of at most 2^10 by n 2^-24 <= 2^-14."""
import sys

import numpy as np
import pytest

import neonengine_amd as ne
from tests.gpu_util import empty_dev, to_dev, to_host, torch_cuda
from tests.paged_util import Batch, attention, bf16, f32, quantise, values

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def rope_table(n_pos, D):
    f = 150000.0 ** (-np.arange(0, D, 2) / D)
    a = np.arange(n_pos)[:, None] * f
    return np.stack((np.cos(a), np.sin(a))).astype(np.float32)


def rotate(x, table, pos):
    """fp32, each product and sum rounded: x [n][heads][D] at pos [n]."""
    half = x.shape[-1] // 2
    c, s = table[0, pos][:, None], table[1, pos][:, None]
    x1, x2 = x[..., :half], x[..., half:]
    return np.concatenate((x1 * c - x2 * s, x2 * c + x1 * s), -1).astype(np.float32)


APPEND = [
    # (mx, D, Hq, Hkv, page, lens, q_start)
    (False, 64, 64, 8, 64, [(1, 1), (1, 64), (1, 65), (1, 1000)], False),
    (True, 64, 64, 8, 16, [(1, 1), (1, 16), (1, 17), (1, 333)], False),
    (False, 128, 6, 2, 32, [(3, 3), (0, 5), (40, 77), (1, 1), (0, 0)], True),
    (True, 128, 1, 1, 256, [(300, 300), (2, 700)], True),
    (True, 64, 3, 1, 16, [(17, 40)], True),
    (False, 64, 0, 4, 128, [(9, 200), (130, 131)], True),
    (True, 64, 8, 8, 64, [(1, 50)] * 300, False),
    (False, 64, 8, 8, 64, [(b % 3, 10 + b) for b in range(300)], True),
]


@pytest.mark.parametrize("mx,D,Hq,Hkv,page,lens,q_start", APPEND)
@pytest.mark.parametrize("rot", [True, False])
def test_append_and_gather(mx, D, Hq, Hkv, page, lens, q_start, rot):
    torch_cuda()
    say(f"append mx={mx} D={D} Hq={Hq} Hkv={Hkv} page={page} B={len(lens)} rot={rot}")
    rng = np.random.default_rng(D + Hq + len(lens))
    bt = Batch(rng, lens, page, Hkv, D, mx, q_start=q_start, pad=3 if q_start else 0)
    heads = Hq + 2 * Hkv
    wide = heads * D + 8 * (D == 64)  # rows of a wider matrix
    x = bf16(rng.normal(size=(bt.n_rows, wide)).astype(np.float32) * 3)
    x[0, :D] = 0x8000  # a row of -0: zero blocks
    if bt.n_rows > 1 and heads > 2:
        x[1, (Hq + Hkv) * D:(Hq + Hkv) * D + 32] = 0  # a zero block of v
        x[1, (Hq + Hkv) * D + 32:(Hq + Hkv) * D + 64] = bf16(
            np.array([7.0, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25] * 4, np.float32))  # borders
    table = rope_table(max(t for _, t in lens) + 1, D)
    d = bt.dev()
    dx = to_dev(x)[:, :heads * D]
    q_out = to_dev(np.full((bt.n_rows, max(Hq, 1), D), 0x1234, np.uint16))
    ne.paged_append(d["kv"], dx, to_dev(table) if rot else None, d["q_start"], d["kv_len"],
                    d["table"], q_out if Hq else None, Hq)
    k_out, v_out = (to_dev(np.full((bt.n_rows, Hkv, D), 0x4321, np.uint16)) for _ in "kv")
    ne.paged_gather(d["kv"], d["q_start"], d["kv_len"], d["table"], k_out, v_out)
    ne.device_check()
    want_q = np.full((bt.n_rows, max(Hq, 1), D), 0x1234, np.uint16)
    want = {c: np.full((bt.n_rows, Hkv, D), 0x4321, np.uint16) for c in "kv"}
    for b, (n, t) in enumerate(lens):
        r = slice(bt.starts[b], bt.starts[b] + n)
        f = f32(x[r, :heads * D]).reshape(n, heads, D)
        pos = np.arange(t - n, t)
        turned = rotate(f[:, :Hq + Hkv], table, pos) if rot else f[:, :Hq + Hkv]
        if Hq:
            want_q[r] = bf16(turned[:, :Hq])
        pg, at = bt.places(b, t - n)
        for c, w in (("k", turned[:, Hq:]), ("v", f[:, Hq + Hkv:])):
            bt.put(c, pg, at, w)
            want[c][r] = bf16(values(*quantise(w)).astype(np.float32)) if mx else bf16(w)
    assert np.array_equal(to_host(q_out), want_q)
    # the whole pools: what was appended, and nothing else
    for c in ("k", "v") + (("ks", "vs") if mx else ()):
        assert np.array_equal(to_host(d[c]), getattr(bt, c)), c
    assert np.array_equal(to_host(k_out) & 0x7FFF, want["k"] & 0x7FFF)  # zeros of either sign
    assert np.array_equal(to_host(v_out) & 0x7FFF, want["v"] & 0x7FFF)
    assert np.array_equal(to_host(v_out)[f32(want["v"]) != 0], want["v"][f32(want["v"]) != 0])


def test_append_matches_the_engine_s_rotation():
    """q and k as neon_rope_yarn gives them, with neon_rope_table's table."""
    torch = torch_cuda()
    rng = np.random.default_rng(5)
    cfg = ne.config_preset("gpt-oss-20b")
    bt = Batch(rng, [(4, 9), (1, 40)], 16, 2, 64, False)
    x = bf16(rng.normal(size=(5, 8, 64)).astype(np.float32))
    table = torch.empty((2, 64, 32), dtype=torch.float32, device="cuda")
    ne.rope_table(cfg, 64, table)
    d = bt.dev()
    q_out, k_out, v_out = (empty_dev((5, h, 64), np.uint16) for h in (4, 2, 2))
    ne.paged_append(d["kv"], to_dev(x), table, d["q_start"], d["kv_len"], d["table"], q_out, 4)
    ne.paged_gather(d["kv"], d["q_start"], d["kv_len"], d["table"], k_out, v_out)
    qk = to_dev(x[:, :6])
    ne.rope_yarn(qk, to_dev(np.array([5, 6, 7, 8, 39], np.int32)), 5, 6, 64, table, 64)
    qk = to_host(qk)
    assert np.array_equal(to_host(q_out), qk[:, :4])
    assert np.array_equal(to_host(k_out), qk[:, 4:])
    assert np.array_equal(to_host(v_out), x[:, 6:])


def test_append_mxfp4_special_values():
    """Every binade and border of the quantiser, denormals, the largest values,
    and blocks with a NaN or an infinity."""
    torch_cuda()
    rng = np.random.default_rng(9)
    n = 700
    bt = Batch(rng, [(n, n)], 64, 1, 64, True)
    v = np.empty((n, 2, 32), np.float32)
    for i in range(n):
        e = rng.integers(-132, 125)
        m = rng.choice([1.0, 1.4921875, 1.5, 1.5078125, 1.75, 1.7578125, 1.9921875])
        v[i] = np.ldexp(rng.choice([0, .0625, .125, .1875, .25, .3125, .375, .4375, .5, .625, .75,
                                    .875, 1.0], size=(2, 32)) * rng.choice([-1, 1], (2, 32)), e)
        v[i, :, rng.integers(32)] = np.ldexp(m, e)
    v[3, 0, 5], v[3, 1, 0], v[4, 1, 31] = np.nan, np.inf, -np.inf
    x = np.zeros((n, 3, 64), np.uint16)
    bits = v.reshape(n, 64).view(np.uint32)
    x[:, 2] = bits >> 16  # every value is a bf16 one, or loses bits below it
    x[:, 1] = x[:, 2]
    d = bt.dev()
    q_out = empty_dev((n, 1, 64), np.uint16)
    ne.paged_append(d["kv"], to_dev(x), None, d["q_start"], d["kv_len"], d["table"], q_out, 1)
    pg, at = bt.places(0)
    codes, scales = quantise(f32(x[:, 2])[:, None])
    for c in "kv":
        got_s = to_host(d[c + "s"])[pg, :, at]
        assert np.array_equal(got_s, scales), np.argwhere(got_s != scales)[:4]
        assert np.array_equal(to_host(d[c])[pg, :, at], codes)


def attn_case(mx, D, Hq, Hkv, page, lens, window=0, sinks=True, q_start=True, pad=0, seed=0,
              dev=None, scale=2.0):
    rng = np.random.default_rng(seed)
    bt = Batch(rng, lens, page, Hkv, D, mx, q_start=q_start, pad=pad).fill(rng)
    q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32) * scale)
    sk = f32(bf16(rng.normal(size=Hq).astype(np.float32))) if sinks else None
    return bt, q, sk


def check(got, ref, mag, left):
    """got: bf16 bits [n_rows][Hq][D]; rows of no sequence hold `left`."""
    none = np.isnan(mag)
    assert np.array_equal(got[none], np.full(none.sum(), left, np.uint16))
    g = f32(got).astype(np.float64)
    bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -12) * mag + 1e-30
    off = np.where(none, 0, np.abs(g - np.where(none, 0, ref)) / np.where(none, 1, bound))
    assert np.isfinite(g[~none]).all()
    assert off.max() <= 1.0, (off.max(), np.unravel_index(off.argmax(), off.shape))


def run_attn(bt, q, sk, window, d=None, **kw):
    d = d or bt.dev()
    out = to_dev(np.full(q.shape, 0x1357, np.uint16))
    ne.paged_attn(d["kv"], to_dev(q), None if sk is None else to_dev(bf16(sk)), d["q_start"],
                  d["kv_len"], d["table"], out, q.shape[1], window=window, **kw)
    return to_host(out)


ONE = [(1, n) for n in (1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 300, 1025)]
ATTN = [
    # (mx, D, Hq, Hkv, page, lens, window, sinks, q_start, pad)
    (False, 64, 64, 8, 16, ONE, 0, True, False, 0),
    (True, 64, 64, 8, 16, ONE, 0, True, False, 0),
    (False, 128, 32, 8, 32, ONE, 0, False, False, 0),
    (True, 128, 32, 8, 64, ONE, 0, True, False, 0),
    (False, 64, 8, 8, 256, ONE, 0, False, True, 2),         # one query head per KV head
    (True, 64, 3, 1, 16, ONE, 0, False, True, 0),           # odd groups
    (False, 128, 14, 2, 16, ONE, 0, True, True, 0),
    (False, 64, 64, 1, 64, ONE, 0, True, False, 0),         # 64 per KV head
    (True, 64, 40, 2, 32, ONE, 0, True, True, 1),
    (False, 64, 64, 8, 64, ONE, 128, True, False, 0),       # windows
    (True, 64, 64, 8, 64, ONE, 128, True, False, 0),
    (False, 64, 16, 2, 16, ONE, 1, True, True, 0),
    (True, 128, 16, 2, 16, ONE, 17, False, True, 0),
    (False, 64, 16, 2, 16, ONE, 100000, True, False, 0),
    # several rows each, free places, sequences without rows, padding
    (False, 64, 64, 8, 16, [(2, 2), (0, 7), (3, 50), (0, 0), (1, 1), (5, 300)], 0, True, True, 5),
    (True, 64, 64, 8, 16, [(2, 2), (0, 7), (3, 50), (0, 0), (1, 1), (5, 300)], 0, True, True, 5),
    (False, 128, 12, 4, 32, [(7, 40), (8, 8), (9, 1000)], 20, False, True, 0),
    (False, 64, 16, 2, 64, [(1, 0), (1, 70), (1, 0), (1, 5)], 0, True, False, 0),
    # prompt chunks
    (False, 64, 64, 8, 64, [(130, 130), (1, 200), (65, 400)], 0, True, True, 3),
    (True, 64, 64, 8, 64, [(130, 130), (1, 200), (65, 400)], 0, True, True, 3),
    (False, 64, 64, 8, 128, [(200, 500)], 128, True, True, 0),
    (True, 128, 24, 8, 16, [(97, 97), (33, 333)], 50, False, True, 0),
    (False, 128, 5, 1, 32, [(257, 600)], 0, True, True, 0),
    (False, 64, 4, 4, 16, [(511, 513), (1, 9), (300, 300)], 0, False, True, 0),
    (True, 64, 8, 1, 256, [(70, 2000)], 0, True, True, 0),
]


@pytest.mark.parametrize("mx,D,Hq,Hkv,page,lens,window,sinks,q_start,pad", ATTN)
def test_attention(mx, D, Hq, Hkv, page, lens, window, sinks, q_start, pad):
    torch_cuda()
    say(f"attn mx={mx} D={D} Hq={Hq} Hkv={Hkv} page={page} lens={lens} window={window}")
    bt, q, sk = attn_case(mx, D, Hq, Hkv, page, lens, window, sinks, q_start, pad,
                          seed=D + Hq + len(lens) + window)
    got = run_attn(bt, q, sk, window)
    ne.device_check()
    ref, mag = attention(bt, f32(q), sk, window)
    check(got, ref, mag, 0x1357)


@pytest.mark.parametrize("mx,D,Hq,Hkv,page,lens,window", [
    (False, 64, 16, 2, 16, [(1, 40000), (1, 3)], 0),
    (True, 128, 8, 1, 32, [(1, 33333), (2, 70)], 0),
    (False, 64, 8, 1, 64, [(1, 40000)], 5000),
    (True, 64, 16, 2, 64, [(40, 20000)], 0),
    (False, 128, 8, 2, 16, [(19, 9001), (1, 1)], 3000),
])
def test_attention_long(mx, D, Hq, Hkv, page, lens, window):
    """Long axes that are split and joined."""
    torch_cuda()
    say(f"attn long mx={mx} D={D} lens={lens}")
    bt, q, sk = attn_case(mx, D, Hq, Hkv, page, lens, window, seed=3)
    got = run_attn(bt, q, sk, window)
    ref, mag = attention(bt, f32(q), sk, window)
    check(got, ref, mag, 0x1357)


def test_attention_many_sequences():
    """More sequences than a block has threads, few and many rows mixed."""
    torch_cuda()
    lens = [(b % 4, 5 + (b * 37) % 90) for b in range(700)]
    bt, q, sk = attn_case(False, 64, 8, 2, 16, lens, seed=4)
    got = run_attn(bt, q, sk, 0)
    ref, mag = attention(bt, f32(q), sk, 0)
    check(got, ref, mag, 0x1357)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("lens", [[(1, 500), (1, 90), (1, 33)], [(130, 400), (1, 90)]])
def test_attention_shared_and_repeated_pages(mx, lens):
    """Sequences that share a prefix's pages, and a page twice in one table."""
    torch_cuda()
    bt, q, sk = attn_case(mx, 64, 16, 2, 16, lens, seed=6)
    bt.table[1, :3] = bt.table[0, :3]
    bt.table[0, 5] = bt.table[0, 2]
    got = run_attn(bt, q, sk, 0)
    ref, mag = attention(bt, f32(q), sk, 0)
    check(got, ref, mag, 0x1357)


@pytest.mark.parametrize("lens", [[(1, 500), (1, 90)], [(1, 17), (1, 16)], [(100, 300), (2, 90)]])
def test_attention_bad_pages_are_hidden(lens):
    torch_cuda()
    bt, q, sk = attn_case(False, 64, 16, 2, 16, lens, seed=7)
    good = bt.table.copy()
    bad = [(0, 1), (1, 0)]
    dead = {}
    for b, j in bad:
        dead[b] = j
    d = bt.dev()
    t = good.copy()
    t[0, 1], t[1, 0] = bt.n_pages, -1
    d["table"] = to_dev(t)
    got = run_attn(bt, q, sk, 0, d=d)
    with pytest.raises(ne.NeonError) as e:
        ne.device_check()
    assert e.value.status == ne.NEON_EINVAL and "page id" in str(e.value)
    ne.device_check()  # reported once
    ref, mag = attention(bt, f32(q), sk, 0, hidden=lambda b, n: np.arange(n) // 16 == dead[b])
    check(got, ref, mag, 0x1357)


def test_pages_behind_the_window_may_be_gone():
    """Their table entries are not looked at, their memory is poison."""
    torch_cuda()
    for mx, lens, page, window in ((False, [(1, 1000), (3, 333)], 16, 128),
                                   (True, [(70, 900), (1, 129)], 32, 100)):
        bt, q, sk = attn_case(mx, 64, 16, 2, page, lens, window, seed=15)
        ref, mag = attention(bt, f32(q), sk, window)
        for b, (n, t) in enumerate(lens):
            gone = max(0, t - n - window + 1) // page
            ids = bt.table[b, :gone].copy()
            bt.k[ids], bt.v[ids] = (0x77, 0x77) if mx else (0x7FC1, 0x7FC1)
            if mx:
                bt.ks[ids] = bt.vs[ids] = 255
            bt.table[b, :gone] = -1
        got = run_attn(bt, q, sk, window)
        ne.device_check()
        check(got, ref, mag, 0x1357)


def test_attention_odd_values_stay_with_the_rows_that_see_them():
    """NaNs and infinities among the keys and values of tokens that some rows of a
    tile see and others do not: before a window, and after a row's position."""
    torch_cuda()
    inf, nan = np.inf, np.nan
    for mx, D, Hq, Hkv, lens, window in (
            (False, 64, 16, 2, [(5, 70)], 0), (False, 64, 16, 2, [(6, 200)], 40),
            (False, 128, 12, 4, [(4, 33), (3, 300)], 0), (False, 64, 64, 8, [(90, 150)], 0),
            (False, 128, 16, 2, [(70, 260)], 30), (True, 64, 16, 2, [(5, 70)], 9),
            (True, 128, 8, 1, [(60, 100)], 0)):
        say(f"odd values mx={mx} D={D} lens={lens} window={window}")
        rng = np.random.default_rng(D + window)
        bt = Batch(rng, lens, 16, Hkv, D, mx).fill(rng)
        for b, (n, t) in enumerate(lens):
            at = [t - 1, t - 2, t - n + 1]
            if window:
                at += [t - n - window + 1, t - n - window + 2]
            pg, rows = bt.places(b)
            k, v = bt.get("k", b).astype(np.float32), bt.get("v", b).astype(np.float32)
            k[t - 1, 0, 2] = nan
            for i, a in enumerate(at):
                v[a, 0, i] = (nan, inf, -inf, inf, nan)[i]
                v[a, -1, 33 + i] = (inf, inf, nan, -inf, inf)[i]
            for x, w in (("k", k), ("v", v)):
                if mx:
                    bt.put(x, pg, rows, w)
                else:  # every value is a bf16 one
                    getattr(bt, x)[pg, :, rows] = (w.view(np.uint32) >> 16).astype(np.uint16)
        q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32))
        got = f32(run_attn(bt, q, None, window)).astype(np.float64)
        ne.device_check()
        some = 0
        for b, (n, t) in enumerate(lens):
            k, v = bt.get("k", b), bt.get("v", b)
            for i in range(n):
                p = t - n + i
                lo = max(0, p - window + 1) if window else 0
                for h in range(Hq):
                    row, kv = int(bt.starts[b]) + i, h // (Hq // Hkv)
                    with np.errstate(invalid="ignore"):
                        s = k[lo:p + 1, kv] @ f32(q[row, h]).astype(np.float64) / np.sqrt(D)
                        e = np.exp(s - s.max()) if np.isfinite(s).all() else np.full_like(s, nan)
                        e = (e / e.sum())[:, None]
                        want = (e * v[lo:p + 1, kv]).sum(0)
                        mag = (e * np.abs(v[lo:p + 1, kv])).sum(0)
                    fine = np.isfinite(want)
                    some += int((~fine).sum())
                    g = got[row, h]
                    assert np.array_equal(np.isnan(g), np.isnan(want)), (b, i, h)
                    odd = ~fine & ~np.isnan(want)
                    assert np.array_equal(g[odd], want[odd])
                    bound = 2.0 ** -8 * np.abs(want[fine]) + (2.0 ** -8 + 2.0 ** -12) * mag[fine]
                    assert (np.abs(g[fine] - want[fine]) <= bound + 1e-30).all(), (b, i, h)
        assert some > 0


def test_sinks_of_minus_infinity_are_none():
    torch_cuda()
    bt, q, sk = attn_case(False, 64, 8, 2, 16, [(1, 40), (2, 9)], seed=16)
    d = bt.dev()
    none = to_dev((np.full(8, -np.inf, np.float32).view(np.uint32) >> 16).astype(np.uint16))
    out = to_dev(np.full(q.shape, 0x1357, np.uint16))
    ne.paged_attn(d["kv"], to_dev(q), none, d["q_start"], d["kv_len"], d["table"], out, 8)
    ref, mag = attention(bt, f32(q), None, 0)
    check(to_host(out), ref, mag, 0x1357)
    d["table"] = to_dev(np.full_like(bt.table, -1))
    ne.paged_attn(d["kv"], to_dev(q), none, d["q_start"], d["kv_len"], d["table"], out, 8)
    assert not to_host(out).any()
    with pytest.raises(ne.NeonError):
        ne.device_check()


def test_attention_nothing_visible_gives_zero():
    """Every page of a sequence hidden, with and without sinks."""
    torch_cuda()
    for sinks in (True, False):
        bt, q, sk = attn_case(True, 64, 8, 1, 16, [(1, 20), (3, 40)], sinks=sinks, seed=8)
        d = bt.dev()
        d["table"] = to_dev(np.full_like(bt.table, -1))
        got = run_attn(bt, q, sk, 0, d=d)
        assert not got.any()
        with pytest.raises(ne.NeonError):
            ne.device_check()


@pytest.mark.parametrize("q_start,kv_len", [
    ([0, 1, 0], [5, 5]),      # falling
    ([0, 1, 9], [5, 5]),      # past the rows
    ([-1, 1, 2], [5, 5]),
    ([0, 1, 2], [5, 99]),     # past the table
    ([0, 1, 2], [5, -3]),
    ([0, 1, 4], [5, 2]),      # fewer tokens than rows
])
def test_sequences_that_do_not_fit_are_left_out(q_start, kv_len):
    torch_cuda()
    rng = np.random.default_rng(1)
    bt = Batch(rng, [(1, 5), (1, 5)], 16, 1, 64, False, pad=2, width=2).fill(rng)
    q = bf16(rng.normal(size=(4, 2, 64)).astype(np.float32))
    d = bt.dev()
    d["q_start"] = to_dev(np.array(q_start, np.int32))
    d["kv_len"] = to_dev(np.array(kv_len, np.int32))
    got = run_attn(bt, q, None, 0, d=d)
    with pytest.raises(ne.NeonError) as e:
        ne.device_check()
    assert e.value.status == ne.NEON_EINVAL
    assert (got[2:] == 0x1357).all()
    if q_start[0] == 0 and q_start[1] == 1:  # the sequence that fits is done
        ref, mag = attention(bt, f32(q), None, 0)
        check(got[:1], ref[:1], mag[:1], 0x1357)
    x = to_dev(bf16(rng.normal(size=(4, 4, 64)).astype(np.float32)))
    q_out = to_dev(np.full((4, 2, 64), 0x2468, np.uint16))
    before = to_host(d["k"]).copy()
    ne.paged_append(d["kv"], x, None, d["q_start"], d["kv_len"], d["table"], q_out, 2)
    with pytest.raises(ne.NeonError):
        ne.device_check()
    assert (to_host(q_out)[2:] == 0x2468).all()
    changed = (to_host(d["k"]) != before).any((1, 3))
    assert changed.sum() <= 1


def test_append_refuses_positions_past_the_table_and_bad_pages():
    torch_cuda()
    rng = np.random.default_rng(2)
    bt = Batch(rng, [(1, 5), (1, 12), (1, 3)], 16, 1, 64, False, q_start=False).fill(rng)
    d = bt.dev()
    t = bt.table.copy()
    t[2, 0] = bt.n_pages + 4
    d["table"] = to_dev(t)
    x = bf16(rng.normal(size=(3, 4, 64)).astype(np.float32))
    table = rope_table(8, 64)
    q_out = to_dev(np.full((3, 2, 64), 0x2468, np.uint16))
    ne.paged_append(d["kv"], to_dev(x), to_dev(table), None, d["kv_len"], d["table"], q_out, 2)
    with pytest.raises(ne.NeonError):
        ne.device_check()
    got = to_host(q_out)
    assert (got[1] == 0x2468).all()  # position 11, a table of 8
    want = bf16(rotate(f32(x[2:3, :2]), table, np.array([2])))
    assert np.array_equal(got[2:], want)  # q does not need the page
    pg, at = bt.places(0, 4)
    bt.put("k", pg, at, rotate(f32(x[:1, 2:3]), table, np.array([4])))
    bt.put("v", pg, at, f32(x[:1, 3:]))
    assert np.array_equal(to_host(d["k"]), bt.k) and np.array_equal(to_host(d["v"]), bt.v)


def test_row_starts_or_not_same_result():
    torch_cuda()
    bt, q, sk = attn_case(False, 64, 64, 8, 32, [(1, n) for n in (3, 900, 64)], seed=11)
    d = bt.dev()
    a = run_attn(bt, q, sk, 0, d=d)
    d["q_start"] = None
    b = run_attn(bt, q, sk, 0, d=d)
    ref, mag = attention(bt, f32(q), sk, 0)
    check(a, ref, mag, 0)
    check(b, ref, mag, 0)


def test_strided_queries():
    """q as a slice of the projection's rows."""
    torch_cuda()
    bt, q, sk = attn_case(False, 64, 16, 2, 16, [(3, 90), (1, 20)], seed=12)
    rows = np.full((4, 24 * 64), 0x7FC0, np.uint16)
    rows[:, :16 * 64] = q.reshape(4, -1)
    d = bt.dev()
    out = empty_dev((4, 16 * 64), np.uint16)
    ne.paged_attn(d["kv"], to_dev(rows)[:, :16 * 64], to_dev(bf16(sk)), d["q_start"], d["kv_len"],
                  d["table"], out, 16)
    ref, mag = attention(bt, f32(q), sk, 0)
    check(to_host(out).reshape(4, 16, 64), ref, mag, 0)


@pytest.mark.parametrize("mx,D", [(False, 128), (True, 128)])
def test_pools_past_4_gib(mx, D):
    """Pages whose offsets pass 32 bits."""
    torch = torch_cuda()
    rng = np.random.default_rng(13)
    Hkv, page = 8, 256
    per = Hkv * page * (D // 2 if mx else D * 2)  # bytes
    n_pages = (1 << 32) // per + 40
    bt = Batch(rng, [(2, 700), (1, 300)], page, Hkv, D, mx).fill(rng)
    shift = n_pages - bt.n_pages  # the batch's pages at the end of a larger pool
    d = bt.dev()
    big = {}
    for c in ("k", "v") + (("ks", "vs") if mx else ()):
        big[c] = torch.empty((n_pages,) + tuple(d[c].shape[1:]), dtype=d[c].dtype, device="cuda")
        big[c][shift:] = d[c]
    d["kv"] = ne.paged_kv(big["k"], big["v"], big.get("ks"), big.get("vs"))
    d["table"] = to_dev(np.where(bt.table >= 0, bt.table + shift, bt.table).astype(np.int32))
    q = bf16(rng.normal(size=(3, 16, D)).astype(np.float32))
    got = run_attn(bt, q, None, 0, d=d)
    ref, mag = attention(bt, f32(q), None, 0)
    check(got, ref, mag, 0)
    x = bf16(rng.normal(size=(3, 16 + 2 * Hkv, D)).astype(np.float32))
    q_out, k_out, v_out = (empty_dev((3, h, D), np.uint16) for h in (16, Hkv, Hkv))
    ne.paged_append(d["kv"], to_dev(x), None, d["q_start"], d["kv_len"], d["table"], q_out, 16)
    ne.paged_gather(d["kv"], d["q_start"], d["kv_len"], d["table"], k_out, v_out)
    w = f32(x[:, 16:16 + Hkv])
    want = bf16(values(*quantise(w)).astype(np.float32)) if mx else bf16(w)
    assert np.array_equal(to_host(k_out) & 0x7FFF, want & 0x7FFF)
    ne.device_check()


@pytest.mark.parametrize("mx", [False, True])
def test_steps_as_a_server_runs_them(mx):
    """Prompts, then decode steps, each append -> attention -> sample, captured
    into a graph and replayed between eager work; against plain forms."""
    torch = torch_cuda()
    rng = np.random.default_rng(21)
    Hq, Hkv, D, page, V = 16, 2, 64, 16, 500
    B, n0, steps = 3, [20, 1, 70], 5
    lens = [(n, n + steps) for n in n0]
    bt = Batch(rng, lens, page, Hkv, D, mx)
    bt.lens = [(n, n) for n in n0]
    bt.kv_len = np.array(n0, np.int32)
    d = bt.dev()
    table_h = rope_table(100, D)
    table = to_dev(table_h)
    sk = f32(bf16(rng.normal(size=Hq).astype(np.float32)))
    sinks = to_dev(bf16(sk))
    heads = Hq + 2 * Hkv
    x = to_dev(bf16(rng.normal(size=(sum(n0), heads * D)).astype(np.float32)))
    q = empty_dev((sum(n0), Hq, D), np.uint16)
    out = empty_dev((sum(n0), Hq, D), np.uint16)
    ne.paged_append(d["kv"], x, table, d["q_start"], d["kv_len"], d["table"], q, Hq)
    ne.paged_attn(d["kv"], q, sinks, d["q_start"], d["kv_len"], d["table"], out, Hq)

    def pull(bt, lens):
        bt.lens = lens
        for c in ("k", "v") + (("ks", "vs") if mx else ()):
            setattr(bt, c, to_host(d[c]).copy())

    pull(bt, [(n, n) for n in n0])
    ref, mag = attention(bt, f32(to_host(q)), sk, 0)
    check(to_host(out), ref, mag, 0)

    # decode steps: one graph, inputs written into its buffers
    step_x = torch.empty((B, heads * D), dtype=torch.int16, device="cuda")
    q1, o1 = empty_dev((B, Hq, D), np.uint16), empty_dev((B, Hq, D), np.uint16)
    logits = torch.empty((B, V), dtype=torch.float32, device="cuda")
    u = torch.empty(B, dtype=torch.float32, device="cuda")
    top_p = torch.full((B,), 0.9, device="cuda")
    ids = torch.zeros(B, dtype=torch.int32, device="cuda")
    wb, cb = ne.paged_attn_workspace(B, B, Hq, Hkv, D)
    ws = torch.empty(max(wb, 1), dtype=torch.uint8, device="cuda")
    counters = torch.zeros(max(cb, 1), dtype=torch.uint8, device="cuda")
    sws = torch.empty(max(ne.sample_rows_workspace(B, V), 1), dtype=torch.uint8, device="cuda")

    def step():
        ne.paged_append(d["kv"], step_x, table, None, d["kv_len"], d["table"], q1, Hq)
        ne.paged_attn(d["kv"], q1, sinks, None, d["kv_len"], d["table"], o1, Hq, workspace=ws,
                      counters=counters)
        ne.sample_rows(logits, u, ids, top_p=top_p, workspace=sws)

    d["kv_len"] += 1
    step_x.copy_(to_dev(bf16(rng.normal(size=(B, heads * D)).astype(np.float32))))
    logits.normal_()
    u.uniform_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()  # before the capture, as torch asks for
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(1, steps + 1):
        if i > 1:
            d["kv_len"] += 1
        step_x.copy_(to_dev(bf16(rng.normal(size=(B, heads * D)).astype(np.float32))))
        logits.normal_()
        u.uniform_()
        graph.replay()
        got, drawn, qh = to_host(o1), to_host(ids), to_host(q1)
        pull(bt, [(1, n + i) for n in n0])
        bt.starts = np.arange(B + 1)
        ref, mag = attention(bt, f32(qh), sk, 0)
        check(got, ref, mag, 0)
        step()  # eager, on the same inputs
        assert np.array_equal(to_host(o1), got) and np.array_equal(to_host(ids), drawn)
        bt.starts = np.cumsum([0] + n0)
    ne.device_check()


def test_two_streams():
    """Two calls at once, each with its own workspace."""
    torch = torch_cuda()
    made = [attn_case(mx, 64, 64, 8, 64, [(1, 3000), (1, 100)], seed=30 + mx) for mx in (0, 1)]
    devs = [bt.dev() for bt, _, _ in made]
    streams = [torch.cuda.Stream() for _ in made]
    ins = [(to_dev(q), to_dev(bf16(sk)), empty_dev(q.shape, np.uint16)) for _, q, sk in made]
    wb, cb = ne.paged_attn_workspace(2, 2, 64, 8, 64)
    ws = [(torch.empty(max(wb, 1), dtype=torch.uint8, device="cuda"),
           torch.zeros(max(cb, 1), dtype=torch.uint8, device="cuda")) for _ in made]
    torch.cuda.synchronize()
    for _ in range(20):
        for d, s, (q, sk, out), (w, c) in zip(devs, streams, ins, ws):
            ne.paged_attn(d["kv"], q, sk, None, d["kv_len"], d["table"], out, 64, stream=s,
                          workspace=w, counters=c)
    torch.cuda.synchronize()
    for (bt, q, sk), (_, _, out) in zip(made, ins):
        ref, mag = attention(bt, f32(q), sk, 0)
        check(to_host(out), ref, mag, 0)


def test_wrapper_refusals():
    torch = torch_cuda()
    rng = np.random.default_rng(1)
    bt = Batch(rng, [(1, 5), (1, 5)], 16, 2, 64, False, q_start=False).fill(rng)
    d = bt.dev()
    q = empty_dev((2, 4, 64), np.uint16)
    out = empty_dev((2, 4, 64), np.uint16)
    args = (d["kv_len"], d["table"])
    ne.paged_attn(d["kv"], q, None, None, *args, out, 4)
    for call in (
        lambda: ne.paged_attn(d["kv"], q, None, None, *args, out[:1], 4),
        lambda: ne.paged_attn(d["kv"], q, None, None, *args, out, 6),
        lambda: ne.paged_attn(d["kv"], q[:1], None, None, *args, out, 4),
        lambda: ne.paged_attn(d["kv"], q.transpose(1, 2), None, None, *args, out, 4),
        lambda: ne.paged_attn(d["kv"], q, None, None, d["kv_len"].cpu(), d["table"], out, 4),
        lambda: ne.paged_attn(d["kv"], q, None, None, d["kv_len"].long(), d["table"], out, 4),
        lambda: ne.paged_attn(d["kv"], q, q[0, 0, :3], None, *args, out, 4),
        lambda: ne.paged_gather(d["kv"], None, *args, q[:, :1].contiguous(), q),
        lambda: ne.paged_append(d["kv"], q, None, None, *args, out, 4),
        lambda: ne.paged_kv(d["k"], d["v"][:1]),
        lambda: ne.paged_kv(d["k"], d["v"], d["k"], d["v"]),
        lambda: ne.sample_rows(torch.zeros(2, 9, device="cuda"), torch.zeros(1, device="cuda"),
                               torch.zeros(2, dtype=torch.int32, device="cuda")),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ne.NeonError) as e:  # 3 query heads over 2 KV heads
        ne.paged_attn(d["kv"], q[:, :3].contiguous(), None, None, *args, out, 3)
    assert e.value.status == ne.NEON_EINVAL
    if ne.paged_attn_workspace(2, 2, 4, 2, 64)[0] > 1:
        with pytest.raises(ne.NeonError):
            ne.paged_attn(d["kv"], q, None, None, *args, out, 4,
                          workspace=torch.empty(1, dtype=torch.uint8, device="cuda"))


def test_wrapper_takes_no_rows():
    rng = np.random.default_rng(2)
    bt = Batch(rng, [(0, 5), (0, 0)], 16, 2, 64, False, q_start=True).fill(rng)
    d = bt.dev()
    args = (d["q_start"], d["kv_len"], d["table"])
    qkv, q, kv = (empty_dev((0, h, 64), np.uint16) for h in (8, 4, 2))
    ne.paged_append(d["kv"], qkv, None, *args, q, 4)
    ne.paged_gather(d["kv"], *args, kv, kv)
    ne.paged_attn(d["kv"], q, None, *args, q, 4)
    ne.device_check()


def test_wrapper_refuses_overlapping_rows_and_other_kinds():
    torch = torch_cuda()
    rng = np.random.default_rng(1)
    bt = Batch(rng, [(1, 5), (1, 5)], 16, 2, 64, False, q_start=False).fill(rng)
    d = bt.dev()
    q = empty_dev((2, 4, 64), np.uint16)
    args = (d["kv_len"], d["table"])
    logits, u = torch.zeros((2, 99), device="cuda"), torch.zeros(2, device="cuda")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    ne.sample_rows(logits, u, ids)
    for call in (
        lambda: ne.paged_attn(d["kv"], q[:1].expand(2, 4, 64), None, None, *args, q, 4),
        lambda: ne.paged_attn(d["kv"], q, None, None, d["kv_len"].float(), d["table"], q, 4),
        lambda: ne.paged_attn(d["kv"], q, None, None, d["kv_len"], d["table"].float(), q, 4),
        lambda: ne.sample_rows(logits[:1].expand(2, 99), u, ids),
        lambda: ne.sample_rows(logits, u, u),
        lambda: ne.sample_rows(logits, ids, ids),
        lambda: ne.sample_rows(logits, u, ids, temperature=ids),
        lambda: ne.sample_rows(logits, u, ids, top_k=u),
        lambda: ne.sample_rows(logits, u[0].expand(2), ids),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("handle", [False, True])
def test_own_scratch_belongs_to_the_stream_of_the_call(handle):
    """Calls without a workspace, on a stream that is behind, while the current
    stream takes and writes memory of the same size: what a call allocates must
    not be that memory."""
    torch = torch_cuda()
    bt, q, sk = attn_case(False, 64, 64, 8, 64, [(1, 3000), (1, 100)], seed=30)
    d, qd, skd = bt.dev(), to_dev(q), to_dev(bf16(sk))
    outs = [empty_dev(q.shape, np.uint16) for _ in range(8)]
    side = torch.cuda.Stream()
    big = torch.randn((4096, 4096), device="cuda")
    wb, cb = ne.paged_attn_workspace(2, 2, 64, 8, 64)
    ne.paged_attn(d["kv"], qd, skd, None, d["kv_len"], d["table"], outs[0], 64)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            big = big @ big * 1e-3
    for out in outs:
        ne.paged_attn(d["kv"], qd, skd, None, d["kv_len"], d["table"], out, 64,
                      stream=side.cuda_stream if handle else side)
        junk = [torch.full((max(n, 1),), 0x7F, dtype=torch.uint8, device="cuda") for n in (wb, cb)]
    torch.cuda.synchronize()
    del junk
    ref, mag = attention(bt, f32(q), sk, 0)
    for out in outs:
        check(to_host(out), ref, mag, 0)


def test_overlapping_row_starts_leave_the_counters_zero():
    """Starts 0, 1280, 0, 1280, ...: every second sequence is one that fits, and
    all of them together make more units than the grid has blocks, with the long
    one's chunks across its end.  The call reports it, and the next one is right."""
    torch = torch_cuda()
    rng = np.random.default_rng(9)
    n, B, long_at = 1280, 119, 60
    bt = Batch(rng, [(n, n)], 4096, 1, 64, False).fill(rng)
    d = bt.dev()
    q = bf16(rng.normal(size=(n, 1, 64)).astype(np.float32))
    qd, out = to_dev(q), empty_dev(q.shape, np.uint16)
    starts = to_dev(np.array([0, n] * ((B + 1) // 2), np.int32))
    lens = np.full(B, n, np.int32)
    lens[long_at] = 200000
    table = np.full((B, 49), int(bt.table[0, 0]), np.int32)
    wb, cb = ne.paged_attn_workspace(n, B, 1, 1, 64)
    ws = torch.empty(wb, dtype=torch.uint8, device="cuda")
    counters = torch.zeros(cb, dtype=torch.uint8, device="cuda")
    ne.paged_attn(d["kv"], qd, None, starts, to_dev(lens), to_dev(table), out, 1, workspace=ws,
                  counters=counters)
    with pytest.raises(ne.NeonError):
        ne.device_check()
    assert not counters.any().item()
    ne.paged_attn(d["kv"], qd, None, d["q_start"], d["kv_len"], d["table"], out, 1, workspace=ws,
                  counters=counters)
    ref, mag = attention(bt, f32(q), None, 0)
    check(to_host(out), ref, mag, 0)
    ne.device_check()


@pytest.mark.parametrize("mx,D,Hq,Hkv,rows,length", [
    (False, 64, 1, 1, 128, 1000),   # few chunks of a whole tile, of more than 64 rows
    (False, 128, 1, 1, 100, 1000),
    (True, 64, 1, 1, 70, 2000),
    (True, 128, 2, 2, 200, 2000),   # the second tile of 72
    (False, 64, 1, 1, 40, 1000),    # of up to 64
    (False, 128, 3, 1, 11, 1500),
    (False, 64, 1, 1, 130, 6000),   # more than 8 chunks
    (True, 128, 1, 1, 130, 6000),
    (False, 64, 1, 1, 40, 40000),   # more than 32
    (False, 128, 1, 1, 128, 40000),
    (False, 64, 1, 1, 128, 512),    # one
    (False, 64, 1, 1, 128, 513),
])
def test_attention_joins_of_many_rows(mx, D, Hq, Hkv, rows, length):
    torch_cuda()
    bt, q, sk = attn_case(mx, D, Hq, Hkv, 64, [(rows, length)], seed=rows + length)
    ref, mag = attention(bt, f32(q), sk, 0)
    check(run_attn(bt, q, sk, 0), ref, mag, 0x1357)


@pytest.mark.parametrize("D,lens", [(64, [(1, 70)]), (64, [(3, 300)]), (128, [(1, 700)]),
                                    (128, [(60, 300)]), (64, [(200, 600)])])
def test_infinities_that_every_row_sees(D, lens):
    """A row that sees one infinity among the values of a dim gets it; both, or a NaN:
    NaN.  Weights here are above 2^-40, so no product underflows."""
    torch_cuda()
    rng = np.random.default_rng(5)
    bt = Batch(rng, lens, 16, 2, D, False).fill(rng)
    odd = {0: np.inf, 1: -np.inf, 2: np.nan, 40: np.inf}
    for b, (n, t) in enumerate(lens):
        pg, rows = bt.places(b)
        v = bt.get("v", b).astype(np.float32)
        for d, x in odd.items():
            v[7, :, d] = x
        v[3, 1, 40] = -np.inf
        bt.v[pg, :, rows] = (v.view(np.uint32) >> 16).astype(np.uint16)
    q = bf16(rng.normal(size=(bt.n_rows, 4, D)).astype(np.float32))
    got = f32(run_attn(bt, q, None, 0))
    assert (got[:, :, 0] == np.inf).all() and (got[:, :, 1] == -np.inf).all()
    assert np.isnan(got[:, :, 2]).all()
    assert (got[:, :2, 40] == np.inf).all() and np.isnan(got[:, 2:, 40]).all()
    rest = [d for d in range(D) if d not in odd]
    ref, mag = attention(bt, f32(q), None, 0)
    off = np.abs(got[..., rest] - ref[..., rest])
    assert (off <= 2.0 ** -8 * np.abs(ref[..., rest]) + (2.0 ** -8 + 2.0 ** -12) * mag[..., rest]).all()


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens,width,window,q_start", [
    (False, 64, 8, 1, [(250, 254)], None, 0, True),
    (False, 64, 8, 1, [(250, 254)], 900, 0, True),  # the host cannot tell that it is small
    (True, 128, 2, 2, [(319, 583), (85, 227), (221, 418)], 100, 0, True),
    (False, 128, 12, 2, [(150, 254), (149, 149), (1, 90), (0, 0)], 300, 33, True),
    (True, 64, 1, 1, [(40, 60)] * 70, 90, 0, True),  # more than 64 sequences
    (False, 64, 8, 1, [(256, 1024)], 900, 0, True),  # 128 tiles of 16 rows x 1024: the border
    (False, 64, 8, 1, [(256, 1026)], 900, 0, True),
    (False, 64, 64, 1, [(1, 500), (1, 30), (1, 1)], None, 0, False),  # 64 rows of one token
    (False, 64, 64, 1, [(1, 500), (1, 30), (1, 1)], 2000, 0, False),
])
def test_attention_of_small_calls(mx, D, Hq, Hkv, lens, width, window, q_start):
    torch_cuda()
    rng = np.random.default_rng(len(lens) + D)
    bt = Batch(rng, lens, 16, Hkv, D, mx, q_start=q_start, width=width).fill(rng)
    q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32) * 2)
    sk = f32(bf16(rng.normal(size=Hq).astype(np.float32)))
    ref, mag = attention(bt, f32(q), sk, window)
    check(run_attn(bt, q, sk, window), ref, mag, 0x1357)
    ne.device_check()
