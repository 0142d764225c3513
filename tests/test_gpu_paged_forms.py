"""GPU tests of the paged calls form by form: which kernel and which split a case
reaches is asserted from the launch's own rules (paged_util.Route).

Bounds are computed from the inputs.  With S = max_j sum_d |q_d k_d| / sqrt(D) over
the keys that a row sees, n of them, and A = sum_j p_j |v_j| in 64 bits:
  a score is a sum of D exact products in fp32, each addition off by at most 2^-23
  of S (truncated or rounded), then scaled, shifted by the maximum and raised to a
  power by instructions good to 2^-22 of S and 2^-22: (D + 4) 2^-23 S + 2^-22;
  a weight p_j is off by that relative to itself, and by as much again from the
  normalising sum;
  P is kept in two bf16 terms: 2^-16;
  sums of n terms in fp32: n 2^-23, and again in the normalising sum; of a cut axis a
  chunk's keys and then the chunks;
  the output is rounded to bf16: 2^-8 of itself.
So |got - ref| <= 2^-8 |ref| + 1.01 A (2 ((D + 4) 2^-23 S + 2^-22) + 2^-16 + n 2^-22)."""
import sys

import numpy as np
import pytest

import neonengine_amd as ne
from tests.gpu_util import empty_dev, to_dev, to_host, torch_cuda
from tests.paged_util import Batch, Route, attention, bf16, f32

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def limits(bt, q, ref, mag, window, route=None):
    """The bound above, per row, head and dim (rows of no sequence: 0)."""
    n_rows, Hq, D = q.shape
    S, seen = np.zeros((n_rows, Hq)), np.zeros(n_rows)
    for b, (n, t) in enumerate(bt.lens):
        if n == 0 or t == 0:
            continue
        k, r0 = np.abs(bt.get("k", b)), int(bt.starts[b])
        pos = np.arange(t - n, t)
        lo = np.maximum(0, pos - window + 1) if window else np.zeros(n, int)
        vis = (np.arange(t) <= pos[:, None]) & (np.arange(t) >= lo[:, None])
        seen[r0:r0 + n] = vis.sum(1)
        for h in range(Hq):
            s = np.abs(q[r0:r0 + n, h]).astype(np.float64) @ k[:, h // (Hq // bt.Hkv)].T
            S[r0:r0 + n, h] = np.where(vis, s, 0).max(1) / np.sqrt(D)
        if route is not None:
            seen[r0:r0 + n] = np.minimum(seen[r0:r0 + n], route.run(b))
    rel = 2 * ((D + 4) * 2.0 ** -23 * S + 2.0 ** -22) + 2.0 ** -16 + seen[:, None] * 2.0 ** -22
    return 2.0 ** -8 * np.abs(ref) + 1.01 * rel[..., None] * mag + 1e-30


def attend(bt, q, sk, window, left=0x1357, **kw):
    d = bt.dev()
    out = to_dev(np.full(q.shape, left, np.uint16))
    ne.paged_attn(d["kv"], to_dev(q), None if sk is None else to_dev(bf16(sk)), d["q_start"],
                  d["kv_len"], d["table"], out, q.shape[1], window=window, **kw)
    return to_host(out)


def compare(bt, q, sk, window, got=None, left=0x1357):
    if got is None:
        got = attend(bt, q, sk, window, left)
    ref, mag = attention(bt, f32(q), sk, window)
    none = np.isnan(mag)
    assert np.array_equal(got[none], np.full(none.sum(), left, np.uint16))
    bound = limits(bt, f32(q), np.where(none, 0, ref), np.where(none, 0, mag), window,
                   Route(bt, q.shape[1], window))
    g = f32(got).astype(np.float64)
    off = np.where(none, 0, np.abs(g - np.where(none, 0, ref)) / bound)
    say(f"  worst error / bound = {off.max():.3f}")
    assert off.max() <= 1.0, (off.max(), np.unravel_index(off.argmax(), off.shape))


def make(mx, D, Hq, Hkv, page, lens, window, seed, scale=0.5, sinks=True, **kw):
    rng = np.random.default_rng(seed)
    bt = Batch(rng, lens, page, Hkv, D, mx, **kw).fill(rng)
    q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32) * scale)
    sk = f32(bf16(rng.normal(size=Hq).astype(np.float32))) if sinks else None
    return bt, q, sk


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens,window,many", [
    (False, 64, 64, 8, [(1200, 1200)], 4, True),
    (False, 128, 32, 8, [(1100, 1300), (900, 900)], 3, True),
    (True, 64, 64, 8, [(1200, 1200)], 4, True),
    (True, 128, 32, 8, [(1100, 1300), (900, 900)], 3, True),
    (False, 64, 64, 8, [(n, n) for n in (5, 6, 3, 8, 2, 1, 4)] + [(500, 500)], 0, True),
    (False, 64, 64, 8, [(1, n) for n in (1, 2, 3, 4, 5, 6, 7, 8)], 0, False),
    (False, 128, 32, 8, [(2, n) for n in (2, 3, 4, 5, 6, 7, 8)], 4, False),
    (True, 64, 64, 8, [(1, n) for n in (1, 2, 3, 4, 5, 6, 7, 8)], 0, False),
    (True, 128, 32, 8, [(2, n) for n in (2, 3, 4, 5, 6, 7, 8)], 4, False),
])
def test_weights_keep_sixteen_bits(mx, D, Hq, Hkv, lens, window, many):
    """Rows that see few keys, where a weight's own rounding shows."""
    torch_cuda()
    say(f"weights mx={mx} D={D} Hq={Hq} Hkv={Hkv} lens={lens} window={window}")
    bt, q, sk = make(mx, D, Hq, Hkv, 16, lens, window, seed=D + window + mx)
    r = Route(bt, Hq, window)
    assert not r.near and any(r.many) is many
    compare(bt, q, sk, window)
    ne.device_check()


def odd_attention(bt, q, window):
    """attention() without sinks where keys and values hold NaNs and infinities: a
    row has those of the tokens that it sees, whatever their weight; and mag."""
    n_rows, Hq, D = q.shape
    out, mag = np.full((n_rows, Hq, D), np.nan), np.full((n_rows, Hq, D), np.nan)
    for b, (n, t) in enumerate(bt.lens):
        k, v, r0 = bt.get("k", b), bt.get("v", b), int(bt.starts[b])
        v = np.where(np.abs(v) >= 2.0 ** 128, np.copysign(np.inf, v), v)  # as bf16 reads them
        pos, key = np.arange(t - n, t), np.arange(t)
        seen = key[None] <= pos[:, None]
        if window:
            seen &= key[None] > pos[:, None] - window
        for h in range(Hq):
            g = h // (Hq // bt.Hkv)
            bad = ~np.isfinite(k[:, g]).all(1)
            kg = np.where(bad[:, None], 0, k[:, g])
            s = np.where(seen, q[r0:r0 + n, h].astype(np.float64) @ kg.T / np.sqrt(D), -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            p = e / e.sum(1, keepdims=True)
            vg = np.where(np.isfinite(v[:, g]), v[:, g], 0)
            o = p @ vg
            up, down, nan = (seen.astype(np.float64) @ x > 0 for x in
                             (v[:, g] == np.inf, v[:, g] == -np.inf, np.isnan(v[:, g])))
            o = np.where(up, np.inf, np.where(down, -np.inf, o))
            o = np.where(nan | (up & down) | (seen & bad).any(1)[:, None], np.nan, o)
            out[r0:r0 + n, h], mag[r0:r0 + n, h] = o, p @ np.abs(vg)
    return out, mag


def put_odd(bt, x, b, tok, head, dim, value):
    """One element of a token's key or value (MXFP4: its whole block is NaN then)."""
    pg, at = (int(i[0]) for i in bt.places(b, tok, tok + 1))
    if bt.mx:
        getattr(bt, x + "s")[pg, head, at, dim // 32] = 255
    else:
        getattr(bt, x)[pg, head, at, dim] = np.float32(value).view(np.uint32) >> 16


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens,window", [
    (False, 64, 64, 8, [(400, 450), (1, 30)], 0),
    (False, 64, 64, 8, [(500, 900)], 100),
    (False, 128, 32, 8, [(300, 700)], 0),
    (False, 128, 32, 8, [(900, 1000)], 70),
    (True, 64, 64, 8, [(400, 450), (1, 30)], 0),
    (True, 128, 32, 8, [(900, 1000)], 70),
])
def test_odd_values_in_tiles_of_many_rows(mx, D, Hq, Hkv, lens, window):
    """NaNs and infinities in tokens that all rows of a tile see (both terms of a
    weight meet them), that some see, and behind a window."""
    torch_cuda()
    say(f"odd values mx={mx} D={D} lens={lens} window={window}")
    bt, q, _ = make(mx, D, Hq, Hkv, 16, lens, window, seed=D + window + 7, sinks=False)
    r = Route(bt, Hq, window)
    assert not r.near and r.many[0]
    inf, nan = np.inf, np.nan
    n, t = lens[0]
    for i, tok in enumerate((t - n, t - n + 1, t - n + 66, t - 70, t - 2, t - 1)):
        put_odd(bt, "v", 0, tok, 0, i, (inf, nan, -inf, inf, nan, -inf)[i])
        put_odd(bt, "v", 0, tok, Hkv - 1, D - 10 + i % 2, (inf, inf, -inf, inf, inf, -inf)[i])
    if t > n:
        put_odd(bt, "v", 0, 0, 1, 5, inf)
        put_odd(bt, "v", 0, 1, 2, 6, nan)
    put_odd(bt, "k", 0, t - 1, 3, 2, nan)
    got = f32(attend(bt, q, None, window)).astype(np.float64)
    ne.device_check()
    want, mag = odd_attention(bt, f32(q), window)
    fine = np.isfinite(want)
    assert 0 < (~fine).sum() < fine.size
    assert np.array_equal(np.isnan(got), np.isnan(want))
    odd = ~fine & ~np.isnan(want)
    assert mx or odd.any()
    assert np.array_equal(got[odd], want[odd])
    k = getattr(bt, "ks" if mx else "k")  # for the bound: the NaN key counts as a zero
    pg, at = (int(i[0]) for i in bt.places(0, t - 1, t))
    k[pg, 3, at] = 0
    bound = limits(bt, f32(q), np.where(fine, want, 0), mag, window)
    off = np.where(fine, np.abs(np.where(fine, got - np.where(fine, want, 0), 0)) / bound, 0)
    say(f"  worst error / bound = {off.max():.3f}")
    assert off.max() <= 1.0


@pytest.mark.parametrize("D,Hq,Hkv,lens,window,many", [
    (64, 16, 2, [(2, 70), (2, 40)], 0, False),
    (64, 16, 2, [(4, 300)], 40, False),
    (128, 8, 2, [(6, 90)], 0, False),
    (128, 8, 2, [(5, 300)], 17, False),
    (64, 64, 8, [(400, 450)], 0, True),
    (128, 32, 8, [(900, 1000)], 70, True),
])
def test_mxfp4_values_past_bf16(D, Hq, Hkv, lens, window, many):
    """Scales of 2^126 and 2^127 make infinities of the larger codes: theirs are the
    rows that see them, and the finite values beside them stay."""
    torch_cuda()
    say(f"mxfp4 past bf16 D={D} lens={lens} window={window}")
    bt, q, _ = make(True, D, Hq, Hkv, 16, lens, window, seed=D + window, sinks=False)
    r = Route(bt, Hq, window)
    assert not r.near and r.many[0] is many

    def put(b, tok, head, block, scale, codes):  # codes: {dim of the block: code}
        pg, at = (int(i[0]) for i in bt.places(b, tok, tok + 1))
        bt.vs[pg, head, at, block] = scale
        row = bt.v[pg, head, at, 16 * block:16 * block + 16]
        row[:] = 0
        for d, code in codes.items():
            row[d // 2] |= code << 4 * (d % 2)

    n, t = lens[0]
    for i, tok in enumerate((t - 1, t - 2, t - n + 1)):
        put(0, tok, i % 2, 0, 254, {i: 7, 5 + i: 12})          # 6 and -2 times 2^127
        put(0, tok, i % 2, 1, 253, {i: 6, 9 + i: 15, 20: 0})   # 4 and -6 times 2^126
    put(0, t - 1, 1, 0, 253, {30: 5})                          # 3 times 2^126: finite
    if window:
        put(0, t - n - window + 1, 0, 1, 254, {31: 4})
    got = f32(attend(bt, q, None, window)).astype(np.float64)
    ne.device_check()
    want, mag = odd_attention(bt, f32(q), window)
    fine = np.isfinite(want)
    assert 0 < (~fine).sum() < fine.size
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert (np.abs(want[fine]) > 2.0 ** 100).any()
    bound = limits(bt, f32(q), np.where(fine, want, 0), mag, window)
    off = np.where(fine, np.abs(np.where(fine, got - np.where(fine, want, 0), 0)) / bound, 0)
    say(f"  worst error / bound = {off.max():.3f}")
    assert off.max() <= 1.0


@pytest.mark.parametrize("mx", [False, True])
def test_append_leaves_out_a_sequence_that_crosses_the_angles(mx):
    """Positions 6 .. 11 and a table of 8: none of the rows is written; the others
    are, and a sequence without rows may be longer than the table."""
    torch_cuda()
    rng = np.random.default_rng(31)
    Hq, Hkv, D, lens = 2, 1, 64, [(2, 8), (6, 12), (0, 30), (3, 5)]
    bt = Batch(rng, lens, 16, Hkv, D, mx).fill(rng)
    x = to_dev(bf16(rng.normal(size=(bt.n_rows, Hq + 2 * Hkv, D)).astype(np.float32)))
    table = rng.normal(size=(2, 12, D // 2)).astype(np.float32)

    def append(n_pos, starts, kv_len):
        d = bt.dev()
        q_out = to_dev(np.full((bt.n_rows, Hq, D), 0x2468, np.uint16))
        ne.paged_append(d["kv"], x, to_dev(np.ascontiguousarray(table[:, :n_pos])), to_dev(starts),
                        to_dev(kv_len), d["table"], q_out, Hq)
        return [to_host(q_out)] + [to_host(d[c]) for c in ("k", "v") + (("ks", "vs") if mx else ())]

    got = append(8, bt.q_start, bt.kv_len)
    with pytest.raises(ne.NeonError) as e:
        ne.device_check()
    assert e.value.status == ne.NEON_EINVAL
    gone = bt.kv_len.copy()
    gone[1] = 0  # a free place: its rows are left as they are
    want = append(12, bt.q_start, gone)
    ne.device_check()
    assert all(np.array_equal(g, w) for g, w in zip(got, want))
    assert (got[0][2:8] == 0x2468).all() and (got[0][[0, 1, 8, 9, 10]] != 0x2468).any((1, 2)).all()
    fits = bt.kv_len.copy()
    fits[1] = 8  # 6 rows, the last at position 7
    append(8, bt.q_start, fits)
    ne.device_check()


def test_wrappers_refuse_other_number_types():
    """fp16 has the size of bf16, int32 that of fp32."""
    torch = torch_cuda()
    rng = np.random.default_rng(1)
    bt = Batch(rng, [(1, 5), (1, 5)], 16, 2, 64, False, q_start=False).fill(rng)
    d = bt.dev()
    args = (None, d["kv_len"], d["table"])

    def rows(heads, dtype):
        return torch.zeros((2, heads, 64), dtype=dtype, device="cuda")

    b, h = torch.bfloat16, torch.float16
    sinks = torch.zeros(4, dtype=b, device="cuda")
    logits, ids = torch.zeros((2, 99), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    u = torch.zeros(2, device="cuda")
    ne.paged_attn(d["kv"], rows(4, b), sinks, *args, rows(4, b), 4)
    ne.paged_append(d["kv"], rows(8, b), None, *args, rows(4, b), 4)
    ne.paged_append(d["kv"], rows(8, torch.int16), None, *args, rows(4, torch.int16), 4)  # bf16 bits
    ne.paged_gather(d["kv"], *args, rows(2, b), rows(2, b))
    ne.sample_rows(logits, u, ids)
    ne.device_check()
    for call in (
        lambda: ne.paged_attn(d["kv"], rows(4, h), sinks, *args, rows(4, b), 4),
        lambda: ne.paged_attn(d["kv"], rows(4, b), sinks.half(), *args, rows(4, b), 4),
        lambda: ne.paged_attn(d["kv"], rows(4, b), sinks, *args, rows(4, h), 4),
        lambda: ne.paged_append(d["kv"], rows(8, h), None, *args, rows(4, b), 4),
        lambda: ne.paged_append(d["kv"], rows(8, b), None, *args, rows(4, h), 4),
        lambda: ne.paged_gather(d["kv"], *args, rows(2, h), rows(2, b)),
        lambda: ne.paged_gather(d["kv"], *args, rows(2, b), rows(2, h)),
        lambda: ne.paged_kv(d["k"].view(h), d["v"].view(h)),
        lambda: ne.sample_rows(logits.int(), u, ids),
    ):
        with pytest.raises(ValueError):
            call()


def make_codes(D, Hq, Hkv, page, lens, seed, **kw):
    """As make() over MXFP4 pages, of codes and scales that are random themselves
    (quantising long caches on the host takes longer than the rest)."""
    rng = np.random.default_rng(seed)
    bt = Batch(rng, lens, page, Hkv, D, True, **kw)
    for b, (_, t) in enumerate(lens):
        pg, at = bt.places(b)
        for x in "kv":
            getattr(bt, x)[pg, :, at] = rng.integers(0, 256, (t, Hkv, D // 2), dtype=np.uint8)
            getattr(bt, x + "s")[pg, :, at] = rng.integers(124, 128, (t, Hkv, D // 32), dtype=np.uint8)
    q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32) * 0.3)
    return bt, q, f32(bf16(rng.normal(size=Hq).astype(np.float32)))


def build(mx, D, Hq, Hkv, page, lens, seed, **kw):
    if mx:
        return make_codes(D, Hq, Hkv, page, lens, seed, **kw)
    return make(False, D, Hq, Hkv, page, lens, 0, seed, **kw)


JOINS = [
    # (rows, length, Hkv, chunks): of the longest tile
    (330, 800, 24, (2, 4)),     # every tile has more than 64 rows
    (300, 900, 24, (2, 4)),     # the last one 44
    (200, 1500, 16, (5, 8)),
    (70, 2000, 32, (5, 8)),
    (60, 1900, 48, (5, 8)),     # no tile of more than 64
    (100, 4000, 16, (9, 32)),
    (40, 60000, 2, (33, 64)),
    (100, 60000, 2, (33, 64)),
]


@pytest.mark.parametrize("rows,length,Hkv,chunks", JOINS)
@pytest.mark.parametrize("mx,D", [(False, 64), (False, 128), (True, 64), (True, 128)])
def test_joins_in_the_many_row_kernel(rows, length, Hkv, chunks, mx, D):
    torch_cuda()
    say(f"join mx={mx} D={D} rows={rows} length={length} Hkv={Hkv}")
    bt, q, sk = build(mx, D, Hkv, Hkv, 64, [(rows, length)], rows + D)
    r = Route(bt, Hkv, 0)
    assert not r.near and r.many[0] and chunks[0] <= r.chunks(0) <= chunks[1], r.__dict__
    compare(bt, q, sk, 0)
    ne.device_check()


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens,window,why", [
    (False, 64, 64, 8, [(500, 1100)], 0, "share"),           # equal work for every block
    (False, 128, 32, 8, [(900, 1700), (1, 50)], 0, "share"),
    (True, 64, 64, 8, [(500, 1100), (3, 700)], 0, "share"),
    (True, 128, 32, 8, [(900, 1700)], 0, "share"),
    (False, 64, 8, 8, [(300, 5000), (200, 2100)], 1500, "cost"),  # windows and chunks
    (False, 128, 8, 8, [(300, 5000)], 2000, "cost"),
    (True, 64, 16, 8, [(300, 5000), (2, 40)], 1500, "cost"),
    (True, 128, 8, 8, [(300, 3000)], 1999, "cost"),
    (False, 64, 32, 8, [(700, 1900), (600, 1800)], 900, "share"),
])
def test_splits_of_the_many_row_kernel(mx, D, Hq, Hkv, lens, window, why):
    torch_cuda()
    say(f"split mx={mx} D={D} lens={lens} window={window}")
    bt, q, sk = build(mx, D, Hq, Hkv, 32, lens, D + window + len(lens))
    r = Route(bt, Hq, window)
    assert not r.near and r.many[0] and r.why["many"] == why and r.chunks(0) > 1, r.__dict__
    compare(bt, q, sk, window)
    ne.device_check()


def spread(B, short, long, at):
    """One row each: lengths around `short`, those of the places `at` around `long`."""
    return [(1, (long if b in at else short) + (b * 37) % 101) for b in range(B)]


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens", [
    (False, 64, 16, 8, spread(100, 400, 4000, (3, 10, 64, 66, 70, 95, 99))),
    (False, 128, 16, 8, spread(100, 400, 4000, (3, 10, 64, 66, 70, 95, 99))),
    (True, 64, 16, 8, spread(100, 400, 4000, (3, 10, 64, 66, 70, 95, 99))),
    (True, 128, 16, 8, spread(100, 400, 4000, (3, 10, 64, 66, 70, 95, 99))),
    (False, 64, 16, 4, spread(200, 500, 3000, (0, 63, 64, 127, 128, 130, 191, 192, 199))),
    (True, 64, 8, 4, spread(200, 500, 3000, (0, 63, 64, 127, 128, 130, 191, 192, 199))),
])
def test_split_sequences_past_the_first_64(mx, D, Hq, Hkv, lens):
    """The chunk is a block's share of the work, and sequences of every turn of the
    block finder are cut."""
    torch_cuda()
    say(f"past 64 mx={mx} D={D} B={len(lens)}")
    bt, q, sk = build(mx, D, Hq, Hkv, 64, lens, len(lens) + D, q_start=False)
    r = Route(bt, Hq, 0)
    assert r.why["few"] == "share" and not any(r.many), r.__dict__
    cut = [b for b in range(len(lens)) if r.chunks(b) > 1]
    assert cut[0] < 64 and len([b for b in cut if b >= 64]) >= 3
    compare(bt, q, sk, 0)
    ne.device_check()


@pytest.mark.parametrize("mx", [False, True])
def test_mixed_rows_past_the_first_64(mx):
    """Decode steps, drafts and prompt chunks of 150 sequences; both kernels."""
    torch_cuda()
    lens = [((1, 3, 0, 60 + b % 30)[b % 4], 90 + (b * 53) % 200 + (3000 if b in (5, 67, 70, 131, 133)
                                                               else 0)) for b in range(150)]
    bt, q, sk = build(mx, 64, 16, 4, 32, lens, 9, pad=2)
    r = Route(bt, 16, 0)
    assert not r.near and sum(r.many) > 30
    for kind in (True, False):
        cut = [b for b in range(150) if r.many[b] is kind and lens[b][0] and r.chunks(b) > 1]
        assert cut and cut[-1] >= 64, (kind, cut)
    compare(bt, q, sk, 0)
    ne.device_check()


@pytest.mark.parametrize("D,Hq,Hkv,lens,window", [
    (64, 64, 8, [(1, 500 + 110 * b) for b in range(40)], 0),
    (128, 16, 8, [(1, 300 + (b * 701) % 5000) for b in range(48)], 0),
    (64, 16, 8, [(2, 4000 - 50 * b) for b in range(30)], 3000),
])
def test_mxfp4_chunks_that_fit_the_chip_at_once(D, Hq, Hkv, lens, window):
    torch_cuda()
    say(f"fit D={D} B={len(lens)} window={window}")
    bt, q, sk = make_codes(D, Hq, Hkv, 64, lens, D + len(lens))
    r = Route(bt, Hq, window)
    assert r.fitted["few"] > 0 and max(map(r.chunks, range(len(lens)))) > 1, r.__dict__
    compare(bt, q, sk, window)
    ne.device_check()


def free_page_0(bt):
    """Page 0, which a block reads where a page id is no page, is nobody's: poison."""
    spare = np.setdiff1d(np.arange(bt.n_pages), bt.table)
    if 0 not in spare:
        bt.table[bt.table == 0] = spare[0]
    return bt


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens", [
    (False, 64, 64, 8, [(400, 450), (200, 333)]),
    (False, 128, 32, 8, [(500, 700)]),
    (True, 64, 64, 8, [(400, 450), (200, 333)]),
    (True, 128, 32, 8, [(500, 700)]),
])
def test_hidden_pages_in_tiles_of_many_rows(mx, D, Hq, Hkv, lens):
    torch_cuda()
    say(f"hidden mx={mx} D={D} lens={lens}")
    rng = np.random.default_rng(D)
    bt = free_page_0(Batch(rng, lens, 16, Hkv, D, mx)).fill(rng)
    q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32) * 0.5)
    r = Route(bt, Hq, 0)
    assert not r.near and all(r.many)
    good, t = bt.table, bt.table.copy()
    dead = {0: (0, 1, 5, 20, 27), 1: (2, 20)}  # groups of a tile, at its edges, a whole tile
    if len(lens) > 1:
        dead[1] = (4, 5, 6, 7)
    for b in range(len(lens)):
        for i, j in enumerate(dead[b]):
            t[b, j] = (bt.n_pages, -1, 1 << 30)[i % 3]
    bt.table = t
    got = attend(bt, q, None, 0)
    with pytest.raises(ne.NeonError):
        ne.device_check()
    bt.table = good
    ref, mag = attention(bt, f32(q), None, 0,
                         hidden=lambda b, n: np.isin(np.arange(n) // 16, dead[b]))
    off = np.abs(f32(got) - ref) / limits(bt, f32(q), ref, mag, 0)
    say(f"  worst error / bound = {off.max():.3f}")
    assert off.max() <= 1.0


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens,window", [
    (False, 64, 64, 8, [(600, 1500)], 200),
    (True, 128, 32, 8, [(900, 1600)], 100),
])
def test_many_rows_and_pages_behind_the_window(mx, D, Hq, Hkv, lens, window):
    """Their table entries are not looked at, their memory is poison."""
    torch_cuda()
    rng = np.random.default_rng(D)
    bt = free_page_0(Batch(rng, lens, 16, Hkv, D, mx)).fill(rng)
    q = bf16(rng.normal(size=(bt.n_rows, Hq, D)).astype(np.float32) * 0.5)
    r = Route(bt, Hq, window)
    assert not r.near and all(r.many)
    ref, mag = attention(bt, f32(q), None, window)
    bound = limits(bt, f32(q), ref, mag, window)
    n, t = lens[0]
    gone = (t - n - window + 1) // 16
    ids = bt.table[0, :gone].copy()
    bt.k[ids], bt.v[ids] = (0x77, 0x77) if mx else (0x7FC1, 0x7FC1)
    if mx:
        bt.ks[ids] = bt.vs[ids] = 255
    bt.table[0, :gone] = -1
    off = np.abs(f32(attend(bt, q, None, window)) - ref) / bound
    ne.device_check()
    assert off.max() <= 1.0


@pytest.mark.parametrize("mx", [False, True])
def test_many_rows_over_shared_and_repeated_pages(mx):
    torch_cuda()
    rng = np.random.default_rng(6)
    bt = Batch(rng, [(400, 900), (300, 500)], 16, 8, 64, mx).fill(rng)
    bt.table[1, :10] = bt.table[0, :10]
    bt.table[0, 30] = bt.table[0, 2]
    q = bf16(rng.normal(size=(bt.n_rows, 64, 64)).astype(np.float32) * 0.5)
    r = Route(bt, 64, 0)
    assert not r.near and all(r.many)
    compare(bt, q, None, 0)
    ne.device_check()


@pytest.mark.parametrize("mx,D,Hq,Hkv,rows,length,small", [
    (False, 64, 64, 8, 100, 500, True),    # 200000
    (True, 64, 64, 8, 100, 500, True),
    (False, 128, 8, 8, 300, 1000, True),   # 152000
    (True, 128, 8, 1, 300, 1000, True),
    (False, 128, 1, 1, 40, 60000, True),   # 180000, cut into many chunks
    (True, 64, 2, 2, 34, 40000, True),     # 240000
    (False, 64, 64, 8, 100, 700, False),   # 280000
    (False, 64, 8, 1, 512, 1050, False),   # 268800
])
def test_small_calls_on_both_sides_of_the_border(mx, D, Hq, Hkv, rows, length, small):
    torch_cuda()
    say(f"border mx={mx} D={D} rows={rows} length={length}")
    bt, q, sk = build(mx, D, Hq, Hkv, 32, [(rows, length)], rows + length)
    r = Route(bt, Hq, 0)
    assert not r.near and r.small is small
    compare(bt, q, sk, 0)
    ne.device_check()


@pytest.mark.parametrize("mx,D,Hq,Hkv,lens,window,many", [
    (False, 64, 16, 2, [(5, 300), (1, 40)], 0, False),
    (True, 128, 8, 2, [(3, 200), (2, 2)], 50, False),
    (False, 64, 64, 8, [(400, 450)], 0, True),
    (True, 128, 32, 8, [(500, 700)], 0, True),
])
def test_odd_queries_stay_in_their_rows(mx, D, Hq, Hkv, lens, window, many):
    """A NaN or an infinity in a query makes its row NaN, and no other; infinities
    among the values are found beside it."""
    torch_cuda()
    say(f"odd queries mx={mx} D={D} lens={lens}")
    bt, q, sk = make(mx, D, Hq, Hkv, 16, lens, window, seed=D + 77)
    r = Route(bt, Hq, window)
    assert not r.near and r.many[0] is many
    last = bt.n_rows - 1
    odd = [(0, 0), (1, Hq - 1), (last, 1)]
    for (row, h), x in zip(odd, (0x7FC0, 0x7F80, 0xFFC0)):
        q[row, h, 3] = x
    put_odd(bt, "v", 0, lens[0][1] - lens[0][0], 0, 5, np.inf)  # the first row's last key
    got = f32(attend(bt, q, sk, window)).astype(np.float64)
    ne.device_check()
    ok = np.ones(q.shape[:2], bool)
    for row, h in odd:
        assert np.isnan(got[row, h]).all()
        ok[row, h] = False
        q[row, h] = 0
    sees = np.zeros(q.shape, bool)
    sees[:lens[0][0], :Hq // Hkv, 0 if mx else 5:32 if mx else 6] = True
    if window:
        sees[window:] = False
    assert (np.isnan(got) if mx else got == np.inf)[sees & ok[..., None]].all()
    if mx:  # the block counts as zeros below
        pg, at = (int(i[0]) for i in bt.places(0, lens[0][1] - lens[0][0], lens[0][1] - lens[0][0] + 1))
        bt.vs[pg, 0, at, 0], bt.v[pg, 0, at, :16] = 127, 0
    else:
        put_odd(bt, "v", 0, lens[0][1] - lens[0][0], 0, 5, 0.0)
    ref, mag = attention(bt, f32(q), sk, window)
    off = np.abs(got - ref) / limits(bt, f32(q), ref, mag, window)
    assert off[ok[..., None] & ~sees].max() <= 1.0
