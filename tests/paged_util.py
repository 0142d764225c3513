"""Batches over a paged KV cache, and plain 64-bit forms of the paged
operators, for the tests of neon_paged_*."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def quantise(x):
    """MXFP4 of x [..., D] (float32 or float64) by the rule that
    neon_paged_append states: codes [..., D/2], scale bytes [..., D/32]."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    amax = np.where(bad, 1.0, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    m, e = np.frexp(amax)
    byte = np.where(amax > 0, np.clip(e - 3 + (m > 0.875) + 127, 0, 254), 127)
    y = np.abs(np.ldexp(np.where(bad[..., None], 0, b), 127 - byte[..., None]))
    # the nearest of the eight magnitudes; of two as near, the even code
    dist = np.abs(y[..., None] - E2M1[:8])
    near = dist == dist.min(-1, keepdims=True)
    code = np.where(near, np.arange(8) % 2 * 8 + np.arange(8), 99).argmin(-1)
    code = code | (np.signbit(b) * 8)
    code = np.where(bad[..., None], 0, code).reshape(x.shape).astype(np.uint8)
    byte = np.where(bad, 255, byte).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def values(codes, scales):
    """float64 values of MXFP4 codes and scale bytes."""
    v = E2M1[np.stack((codes & 15, codes >> 4), -1)].reshape(*scales.shape, 32)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * s[..., None]).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def bf16(x):
    """float32 -> bf16 bits, nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def f32(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


class Batch:
    """Sequences (rows, tokens) over randomly ordered pages.  Pages and rows
    that no sequence holds, and table entries past its pages, are poison."""

    def __init__(self, rng, lens, page, Hkv, D, mx, q_start=True, pad=0, spare=2, width=None):
        self.lens, self.page, self.Hkv, self.D, self.mx = lens, page, Hkv, D, mx
        need = [-(-t // page) for _, t in lens]
        self.n_pages = sum(need) + spare
        self.width = width or max(max(need), 1) + 1
        perm = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.width), -7, np.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = perm[at:at + k]
            at += k
        rows = [n for n, _ in lens]
        self.q_start = np.cumsum([0] + rows).astype(np.int32) if q_start else None
        self.starts = np.cumsum([0] + rows)
        self.n_rows = sum(rows) + pad
        self.kv_len = np.array([t for _, t in lens], np.int32)
        shape = (self.n_pages, Hkv, page)
        if mx:
            self.k, self.v = (np.full(shape + (D // 2,), 0x77, np.uint8) for _ in "kv")
            self.ks, self.vs = (np.full(shape + (D // 32,), 255, np.uint8) for _ in "kv")
        else:
            self.k, self.v = (np.full(shape + (D,), 0x7FC1, np.uint16) for _ in "kv")
            self.ks = self.vs = None

    def places(self, b, t0=0, t1=None):
        t = np.arange(t0, self.lens[b][1] if t1 is None else t1)
        return self.table[b, t // self.page], t % self.page

    def fill(self, rng, scale=1.0):
        """Random keys and values at every token that a sequence holds."""
        for b, (_, t) in enumerate(self.lens):
            pg, at = self.places(b)
            for x in "kv":
                w = f32(bf16(rng.normal(size=(t, self.Hkv, self.D)).astype(np.float32) * scale))
                self.put(x, pg, at, w)
        return self

    def put(self, x, pg, at, w):
        if self.mx:
            c, s = quantise(w)
            getattr(self, x)[pg, :, at] = c
            getattr(self, x + "s")[pg, :, at] = s
        else:
            getattr(self, x)[pg, :, at] = bf16(w)

    def get(self, x, b):
        """float64 rows [t][Hkv][D] of a sequence."""
        pg, at = self.places(b)
        if self.mx:
            return values(getattr(self, x)[pg, :, at], getattr(self, x + "s")[pg, :, at])
        return f32(getattr(self, x)[pg, :, at]).astype(np.float64)

    def dev(self):
        """The pools, the batch and the PagedKV on the device."""
        import neonengine_amd as ne
        from tests.gpu_util import to_dev
        d = {n: None if getattr(self, n) is None else to_dev(getattr(self, n))
             for n in ("k", "v", "ks", "vs", "table", "q_start", "kv_len")}
        d["kv"] = ne.paged_kv(d["k"], d["v"], d["ks"], d["vs"])
        return d


def attention(batch, q, sinks, window, hidden=lambda b, t: None):
    """float64 attention of q [n_rows][Hq][D], and per row and head the bound
    sum_j p_j |v_j| [n_rows][Hq][D].  Rows of no sequence are NaN in both.
    hidden(b, t): positions of sequence b that a bad page hides, or None."""
    n_rows, Hq, D = q.shape
    out = np.full((n_rows, Hq, D), np.nan)
    mag = out.copy()
    G = Hq // batch.Hkv
    for b, (n, t) in enumerate(batch.lens):
        if n == 0 or t == 0:
            continue
        k, v = batch.get("k", b), batch.get("v", b)
        gone = hidden(b, t)
        r0 = int(batch.starts[b])
        pos = np.arange(t - n, t)
        key = np.arange(t)
        seen = key[None] <= pos[:, None]
        if window:
            seen &= key[None] > pos[:, None] - window
        if gone is not None:
            seen &= ~gone[None]
        for h in range(Hq):
            g = h // G
            s = q[r0:r0 + n, h].astype(np.float64) @ k[:, g].T / np.sqrt(D)
            s = np.where(seen, s, -np.inf)
            top = np.maximum(s.max(1), sinks[h] if sinks is not None else -np.inf)
            top = np.where(np.isfinite(top), top, 0)
            e = np.where(seen, np.exp(s - top[:, None]), 0)
            den = e.sum(1) + (np.exp(sinks[h] - top) if sinks is not None else 0)
            p = e / np.where(den == 0, 1, den)[:, None]
            vg = np.where(seen.any(0)[:, None], v[:, g], 0)
            out[r0:r0 + n, h] = p @ vg
            mag[r0:r0 + n, h] = p @ np.abs(vg)
    return out, mag


SMALL = 262144  # 16-row tiles x keys x KV heads of a call that takes 16 rows at a time


class Route:
    """How neon_paged_attn takes a batch (the rules of its launch and of its block
    finder), so that a test can say which kernel and which split it reaches.
    many[b]: sequence b's rows are the many-row kernel's; of each kernel ("few",
    "many") chunk, its keys, and why: "share" (equal work for every block), "cost"
    (of the join) or "uncut"; fitted: chunks made larger to fit the chip at once."""

    def __init__(self, batch, Hq, window):
        lens, page, Hkv, B = batch.lens, batch.page, batch.Hkv, len(batch.lens)
        self.G = G = Hq // Hkv
        self.batch, self.Hkv, self.window = batch, Hkv, window
        holds = min(batch.table.shape[1] * page, 1 << 30)

        def keys(R, align):
            return min(holds, window + (R - 1) // G + align) if window > 0 else holds

        def blocks(units, most, target):
            return min(target // Hkv + 1 + units, units * -(-most // 256)) * Hkv

        rows, starts = batch.n_rows * G, batch.q_start is not None
        units = rows // 16 + B
        few = 0 if not starts and G > 32 else blocks(min(units, 2 * B), keys(16, 32), 1024)
        small = units * Hkv + SMALL // 256 + 2
        can = (rows > 32 if starts else G > 32) and small <= max(few, 2048)
        work = sum(-(-n * G // 16) * self.span(t, 16, 32) for n, t in lens) * Hkv
        self.small = can and work <= SMALL
        self.near = can and abs(work / SMALL - 1) < 0.01  # the kernel's fp32 sum may differ
        self.many = [t > 0 and n * G > 32 and not self.small for n, t in lens]
        self.chunk, self.why, self.fitted = {}, {}, {}
        for kind, R, align, target, places in (
                ("few", 16, 32, 1024, 256 * (3 if batch.D == 64 or batch.mx else 2)),
                ("many", 128, 64, 512, 512)):
            self._cut(kind, R, align, target, places)

    def span(self, t, R, align):
        return t if self.window <= 0 or self.window >= t else \
            min(t, self.window + (R - 1) // self.G + align)

    def _cut(self, kind, R, align, target, places):
        mine = [(n, t) for (n, t), m in zip(self.batch.lens, self.many)
                if n and t and m == (kind == "many")]
        if not mine:
            return
        tiles = [-(-n * self.G // R) for n, _ in mine]
        span = [self.span(t, R, align) for _, t in mine]
        share = sum(a * s for a, s in zip(tiles, span)) * self.Hkv * 1.001 / target
        most, fit = max(span), kind == "few" and self.batch.mx
        cost = ((10 if kind == "few" else 25) * most) ** 0.5
        least, why = max((share, "share"), (511, "uncut") if most <= 512 else (cost, "cost"))
        if kind == "few" and sum(tiles) * self.Hkv <= places and \
                most <= share * (target / (384 if fit else 256)) + 512 and most > least:
            least, why = most, "uncut"
        chunk = max(256, (int(least) + 128) & ~127)
        n = 0
        while fit and n < 3 and len(self.batch.lens) <= 64:
            over = sum(a * -(-s // chunk) for a, s in zip(tiles, span)) * self.Hkv / places
            if not 1 < over <= 2:
                break
            chunk, n = (int(chunk * over) + 128) & ~127, n + 1
        self.chunk[kind], self.why[kind], self.fitted[kind] = chunk, why, n

    def chunks(self, b):
        """Chunks of sequence b's longest tile."""
        n, t = self.batch.lens[b]
        kind = "many" if self.many[b] else "few"
        span = self.span(t, *((128, 64) if self.many[b] else (16, 32)))
        return -(-span // self.chunk[kind]) if n and t else 0

    def run(self, b):
        """The most terms that follow one another in a sum: a chunk's, then chunks."""
        return self.chunk["many" if self.many[b] else "few"] + self.chunks(b)
