"""The paged-serving operators as they are measured: appending rotated keys and
values to a paged cache (bf16 or MXFP4 pages), attention over it, and sampling
with a setting per row.

One step of a continuous batch is an append and an attention per layer and one
sampling call.  Shapes are those of the gpt-oss presets (64 query heads, 8 KV
heads of 64, a vocabulary of 201088, a window of 128) and generic ones (heads of
128, other group sizes and vocabularies).
"""
import math
import random

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _append(name, **k):
    return dict({"op": "append", "name": name, "format": "bf16", "B": 1, "rows": 1, "max_len": 1024,
                 "page": 64, "Hq": 64, "Hkv": 8, "D": 64}, **k)


def _attn(name, **k):
    return dict({"op": "attn", "name": name, "format": "bf16", "B": 1, "rows": 1, "max_len": 1024,
                 "page": 64, "Hq": 64, "Hkv": 8, "D": 64, "window": 0}, **k)


def _sample(name, **k):
    return dict({"op": "sample", "name": name, "B": 1, "V": 201088, "spread": 2.5}, **k)


def listed():
    """rows: of the longest sequence (the others have about as many, or fewer);
    max_len: the longest sequence's tokens; the other lengths are spread below."""
    return [
        # one token of each of 64 running sequences
        _append("append_decode", B=64, max_len=1500),
        # prompts of three requests, prefilled together
        _append("append_prompt", B=3, rows=4001, max_len=5000, page=128),
        # the same into a 4-bit cache, and the rows as the cache now holds them
        _append("append_prompt_mxfp4", format="mxfp4", B=3, rows=3001, max_len=4100, page=64),
        # the smallest call: one short chat, latency counts
        _attn("attn_one", max_len=301, page=16),
        # a full batch of chats of very different lengths
        _attn("attn_batch", B=64, max_len=8192),
        # the same on a sliding-window layer
        _attn("attn_window", B=64, max_len=8192, window=128),
        # prompt chunks behind a cached prefix
        _attn("attn_chunk", B=2, rows=2048, max_len=6001, page=128),
        # few very long contexts held in 4 bits
        _attn("attn_mxfp4_long", format="mxfp4", B=4, max_len=131072, page=256),
        # a batch in 4 bits, heads of 128
        _attn("attn_mxfp4_batch", format="mxfp4", B=48, max_len=6000, page=32, Hq=32, D=128),
        # one chat's next token
        _sample("sample_one"),
        # a full batch's next tokens
        _sample("sample_batch", B=64),
        # a smaller vocabulary of odd size, flatter logits
        _sample("sample_small", B=7, V=32003, spread=1.3),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(("append", "attn", "attn", "sample"))
    if op == "sample":
        B = log(1, 64)
        return {"op": op, "B": B, "V": log(700, 201088), "spread": round(rng.uniform(1.0, 3.5), 2)}
    Hkv = rng.choice((1, 2, 4, 8))
    D = rng.choice((64, 64, 128))
    c = {"op": op, "format": rng.choice(("bf16", "mxfp4")), "page": rng.choice((16, 32, 64, 128, 256)),
         "Hkv": Hkv, "Hq": Hkv * rng.choice((1, 2, 3, 4, 6, 8)), "D": D}
    kind = rng.choice(("single", "few", "chunk"))
    if kind == "chunk":
        c["B"] = rng.randint(1, 3)
        c["rows"] = log(64, 2000)
        c["max_len"] = c["rows"] + log(1, 3000)
    else:
        c["B"] = log(1, 64)
        c["rows"] = 1 if kind == "single" else rng.randint(2, 8)
        c["max_len"] = c["rows"] + log(16, max(17, min(60000, 400000 // c["B"])))
    if op == "append":
        c["max_len"] = min(c["max_len"], 4096)
    else:
        c["window"] = rng.choice((0, 0, 128, log(20, 4000)))
    return c


def _lengths(c):
    """(rows, tokens) of each sequence: the first is the longest, the others
    are spread over a factor of 64 below; every case has its own, fixed ones."""
    r = random.Random("%d %d %d" % (c["B"], c["rows"], c["max_len"]))
    out = [(c["rows"], c["max_len"])]
    for _ in range(c["B"] - 1):
        n = c["rows"] if c["rows"] == 1 else r.randint(max(1, c["rows"] // 4), c["rows"])
        top = max(c["max_len"], n)
        lo = max(n, top // 64)
        out.append((n, int(round(math.exp(r.uniform(math.log(lo), math.log(top)))))))
    return out


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _round_e2m1(y):
    """Codes (0..7) of magnitudes y, to the nearest E2M1 value, ties to even."""
    return ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5)
            + (y > 5.0))


def _quantise(x):
    """MXFP4 of x [..., D] (fp32): codes [..., D/2], scales [..., D/32]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    byte = torch.where(amax > 0, e - 1 - 2 + (m > 0.875).to(e.dtype) + 127, torch.full_like(e, 127))
    byte = byte.clamp(0, 254)
    y = torch.ldexp(b, (127 - byte).unsqueeze(-1))
    code = _round_e2m1(y.abs()) | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.reshape(x.shape)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), byte.to(torch.uint8)


def _values(codes, scales):
    """fp32 values of MXFP4 codes [..., D/2] with scales [..., D/32]."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1)
    v = v.reshape(*scales.shape, 32)
    v = torch.ldexp(v, (scales.to(torch.int32) - 127).unsqueeze(-1))
    return v.reshape(*codes.shape[:-1], -1)


def _pages(c, lens, g):
    """Page table [B][max_pages] of distinct pages in random order (-1 where a
    sequence has none), and the pool's page count."""
    page = c["page"]
    need = [-(-n // page) for _, n in lens]
    width = max(need)
    n_pages = sum(need) + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    return table, n_pages


def _rope_table(D, n_pos):
    """cos, then sin [2][n_pos][D/2], computed in 64 bits."""
    f = 150000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * f
    return torch.stack((a.cos(), a.sin())).to(torch.float32).cuda()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    if c["op"] == "sample":
        B, V = c["B"], c["V"]
        l = normal(B, V, scale=c["spread"], dtype=torch.float32)
        l[:, 7::50] = -math.inf  # tokens that a grammar forbids
        r = torch.rand((5, B), generator=g, device="cuda")
        s = {"c": c, "logits": l, "u": r[0].contiguous(),
             "temperature": (0.5 + r[1]).contiguous(),
             "top_p": (0.7 + 0.3 * r[2]).contiguous(),
             "min_p": (0.02 * r[3]).contiguous(),
             "top_k": torch.where(r[4] < 0.3, torch.zeros_like(r[4]), 20 + 2000 * r[4]).to(torch.int32)}
        s["top_k"].clamp_(max=V)
        s["out"] = torch.empty(B, dtype=torch.int32, device="cuda")
        if own:
            import neonengine_amd as ne
            n = ne.sample_rows_workspace(B, V)
            s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        return s

    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    lens = _lengths(c)
    table, n_pages = _pages(c, lens, g)
    rows = [n for n, _ in lens]
    n_rows = sum(rows)
    start = torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda()
    s = {"c": c, "table": table, "n_rows": n_rows, "q_start": start, "most": max(rows),
         "kv_len": torch.tensor([n for _, n in lens], dtype=torch.int32).cuda()}
    shape = (n_pages, Hkv, c["page"], D)
    if c["format"] == "bf16":
        s["k"], s["v"] = normal(*shape), normal(*shape)
    else:
        for x in "kv":
            s[x], s[x + "_scales"] = _quantise(normal(*shape).float())
    if c["op"] == "append":
        s["qkv"] = normal(n_rows, (Hq + 2 * Hkv) * D)
        s["rope"] = _rope_table(D, c["max_len"])
        s["q_out"] = torch.empty(n_rows, Hq, D, dtype=torch.bfloat16, device="cuda")
        if c["format"] != "bf16":
            for x in ("k_out", "v_out"):
                s[x] = torch.empty(n_rows, Hkv, D, dtype=torch.bfloat16, device="cuda")
    else:
        s["q"] = normal(n_rows, Hq, D, scale=2.0)
        s["sinks"] = normal(Hq)
        s["out"] = torch.empty(n_rows, Hq * D, dtype=torch.bfloat16, device="cuda")
    if own:
        import neonengine_amd as ne
        s["kv"] = ne.paged_kv(s["k"], s["v"], s.get("k_scales"), s.get("v_scales"))
        if c["op"] == "attn":
            wb, cb = ne.paged_attn_workspace(n_rows, c["B"], Hq, Hkv, D)
            s["ws"] = torch.empty(max(wb, 1), dtype=torch.uint8, device="cuda")
            s["counters"] = torch.zeros(max(cb, 1), dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------------------
# the operators
# --------------------------------------------------------------------------
def run(s):
    op = s["c"]["op"]
    if own:
        return _own_sample(s) if op == "sample" else _own_append(s) if op == "append" else _own_attn(s)
    return _plain_sample(s) if op == "sample" else _plain_append(s) if op == "append" else _plain_attn(s)


def _own_append(s):
    import neonengine_amd as ne
    c = s["c"]
    # one token a sequence needs no row starts
    start = None if s["most"] == 1 else s["q_start"]
    ne.paged_append(s["kv"], s["qkv"], s["rope"], start, s["kv_len"], s["table"], s["q_out"], c["Hq"])
    if c["format"] == "bf16":
        return s["q_out"], s["k"], s["v"]
    ne.paged_gather(s["kv"], start, s["kv_len"], s["table"], s["k_out"], s["v_out"])
    return s["q_out"], s["k_out"], s["v_out"]


def _own_attn(s):
    import neonengine_amd as ne
    c = s["c"]
    start = None if s["most"] == 1 else s["q_start"]
    ne.paged_attn(s["kv"], s["q"], s["sinks"], start, s["kv_len"], s["table"], s["out"], c["Hq"],
                  window=c["window"], workspace=s["ws"], counters=s["counters"])
    return s["out"]


def _own_sample(s):
    import neonengine_amd as ne
    ne.sample_rows(s["logits"], s["u"], s["out"], temperature=s["temperature"], top_k=s["top_k"],
                   top_p=s["top_p"], min_p=s["min_p"], workspace=s["ws"])
    return s["out"]


def _row_places(s):
    """Sequence and position of every row."""
    start, n = s["q_start"].long(), s["n_rows"]
    row = torch.arange(n, device="cuda")
    b = torch.bucketize(row, start[1:], right=True)
    return b, s["kv_len"].long()[b] - (start[b + 1] - row)


def _plain_append(s):
    c = s["c"]
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    b, p = _row_places(s)
    x = s["qkv"].view(s["n_rows"], Hq + 2 * Hkv, D).float()
    cos, sin = s["rope"][0, p][:, None], s["rope"][1, p][:, None]
    x1, x2 = x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:]
    r = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)
    s["q_out"].copy_(r[:, :Hq])
    k, v = r[:, Hq:], x[:, Hq + Hkv:]
    at = s["table"].long()[b, p // page], slice(None), p % page
    if c["format"] == "bf16":
        s["k"][at], s["v"][at] = k.bfloat16(), v.bfloat16()
        return s["q_out"], s["k"], s["v"]
    (s["k"][at], s["k_scales"][at]), (s["v"][at], s["v_scales"][at]) = _quantise(k), _quantise(v)
    return (s["q_out"], _values(s["k"][at], s["k_scales"][at]).bfloat16(),
            _values(s["v"][at], s["v_scales"][at]).bfloat16())


def _cached(s, x, page, slot):
    """fp32 keys or values [B][Hkv][T][D] at the places of a padded batch."""
    if s["c"]["format"] == "bf16":
        return s[x][page, :, slot].permute(0, 2, 1, 3).float()
    v = _values(s[x][page, :, slot], s[x + "_scales"][page, :, slot])
    return v.permute(0, 2, 1, 3).contiguous()


def _plain_attn(s):
    c = s["c"]
    Hq, Hkv, D, page, B, most = c["Hq"], c["Hkv"], c["D"], c["page"], c["B"], s["most"]
    G = Hq // Hkv
    T = s["table"].shape[1] * page
    t = torch.arange(T, device="cuda")
    pages, slot = s["table"].long().clamp(min=0)[:, t // page], (t % page).expand(B, T)
    k = _cached(s, "k", pages, slot)
    v = _cached(s, "v", pages, slot)
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    i = torch.arange(most, device="cuda")
    n = start[1:] - start[:-1]
    inside = i < n[:, None]
    row = torch.where(inside, start[:-1, None] + i, torch.zeros_like(i))
    p = torch.where(inside, (kv_len - n)[:, None] + i, torch.full_like(i, -1))  # [B][most]
    q = s["q"][row].float().view(B, most, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, most * G, D)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * D ** -0.5
    score = score.view(B, Hkv, most, G, T)
    seen = t <= p[..., None]
    if c["window"] > 0:
        seen = seen & (t > p[..., None] - c["window"])
    score = score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    sink = s["sinks"].float().view(1, Hkv, 1, G, 1)
    top = torch.maximum(score.amax(-1, keepdim=True), sink)
    e = score.sub_(top).exp_()
    e = e / (e.sum(-1, keepdim=True) + (sink - top).exp())
    o = torch.matmul(e.view(B, Hkv, most * G, T), v)
    o = o.view(B, Hkv, most, G, D).permute(0, 2, 1, 3, 4).reshape(B, most, Hq * D)
    s["out"][row[inside]] = o[inside].bfloat16()
    return s["out"]


def _plain_sample(s):
    x, V = s["logits"].double(), s["c"]["V"]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = ((x - x[:, :1]) / s["temperature"].double()[:, None]).exp()
    rank = torch.arange(V, device="cuda")
    k = s["top_k"].long()[:, None]
    w = w * ((k <= 0) | (rank < k))
    before = w.cumsum(-1) - w
    goal = s["top_p"].double()[:, None] * w.sum(-1, keepdim=True)
    w = w * ((before < goal) & (w >= s["min_p"].double()[:, None]))
    kept = torch.zeros_like(w).scatter_(-1, order, w)
    run = kept.cumsum(-1)
    over = run > s["u"].double()[:, None] * run[:, -1:]
    s["out"].copy_(over.to(torch.uint8).argmax(-1))
    return s["out"]


# --------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# --------------------------------------------------------------------------
def work(c):
    if c["op"] == "sample":
        return {"bytes": c["B"] * (4.0 * c["V"] + 24), "flops": 0.0}
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    lens = _lengths(c)
    rows = sum(n for n, _ in lens)
    head = 2 * D if c["format"] == "bf16" else D // 2 + D // 32  # bytes of one cached row
    if c["op"] == "append":
        b = rows * ((Hq + 2 * Hkv) * D * 2 + Hq * D * 2 + 2 * Hkv * head) + min(rows, c["max_len"]) * D * 4
        if c["format"] != "bf16":
            b += rows * 2 * Hkv * (head + 2 * D)  # read back
        return {"bytes": float(b), "flops": 3.0 * rows * (Hq + Hkv) * D}
    keys = pairs = 0
    for n, t in lens:
        w = c["window"] or t
        keys += min(t, n - 1 + w)
        pairs += sum(min(p + 1, w) for p in range(t - n, t))
    return {"bytes": float(rows * Hq * D * 4 + keys * 2 * Hkv * head + keys // c["page"] * 4),
            "flops": 4.0 * D * Hq * pairs}


def _exact_values(s, x, pages, at):
    """float64 cached rows at (page, slot): [n][Hkv][D]."""
    if s["c"]["format"] == "bf16":
        return s[x][pages, :, at].double()
    codes, byte = s[x][pages, :, at].long(), s[x + "_scales"][pages, :, at].double()
    nib = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    mag = nib % 8
    # E2M1: 0, 1/2, then (1 + m/2) 2^(e-1) for exponent field e = 1, 2, 3
    val = torch.where(mag < 2, mag * 0.5, (1 + 0.5 * (mag % 2)) * torch.exp2((mag // 2 - 1).double()))
    val = val * (1 - 2 * (nib // 8))
    return val * torch.exp2(byte - 127).repeat_interleave(32, -1)


def exact(case, seed):
    c = dict(case)
    if c["op"] == "sample":
        return None  # ids: whole numbers
    s = prepare(c, seed)
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    lens = _lengths(c)
    if c["op"] == "append":
        q, kk, vv = [], [], []
        k_pool = v_pool = None
        if c["format"] == "bf16":
            k_pool, v_pool = s["k"].double(), s["v"].double()
        at = 0
        for b, (n, t) in enumerate(lens):
            x = s["qkv"][at:at + n].double().view(n, -1, D)
            at += n
            pos = torch.arange(t - n, t, device="cuda")
            z = torch.complex(s["rope"][0, pos].double(), s["rope"][1, pos].double())[:, None]
            y = torch.complex(x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:]) * z
            y = torch.cat((y.real, y.imag), -1)
            q.append(y[:, :Hq])
            k, v = y[:, Hq:], x[:, Hq + Hkv:]
            pg = s["table"][b].long()[pos // page]
            if c["format"] == "bf16":
                k_pool[pg, :, pos % page], v_pool[pg, :, pos % page] = k, v
            else:
                kk.append(_exact_mx(k))
                vv.append(_exact_mx(v))
        if c["format"] == "bf16":
            return torch.cat(q), k_pool, v_pool
        return torch.cat(q), torch.cat(kk), torch.cat(vv)
    out = torch.zeros_like(s["out"], dtype=torch.float64)
    at = 0
    for b, (n, t) in enumerate(lens):
        lo = 0 if not c["window"] else max(0, t - n - c["window"] + 1)
        key = torch.arange(lo, t, device="cuda")
        pg = s["table"][b].long()[key // page]
        k, v = (_exact_values(s, x, pg, key % page) for x in "kv")
        for r0 in range(0, n, 512):
            m = min(512, n - r0)
            pos = torch.arange(t - n + r0, t - n + r0 + m, device="cuda")
            hidden = key[None] > pos[:, None]
            if c["window"]:
                hidden = hidden | (pos[:, None] - key[None] >= c["window"])
            for h in range(Hq):
                g = h // (Hq // Hkv)
                a = s["q"][at + r0:at + r0 + m, h].double() @ k[:, g].T / math.sqrt(D)
                a[hidden] = -math.inf
                a = torch.cat((a, s["sinks"][h].double().expand(m, 1)), 1)
                out[at + r0:at + r0 + m, h * D:(h + 1) * D] = torch.softmax(a, 1)[:, :-1] @ v[:, g]
        at += n
    return out


def _exact_mx(x):
    """What MXFP4 keeps of x [..., D] (float64)."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300)))
    e = e - 2 + (top > 1.75 * torch.exp2(e))
    e = torch.where(top > 0, e.clamp(min=-127), torch.zeros_like(e))
    y = b / torch.exp2(e)
    # the step of y's binade: 1/2 below 2, 1 below 4, 2 above
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).to(y.dtype)
    return ((torch.round(y / step) * step).clamp(-6, 6) * torch.exp2(e)).reshape(x.shape)

