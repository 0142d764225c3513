"""The operators of beam search over the caches as they are measured: choosing the
next beams from the logits, moving the states of beams in contiguous caches, and
forking, copying and compacting the pages of a paged one.

A step of beam search is one choice and one fork of the page tables for the whole
model, and one copy of the few pages that two beams would both write (or, over
contiguous caches, one move of the states of the beams that ended).  Shapes are those
of the gpt-oss presets (8 KV heads of 64, a vocabulary of 201088, 24 layers) and
generic ones.
"""
import math
import random

import torch

own = False


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _select(name, **k):
    return dict({"op": "select", "name": name, "B": 1, "W": 4, "V": 201088, "stops": 3, "spread": 2.5,
                 "first": False}, **k)


def _reorder(name, **k):
    return dict({"op": "reorder", "name": name, "B": 1, "W": 4, "heads": 8, "T": 2048, "D": 64,
                 "states": 2, "max_len": 300}, **k)


def _fork(name, **k):
    return dict({"op": "fork", "name": name, "kind": "beams", "B": 16, "W": 4, "page": 64,
                 "max_len": 8192, "spare": 256}, **k)


def _copy(name, **k):
    return dict({"op": "copy", "name": name, "layers": 24, "pairs": 20, "page": 64, "heads": 8, "D": 64,
                 "n_pages": 64, "partial": True}, **k)


def _compact(name, **k):
    return dict({"op": "compact", "name": name, "B": 64, "page": 64, "max_len": 2048, "n_pages": 4096}, **k)


def listed():
    """B: requests; W: beams of each."""
    return [
        # one request's next beams: latency counts
        _select("select_one"),
        # a full batch of requests
        _select("select_batch", B=16),
        # wide beams over a smaller vocabulary of odd size
        _select("select_wide", B=8, W=16, V=32003, stops=1, spread=1.5),
        # the first step of many requests: one beam of each is alive
        _select("select_first", B=64, W=5, V=32003, stops=2, first=True),
        # one request's beams in the contiguous cache of a layer
        _reorder("reorder_one"),
        # a batch's, two layers with one call
        _reorder("reorder_batch", B=8, states=4, max_len=2000),
        # a decode step of a batch of requests with 4 beams each
        _fork("fork_step"),
        # a large server: many requests on small pages
        _fork("fork_server", B=256, page=16, max_len=4096, spare=40000),
        # the pages that two beams would both write, in every layer
        _copy("copy_tails"),
        # whole pages, as a compaction or a copy of a prefix moves them
        _copy("copy_whole", layers=2, pairs=600, page=128, D=128, n_pages=1300, partial=False),
        # a small pool
        _compact("compact_small"),
        # the pool of a whole card
        _compact("compact_card", B=512, page=16, max_len=4000, n_pages=131072),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(("select", "select", "reorder", "fork", "copy", "compact"))
    if op == "select":
        W = rng.choice((1, 2, 3, 4, 5, 8, 16, 32))
        return {"op": op, "B": log(1, max(2, 100 // W)), "W": W, "V": log(700, 201088),
                "stops": rng.randint(0, 4), "spread": round(rng.uniform(1.0, 3.5), 2),
                "first": rng.random() < 0.2}
    if op == "reorder":
        T = log(64, 4096)
        return {"op": op, "B": log(1, 8), "W": rng.randint(2, 8), "heads": rng.choice((1, 2, 4, 8)), "T": T,
                "D": rng.choice((64, 64, 128)), "states": rng.choice((1, 2, 4)), "max_len": log(16, T)}
    if op == "fork":
        page = rng.choice((16, 32, 64, 128))
        return {"op": op, "kind": rng.choice(("beams", "beams", "samples", "drafts")), "B": log(1, 200),
                "W": rng.randint(2, 8), "page": page, "max_len": log(page, 8192), "spare": log(64, 40000)}
    if op == "copy":
        pairs = log(1, 200)
        return {"op": op, "layers": log(1, 24), "pairs": pairs, "page": rng.choice((16, 32, 64)),
                "heads": rng.choice((1, 2, 4, 8)), "D": rng.choice((64, 128)),
                "n_pages": 2 * pairs + rng.randint(1, 64), "partial": rng.random() < 0.5}
    return {"op": op, "B": log(1, 500), "page": rng.choice((16, 32, 64, 128)), "max_len": log(64, 4000),
            "n_pages": log(100, 131072)}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _parents(B, W):
    """Parent place of each place: a beam that goes on keeps its place, the others
    go to children of those that do.  Every case has its own, fixed ones."""
    r = random.Random("%d %d" % (B, W))
    out = []
    for b in range(B):
        live = [w for w in range(W) if r.random() < 0.65] or [r.randrange(W)]
        if W > 1 and len(live) == W:
            live.remove(r.randrange(W))
        out += [b * W + (w if w in live else r.choice(live)) for w in range(W)]
    return out


def _lengths(c):
    """A token count for each of c["B"] requests: the first has max_len, the others
    are spread over a factor of 16 below; every case has its own, fixed ones."""
    r = random.Random("%d %d" % (c["B"], c["max_len"]))
    top = c["max_len"]
    lo = max(1, top // 16)
    return [top] + [int(round(math.exp(r.uniform(math.log(lo), math.log(top))))) for _ in range(c["B"] - 1)]


def _dev(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _cache(c, W, limit):
    """(page table, lengths, shared whole pages of each request, pages): requests of
    W sequences that share the whole pages of their prompt."""
    page = c["page"]
    rows, lens, shared, at = [], [], [], 0
    for n in _lengths(c):
        prompt = n * 3 // 4 // page if W > 1 else 0
        own_pages = -(-n // page) - prompt
        if at + prompt + W * own_pages > limit:  # the pool is full
            n = prompt = own_pages = 0
        for w in range(W):
            rows.append((at, prompt, at + prompt + w * own_pages, own_pages))
            lens.append(n)
        shared.append(prompt)
        at += prompt + W * own_pages
    return rows, lens, shared, at


def _table(rows, width, ids):
    """Page table [len(rows)][width], -1 where a sequence has no page."""
    i = torch.arange(width)
    r = torch.tensor(rows)
    place = torch.where(i < r[:, 1:2], r[:, :1] + i, r[:, 2:3] + i - r[:, 1:2])
    has = i < r[:, 1:2] + r[:, 3:4]
    return torch.where(has, ids[place.clamp(0, max(0, len(ids) - 1))], torch.tensor(-1)).to(torch.int32)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = random.Random(seed)
    host = torch.Generator()
    host.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    def ints(*shape, fill=-1):
        return torch.full(shape, fill, dtype=torch.int32, device="cuda")

    s = {"c": c}
    op = c["op"]
    if own:
        import neonengine_amd as ne
    if op == "select":
        B, W, V = c["B"], c["W"], c["V"]
        N = B * W
        l = normal(N, V, scale=c["spread"], dtype=torch.float32)
        l[:, 7::50] = -math.inf  # tokens that a grammar forbids
        ids = r.sample(range(V), c["stops"])
        for t in ids:  # in a third of the beams a sentence may end here
            near = torch.rand(N, generator=g, device="cuda") < 0.33
            l[:, t] = torch.where(near, l.amax(-1) - 0.3 * torch.rand(N, generator=g, device="cuda"), l[:, t])
        score = -12.0 - 2.0 * torch.rand((B, W), generator=g, device="cuda")
        if c["first"]:
            score[:, 0] = 0.0
            score[:, 1:] = -math.inf
        s.update(logits=l, score=score.view(N), stop=_dev(ids) if ids else None,
                 token=ints(N), parent=ints(N), out=torch.empty(N, device="cuda"),
                 ended=(ints(N), ints(N), torch.empty(N, device="cuda")))
        if own:
            n = ne.beam_select_workspace(B, W, V, c["stops"])
            s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        return s
    if op == "reorder":
        N = c["B"] * c["W"]
        s["x"] = [normal(N, c["heads"], c["T"], c["D"]) for _ in range(c["states"])]
        s["parent"] = _dev(_parents(c["B"], c["W"]))
        s["len"] = _dev([n for n in _lengths(c) for _ in range(c["W"])])
        if own:
            s["states"] = ne.beam_states(s["x"], c["W"])
        return s
    if op == "fork":
        W = 1 if c["kind"] == "drafts" else c["W"]
        rows, lens, shared, used = _cache(c, W, 1 << 30)
        if c["kind"] == "samples":  # W continuations of each prompt
            rows, lens = rows[::W], lens[::W]
        add = max(1, 8 // c["page"]) + 1
        n_pages = used + c["spare"] + c["B"] * c["W"] * add
        width = -(-(c["max_len"] + 9) // c["page"])
        perm = torch.randperm(n_pages, generator=host)
        table = _table(rows, width, perm[:used])
        refs = torch.bincount(table[table >= 0].long(), minlength=n_pages)
        if c["kind"] == "beams":  # a prefix cache holds some prompts as well
            for q in range(0, len(rows), 4 * W):
                at, prompt, _, _ = rows[q]
                refs[perm[at:at + prompt]] += 1
        s.update(refs=refs.to(torch.int32).cuda(), table=table.cuda(), len=_dev(lens), n_pages=n_pages,
                 parent=None, keep=None, add=None)
        N = len(rows)
        if c["kind"] == "beams":
            s["parent"] = _dev(_parents(c["B"], W))
        elif c["kind"] == "samples":
            N = c["B"] * W
            s["parent"] = _dev([b // W for b in range(N)])
        else:  # some drafted tokens are dropped, others take their place
            s["keep"] = _dev([max(0, n - r.randint(0, 8)) for n in lens])
            s["add"] = _dev([r.randint(1, 9) for _ in lens])
        s.update(refs_out=ints(n_pages, fill=0), table_out=ints(N, width), len_out=ints(N),
                 copies=(ints(N), ints(N), ints(N)))
        if own:
            wb, cb = ne.pages_workspace(n_pages, N)
            s["ws"] = torch.empty(max(wb, 1), dtype=torch.uint8, device="cuda")
            s["counters"] = torch.zeros(max(cb, 1), dtype=torch.uint8, device="cuda")
        return s
    if op == "copy":
        shape = (c["n_pages"], c["heads"], c["page"], c["D"])
        s["pools"] = [(normal(*shape), normal(*shape)) for _ in range(c["layers"])]
        perm = torch.randperm(c["n_pages"], generator=host).to(torch.int32)
        n = c["pairs"]
        # a fork's list: one entry a sequence, most of them empty
        at = torch.arange(n) * (3 if c["partial"] else 1)
        src, dst, cnt = (torch.full((int(at[-1]) + 1,), v, dtype=torch.int32) for v in (-1, -1, 0))
        src[at], dst[at] = perm[:n], perm[n:2 * n]
        if c["partial"]:
            cnt[at] = torch.tensor(_tails(c), dtype=torch.int32)
        s.update(src=src.cuda(), dst=dst.cuda(), rows=cnt.cuda() if c["partial"] else None)
        if own:
            s["layers"] = ne.paged_layers([ne.paged_kv(k, v) for k, v in s["pools"]])
        return s
    rows, lens, _, used = _cache(c, 1, c["n_pages"])
    perm = torch.randperm(c["n_pages"], generator=host)
    width = -(-c["max_len"] // c["page"])
    table = _table(rows, width, perm[:used])
    refs = torch.bincount(table[table >= 0].long(), minlength=c["n_pages"])
    held = perm[used:used + (c["n_pages"] - used) // 8]  # pages of a prefix cache
    refs[held] += 1
    n = c["n_pages"]
    s.update(refs=refs.to(torch.int32).cuda(), table=table.cuda(), len=_dev(lens), refs_out=ints(n),
             table_out=ints(c["B"], width), map=ints(n), copies=(ints(n // 2), ints(n // 2)))
    if own:
        wb, _ = ne.pages_workspace(n, c["B"])
        s["ws"] = torch.empty(max(wb, 1), dtype=torch.uint8, device="cuda")
    return s


def _tails(c):
    """Rows in use of the partial pages of a copy."""
    r = random.Random(c["pairs"])
    return [r.randint(1, c["page"] - 1) for _ in range(c["pairs"])]


# --------------------------------------------------------------------------
# the operators
# --------------------------------------------------------------------------
def run(s):
    op = s["c"]["op"]
    if own:
        return {"select": _own_select, "reorder": _own_reorder, "fork": _own_fork, "copy": _own_copy,
                "compact": _own_compact}[op](s)
    return {"select": _plain_select, "reorder": _plain_reorder, "fork": _plain_fork, "copy": _plain_copy,
            "compact": _plain_compact}[op](s)


def _own_select(s):
    import neonengine_amd as ne
    ne.beam_select(s["logits"], s["score"], s["c"]["W"], s["token"], s["parent"], s["out"], stop=s["stop"],
                   ended=s["ended"], workspace=s["ws"])
    return (s["token"], s["parent"], s["out"], *s["ended"])


def _own_reorder(s):
    import neonengine_amd as ne
    ne.beam_reorder(s["states"], s["parent"], s["len"])
    return s["x"]


def _own_fork(s):
    import neonengine_amd as ne
    ne.pages_fork(s["refs"], s["table"], s["len"], s["c"]["page"], s["refs_out"], s["table_out"], s["len_out"],
                  s["copies"], parent=s["parent"], keep=s["keep"], add=s["add"], workspace=s["ws"],
                  counters=s["counters"])
    return (s["refs_out"], s["table_out"], s["len_out"], *s["copies"])


def _own_copy(s):
    import neonengine_amd as ne
    ne.pages_copy(s["layers"], s["src"], s["dst"], s["rows"])
    return s["pools"]


def _own_compact(s):
    import neonengine_amd as ne
    ne.pages_compact(s["refs"], s["table"], s["len"], s["c"]["page"], s["refs_out"], s["table_out"], s["map"],
                     s["copies"], workspace=s["ws"])
    return (s["refs_out"], s["table_out"], s["map"], *s["copies"])


def _plain_select(s):
    c = s["c"]
    B, W, V, K = c["B"], c["W"], c["V"], c["stops"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    v = (s["score"].double()[:, None] + (x - lse)).view(B, W * V)
    is_stop = torch.zeros(V, dtype=torch.bool, device="cuda")
    if K:
        is_stop[s["stop"].long()] = True
    # the W best of those that go on lie among the first W (1 + K) of all
    v, at = torch.sort(v, dim=-1, descending=True, stable=True)
    n = min(W * (1 + K), W * V)
    v, at = v[:, :n], at[:, :n]
    token, beam = at % V, at // V
    stop = is_stop[token]
    none = v == -math.inf
    # ended: stop tokens of rank < W, in order
    e = stop & ~none & (torch.arange(n, device="cuda") < W)
    rank = torch.where(e, e.cumsum(-1) - 1, W)
    first = torch.arange(0, B * W, W, device="cuda")[:, None]

    def put(place, value, fill):
        o = torch.full((B, W + 1), fill, dtype=value.dtype, device="cuda")
        return o.scatter_(-1, place, value)[:, :W].reshape(B * W)

    neg = torch.full_like(at, -1)
    live_id = torch.where(none, neg, token), torch.where(none, neg, beam + first)
    s["ended"][0].copy_(put(rank, live_id[0], -1))
    s["ended"][1].copy_(put(rank, live_id[1], -1))
    s["ended"][2].copy_(put(rank, v, -math.inf))
    # live: the first W that are no stop tokens; a beam's best child takes its place
    order = (~stop).cumsum(-1) - 1
    j = torch.where(stop | (order >= W), W, order)
    slot = torch.full((B, W + 1), -1, dtype=torch.int64, device="cuda")
    slot.scatter_(-1, j, torch.arange(n, device="cuda").expand(B, n))
    slot = slot[:, :W]
    gone = (slot < 0) | none.gather(-1, slot.clamp(min=0))
    lb = torch.where(gone, torch.full_like(slot, -1), beam.gather(-1, slot.clamp(min=0)))
    same = (lb[:, :, None] == lb[:, None, :]) & torch.ones(W, W, device="cuda").tril(-1).bool()
    keeper = ~same.any(-1) & ~gone
    taken = torch.zeros(B, W + 1, dtype=torch.bool, device="cuda")
    taken.scatter_(-1, torch.where(keeper, lb, W), True)
    free = torch.sort(taken[:, :W].to(torch.uint8), dim=-1, stable=True)[1]
    place = torch.where(keeper, lb, free.gather(-1, ((~keeper).cumsum(-1) - 1).clamp(min=0)))
    pick = slot.clamp(min=0)
    s["token"].copy_(put(place, torch.where(gone, -1, live_id[0].gather(-1, pick)), -1))
    s["parent"].copy_(put(place, torch.where(gone, -1, live_id[1].gather(-1, pick)), -1))
    s["out"].copy_(put(place, torch.where(gone, -math.inf, v.gather(-1, pick)), -math.inf))
    return (s["token"], s["parent"], s["out"], *s["ended"])


def _plain_reorder(s):
    p = s["parent"].long()
    N = p.numel()
    t = torch.arange(s["c"]["T"], device="cuda")
    moved = (p != torch.arange(N, device="cuda"))[:, None] & (t < s["len"].long()[p][:, None])
    for x in s["x"]:
        x.copy_(torch.where(moved[:, None, :, None], x[p], x))
    return s["x"]


def _plain_fork(s):
    c, page, n_pages = s["c"], s["c"]["page"], s["n_pages"]
    table, length = s["table"].long(), s["len"].long()
    N, width = s["table_out"].shape
    parent = torch.arange(N, device="cuda") if s["parent"] is None else s["parent"].long()
    keep = length[parent] if s["keep"] is None else s["keep"].long()
    add = (length[parent] > 0).long() if s["add"] is None else s["add"].long()
    i = torch.arange(width, device="cuda")
    held, kept, goal = (-(-n // page) for n in (length, keep, keep + add))
    rows = table[parent]
    refs = s["refs"].long()
    refs = refs - torch.bincount(table[i < held[:, None]], minlength=n_pages)
    refs = refs + torch.bincount(rows[i < kept[:, None]], minlength=n_pages)
    # the page that a sequence goes on writing, and who else does
    writes = (keep % page != 0) & (add > 0)
    last = rows.gather(-1, (kept - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    writers = torch.bincount(last[writes], minlength=n_pages)
    first = torch.full((n_pages,), N, device="cuda")
    b = torch.arange(N, device="cuda")
    first = first.scatter_reduce(0, torch.where(writes, last, 0), torch.where(writes, b, N), "amin")
    stays = (refs[last] == 1) | ((refs[last] == writers[last]) & (first[last] == b))
    copied = writes & ~stays
    need = goal - kept + copied.long()
    before = need.cumsum(0) - need
    free = (refs == 0).nonzero()[:, 0]
    total = int(need.sum())
    refs[free[:total]] = 1
    refs = refs - torch.bincount(last[copied], minlength=n_pages)
    old_end = kept - copied.long()
    new = before[:, None] + i - old_end[:, None]
    new = torch.cat((free, free.new_full((1,), -1)))[new.clamp(0, free.numel())]
    out = torch.where(i < old_end[:, None], rows, torch.where(i < goal[:, None], new, s["table_out"].long()))
    s["refs_out"].copy_(refs)
    s["table_out"].copy_(out)
    s["len_out"].copy_(keep + add)
    minus = torch.full_like(last, -1)
    s["copies"][0].copy_(torch.where(copied, last, minus))
    s["copies"][1].copy_(torch.where(copied, out.gather(-1, old_end.clamp(max=width - 1)[:, None])[:, 0], minus))
    s["copies"][2].copy_(torch.where(copied, keep % page, torch.zeros_like(keep)))
    return (s["refs_out"], s["table_out"], s["len_out"], *s["copies"])


def _plain_copy(s):
    has = s["src"] >= 0
    src, dst = s["src"][has].long(), s["dst"][has].long()
    if s["rows"] is None:
        for pools in s["pools"]:
            for x in pools:
                x[dst] = x[src]
        return s["pools"]
    inside = torch.arange(s["c"]["page"], device="cuda") < s["rows"][has].long()[:, None]
    for pools in s["pools"]:
        for x in pools:
            x[dst] = torch.where(inside[:, None, :, None], x[src], x[dst])
    return s["pools"]


def _plain_compact(s):
    refs = s["refs"].long()
    n = refs.numel()
    at = torch.arange(n, device="cuda")
    used = refs != 0
    U = used.sum()
    src, dst = (used & (at >= U)).nonzero()[:, 0], (~used & (at < U)).nonzero()[:, 0]
    to = torch.where(used, at, torch.full_like(at, -1))
    to[src] = dst
    out = torch.zeros_like(refs)
    out[to[used]] = refs[used]
    held = -(-s["len"].long() // s["c"]["page"])
    i = torch.arange(s["table"].shape[1], device="cuda")
    moved = to[s["table"].long().clamp(min=0)]
    s["refs_out"].copy_(out)
    s["map"].copy_(to)
    s["table_out"].copy_(torch.where(i < held[:, None], moved, s["table_out"].long()))
    for x, v in zip(s["copies"], (src, dst)):
        x.fill_(-1)
        x[:v.numel()] = v.to(torch.int32)
    return (s["refs_out"], s["table_out"], s["map"], *s["copies"])


# --------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# --------------------------------------------------------------------------
def work(c):
    op = c["op"]
    if op == "select":
        N = c["B"] * c["W"]
        live = c["B"] if c["first"] else N
        return {"bytes": live * 4.0 * c["V"] + N * 28.0, "flops": 0.0}
    if op == "reorder":
        lens = _lengths(c)
        rows = sum(lens[b // c["W"]] for b, p in enumerate(_parents(c["B"], c["W"])) if p != b)
        return {"bytes": 2.0 * rows * c["heads"] * c["D"] * 2 * c["states"], "flops": 0.0}
    if op == "fork":
        W = 1 if c["kind"] == "drafts" else c["W"]
        rows, _, _, used = _cache(c, W, 1 << 30)
        entries = sum(p + q for _, p, _, q in rows)
        read = entries // W if c["kind"] == "samples" else entries
        n_pages = used + c["spare"] + c["B"] * c["W"] * (max(1, 8 // c["page"]) + 1)
        return {"bytes": 8.0 * n_pages + 4.0 * (entries + read) + 32.0 * len(rows), "flops": 0.0}
    if op == "copy":
        rows = sum(_tails(c)) if c["partial"] else c["pairs"] * c["page"]
        return {"bytes": 2.0 * rows * c["heads"] * c["D"] * 2 * 2 * c["layers"], "flops": 0.0}
    rows, _, _, _ = _cache(c, 1, c["n_pages"])
    return {"bytes": 16.0 * c["n_pages"] + 8.0 * sum(q for _, _, _, q in rows) + 4.0 * len(rows), "flops": 0.0}


def exact(case, seed):
    """The scores of a choice; everything else is whole numbers and moved values."""
    c = dict(case)
    if c["op"] != "select":
        return None
    s = prepare(c, seed)
    B, W = c["B"], c["W"]
    stop = set(s["stop"].tolist()) if c["stops"] else set()
    live, over = [], []
    for b in range(B):
        cand = []
        for w in range(W):
            start = s["score"][b * W + w].double()
            if start == -math.inf:
                continue
            logp = torch.log_softmax(s["logits"][b * W + w].double(), -1) + start
            v, t = torch.topk(logp, min(W + len(stop), c["V"]))
            cand += [(-x, w, i) for x, i in zip(v.tolist(), t.tolist()) if x > -math.inf]
        cand.sort()
        over.append([-x for x, _, t in cand[:W] if t in stop])
        place = [None] * W
        rest = []
        for x, w, t in [q for q in cand if q[2] not in stop][:W]:
            if place[w] is None:
                place[w] = -x
            else:
                rest.append(-x)
        live.append([rest.pop(0) if p is None and rest else p for p in place])

    def whole(lists):
        flat = [(list(q) + [None] * W)[:W] for q in lists]
        return torch.tensor([[-math.inf if x is None else x for x in q] for q in flat], dtype=torch.float64,
                            device="cuda").view(-1)

    return None, None, whole(live), None, None, whole(over)
