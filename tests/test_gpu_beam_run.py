"""Beam search as a program runs it: choice, fork of the page tables, copies of the
pages that two beams would both write, append and attention over the pages, eager and
captured; the same over contiguous caches with their states moved in place.

Keys and values of a token depend on the token and the layer alone, so what the
caches hold is known from each beam's tokens, bit for bit."""
import sys

import numpy as np
import pytest

import neonengine_amd as ne
from tests import beam_util
from tests.gpu_util import to_dev, to_host, torch_cuda

pytestmark = pytest.mark.gpu

Hq, Hkv, D, LAYERS, PAGE = 4, 2, 64, 2, 16
V = Hq * D  # a token's logit is one element of the attention's output


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


class Search:
    """B requests of W beams over one pool of pages."""

    def __init__(self, prompts, W, n_pages, max_pages, stop, seed=0):
        torch = torch_cuda()
        rng = np.random.default_rng(seed)
        B = len(prompts)
        self.B, self.W, self.N, self.stop = B, W, B * W, to_dev(np.array(stop, np.int32))
        # token -> q, k and v heads of each layer
        self.rows = torch.from_numpy(rng.normal(0, 1.5, (LAYERS, V, (Hq + 2 * Hkv) * D)).astype(np.float32)) \
            .bfloat16().cuda()
        self.pools = [tuple(torch.full((n_pages, Hkv, PAGE, D), float("nan"), device="cuda").bfloat16()
                            for _ in "kv") for _ in range(LAYERS)]
        self.caches = [ne.paged_kv(k, v) for k, v in self.pools]
        self.layers = ne.paged_layers(self.caches)
        i = lambda *s: torch.full(s, -1, dtype=torch.int32, device="cuda")
        f = lambda *s: torch.zeros(s, dtype=torch.float32, device="cuda")
        N = self.N
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        self.tables = [i(N, max_pages), i(N, max_pages)]
        self.length = torch.zeros(N, dtype=torch.int32, device="cuda")
        self.token, self.parent, self.score = i(N), i(N), f(N)
        self.ended = (i(N), i(N), f(N))
        self.copies = (i(N), i(N), i(N))
        self.out = torch.zeros(LAYERS, N, Hq * D, device="cuda").bfloat16()
        self.logits = f(N, V)
        ws = lambda n: torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
        self.sel_ws = ws(ne.beam_select_workspace(B, W, V, len(stop)))
        wb, cb = ne.pages_workspace(n_pages, N)
        self.plan_ws, self.plan_counters = ws(wb), torch.zeros(cb, dtype=torch.uint8, device="cuda")
        wb, cb = ne.paged_attn_workspace(N, N, Hq, Hkv, D)
        self.attn_ws, self.attn_counters = ws(wb), torch.zeros(max(1, cb), dtype=torch.uint8, device="cuda")
        self.prefill(prompts)

    def prefill(self, prompts):
        torch = torch_cuda()
        B, n = self.B, [len(p) for p in prompts]
        empty = torch.zeros(B, dtype=torch.int32, device="cuda")
        table = torch.full((B, self.tables[0].shape[1]), -1, dtype=torch.int32, device="cuda")
        none = torch.full((B,), -1, dtype=torch.int32, device="cuda")
        copies = tuple(torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(3))
        length = torch.zeros(B, dtype=torch.int32, device="cuda")
        # the prompts are sequences of no past
        ne.pages_fork(self.refs, torch.full_like(table, -5), empty, PAGE, self.refs, table, length, copies,
                      parent=none, add=to_dev(np.array(n, np.int32)))
        assert to_host(length).tolist() == n
        start = to_dev(np.cumsum([0] + n).astype(np.int32))
        ids = torch.from_numpy(np.concatenate(prompts)).cuda()
        last = to_dev((np.cumsum(n) - 1).astype(np.int64))
        q = torch.empty(sum(n), Hq, D, device="cuda").bfloat16()
        total = torch.zeros(B, V, device="cuda")
        for l, kv in enumerate(self.caches):
            ne.paged_append(kv, self.rows[l][ids], None, start, length, table, q, Hq)
            o = torch.empty(sum(n), Hq * D, device="cuda").bfloat16()
            ne.paged_attn(kv, q, None, start, length, table, o, Hq)
            total += o[last].float()
        # one beam of each request is alive; its children start from the prompt's row
        self.logits.copy_((3.0 * total).repeat_interleave(self.W, 0))
        self.score.view(self.B, self.W)[:, 0] = 0.0
        self.score.view(self.B, self.W)[:, 1:] = -float("inf")
        self.prompt = (table, length)

    def choose(self):
        ne.beam_select(self.logits, self.score, self.W, self.token, self.parent, self.score, stop=self.stop,
                       ended=self.ended, workspace=self.sel_ws)

    def advance(self, first=False):
        """The chosen tokens join their beams; logits of the next step."""
        torch = torch_cuda()
        a, b = self.tables
        if first:
            table, length = self.prompt
            parent = torch.where(self.parent >= 0, self.parent // self.W, self.parent).to(torch.int32)
            ne.pages_fork(self.refs, table, length, PAGE, self.refs, a, self.length, self.copies,
                          parent=parent, workspace=self.plan_ws, counters=self.plan_counters)
        else:
            ne.pages_fork(self.refs, a, self.length, PAGE, self.refs, b, self.length, self.copies,
                          parent=self.parent, workspace=self.plan_ws, counters=self.plan_counters)
            self.tables = [b, a]
        ne.pages_copy(self.layers, *self.copies)
        ids = self.token.clamp(min=0).long()
        for l, kv in enumerate(self.caches):
            q = torch.empty(self.N, Hq, D, device="cuda").bfloat16()
            ne.paged_append(kv, self.rows[l][ids], None, None, self.length, self.tables[0], q, Hq)
            ne.paged_attn(kv, q, None, None, self.length, self.tables[0], self.out[l], Hq,
                          workspace=self.attn_ws, counters=self.attn_counters)
        self.logits.copy_((self.out[0].float() + self.out[1].float()) * 3.0)


def attend(rows, ids):
    """The last token's attention over a layer in 64 bits, [Hq D]."""
    x = rows[ids].astype(np.float64).reshape(len(ids), Hq + 2 * Hkv, D)
    out = []
    for h in range(Hq):
        g = h // (Hq // Hkv)
        s = x[:, Hq + g] @ x[-1, h] / np.sqrt(D)
        p = np.exp(s - s.max())
        out.append(p @ x[:, Hq + Hkv + g] / p.sum())
    return np.concatenate(out)


def check_caches(s, beams, others=()):
    """What the pages hold against the beams' tokens, and the counts against the
    tables."""
    torch = torch_cuda()
    length, table = to_host(s.length), to_host(s.tables[0])
    refs = np.zeros(len(s.refs), np.int64)
    n = [len(t) if t else 0 for t in beams]
    assert length.tolist() == n
    for b, t in enumerate(beams):
        np.add.at(refs, table[b, :beam_util.pages(n[b], PAGE)], 1)
    for row, k in others:
        np.add.at(refs, row[:beam_util.pages(k, PAGE)], 1)
    assert np.array_equal(to_host(s.refs), refs)
    start = to_dev(np.cumsum([0] + n).astype(np.int32))
    ids = torch.from_numpy(np.concatenate([t for t in beams if t])).cuda()
    for l, kv in enumerate(s.caches):
        k, v = (torch.empty(sum(n), Hkv, D, device="cuda").bfloat16() for _ in "kv")
        ne.paged_gather(kv, start, s.length, s.tables[0], k, v)
        want = s.rows[l][ids].view(-1, Hq + 2 * Hkv, D)
        assert torch.equal(k, want[:, Hq:Hq + Hkv]) and torch.equal(v, want[:, Hq + Hkv:])


@pytest.mark.parametrize("lens,W,steps", [((1,), 1, 20), ((5, 37, 64), 4, 40), ((16, 100), 3, 35),
                                          ((33, 1, 15, 48, 17), 8, 25)])
def test_search_over_pages(lens, W, steps):
    rng = np.random.default_rng(sum(lens) + W)
    prompts = [rng.integers(0, V, n) for n in lens]
    stop = [int(rng.integers(0, V)), int(rng.integers(0, V))]
    width = (max(lens) + steps) // PAGE + 2
    s = Search(prompts, W, len(lens) * (1 + W) * (width + 1), width, stop, seed=W)
    N = s.N
    say(f"search prompts={lens} W={W}")
    beams = [None] * N
    score = to_host(s.score).copy()
    held = [list(map(int, p)) for p in prompts]
    for step in range(steps):
        want = beam_util.select(to_host(s.logits), score, W, stop)
        s.choose()
        token, parent, got = to_host(s.token), to_host(s.parent), to_host(s.score)
        assert np.array_equal(token, want[0]) and np.array_equal(parent, want[1])
        for x, y in zip((to_host(t) for t in s.ended[:2]), want[3:5]):
            assert np.array_equal(x, y)
        score = got.copy()
        s.advance(first=step == 0)
        old = [held[b // W] for b in range(N)] if step == 0 else beams
        beams = [list(old[p]) + [int(t)] if p >= 0 else None for t, p in zip(token, parent)]
        if step in (0, 1, steps // 2, steps - 1):
            prompt = [(to_host(s.prompt[0])[b], lens[b]) for b in range(len(lens))]
            # the prompts' own rows were given up by the first fork
            check_caches(s, beams)
            for l in range(LAYERS):
                rows, out = s.rows[l].float().cpu().numpy(), s.out[l].float().cpu().numpy()
                for b in range(N):
                    if beams[b]:
                        # bf16 output: half a step; weights 2^-16 each: of values up to 7
                        ref = attend(rows, beams[b])
                        assert (np.abs(out[b] - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -14 * 8).all()
    ne.device_check()


def test_search_captured():
    """Two steps (from one table into the other and back) in a graph, replayed with
    eager work in between, against the same steps run eagerly."""
    torch = torch_cuda()
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, V, n) for n in (20, 47, 3)]
    make = lambda: Search(prompts, 4, 400, 10, [7, 9], seed=5)
    a, b = make(), make()
    for s in (a, b):
        for step in range(2):
            s.choose()
            s.advance(first=step == 0)
    torch.cuda.synchronize()

    def two(s):
        for _ in range(2):
            s.choose()
            s.advance()

    # (a captured pass does not run: a's state is as it was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two(a)
    for replay in range(6):
        say("replay", replay)
        graph.replay()
        two(b)
        torch.cuda.synchronize()
        for name in ("token", "parent", "score", "refs", "length", "logits"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
        n = beam_util.pages(int(b.length.max()), PAGE)
        live = (b.length > 0).nonzero()[:, 0]
        x, y = a.tables[0][live], b.tables[0][live]
        held = torch.arange(n, device="cuda") < ((b.length[live] + PAGE - 1) // PAGE)[:, None]
        assert torch.equal(torch.where(held, x[:, :n], 0), torch.where(held, y[:, :n], 0))
    ne.device_check()


def test_search_on_another_stream():
    torch = torch_cuda()
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, V, n) for n in (20, 47)]
    one, two = (Search(prompts, 3, 300, 10, [7], seed=6) for _ in range(2))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy = torch.zeros(64 << 20, device="cuda")
    for s, stream in ((one, torch.cuda.current_stream()), (two, side)):
        with torch.cuda.stream(stream):
            for step in range(8):
                s.choose()
                s.advance(first=step == 0)
            busy.add_(1.0)
    torch.cuda.synchronize()
    assert torch.equal(one.token, two.token) and torch.equal(one.refs, two.refs)
    # the stream as an argument, with scratch of the call's own
    out = [torch.empty_like(x) for x in (one.token, one.parent, one.score)]
    score = one.score.clone()
    side.wait_stream(torch.cuda.current_stream())
    ne.beam_select(one.logits, score, 3, *out, stream=side)
    side.synchronize()
    want = beam_util.select(to_host(one.logits), to_host(score), 3)
    assert np.array_equal(to_host(out[0]), want[0]) and np.array_equal(to_host(out[1]), want[1])
    refs, length = one.refs.clone(), one.length.clone()
    table = one.tables[0].clone()
    copies = tuple(torch.empty_like(length) for _ in range(3))
    torch.cuda.synchronize()
    ne.pages_fork(refs, table, length, PAGE, refs, table, length, copies, stream=side)
    side.synchronize()
    assert torch.equal(length, torch.where(one.length > 0, one.length + 1, 0).to(torch.int32))


def test_compaction_in_a_run():
    """Sequences leave, the pool is compacted, and the rest decode as before."""
    torch = torch_cuda()
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, V, n) for n in (60, 5, 90, 33)]
    s = Search(prompts, 4, 600, 12, [3], seed=9)
    beams = [None] * s.N
    for step in range(20):
        s.choose()
        token, parent = to_host(s.token), to_host(s.parent)
        old = [list(map(int, prompts[b // 4])) for b in range(s.N)] if step == 0 else beams
        beams = [list(old[p]) + [int(t)] if p >= 0 else None for t, p in zip(token, parent)]
        s.advance(first=step == 0)
    # requests 0 and 2 leave: places without a sequence
    keep = torch.arange(s.N, dtype=torch.int32, device="cuda")
    keep = torch.where((keep // 4) % 2 == 1, keep, -torch.ones_like(keep))
    a, b = s.tables
    ne.pages_fork(s.refs, a, s.length, PAGE, s.refs, b, s.length, s.copies, parent=keep,
                  add=torch.zeros_like(keep))
    s.tables = [b, a]
    beams = [t if (i // 4) % 2 == 1 else None for i, t in enumerate(beams)]
    used = int((s.refs > 0).sum())
    moves = tuple(torch.empty(300, dtype=torch.int32, device="cuda") for _ in range(2))
    moved_to = torch.empty(600, dtype=torch.int32, device="cuda")
    ne.pages_compact(s.refs, s.tables[0], s.length, PAGE, s.refs, s.tables[0], moved_to, moves)
    ne.pages_copy(s.layers, *moves)
    assert int((s.refs[:used] > 0).sum()) == used and int(s.refs[used:].abs().sum()) == 0
    check_caches(s, beams)
    ne.device_check()


@pytest.mark.parametrize("W,T", [(2, 40), (5, 70)])
def test_states_in_contiguous_caches(W, T):
    """Keys and values of neon_attn_decode's caches and the token histories follow the
    beams, whatever the parents are."""
    torch = torch_cuda()
    rng = np.random.default_rng(W)
    B, N = 2, 2 * W
    rows = torch.from_numpy(rng.normal(0, 1, (V, 2, Hkv, D)).astype(np.float32)).bfloat16().cuda()
    cache = [torch.zeros(N, Hkv, T, D, device="cuda").bfloat16() for _ in "kv"]
    history = torch.zeros(N, T, dtype=torch.int32, device="cuda")
    states, tokens = ne.beam_states(cache, W), ne.beam_states([history], W)
    beams = [[] for _ in range(N)]
    for step in range(T):
        length = torch.full((N,), step, dtype=torch.int32, device="cuda")
        parent = np.concatenate([b * W + rng.integers(0, W, W) for b in range(B)])
        if step % 3 == 0:  # a permutation
            parent = np.concatenate([b * W + rng.permutation(W) for b in range(B)])
        new = rng.integers(0, V, N)
        p = to_dev(parent.astype(np.int32))
        ne.beam_reorder(states, p, length)
        ne.beam_reorder(tokens, p, length)
        beams = [list(beams[q]) + [int(t)] for q, t in zip(parent, new)]
        ids = torch.from_numpy(new).cuda()
        for i in (0, 1):
            cache[i][:, :, step] = rows[ids, i]
        history[:, step] = ids.to(torch.int32)
    assert np.array_equal(to_host(history), np.array(beams, np.int32))
    want = rows[torch.from_numpy(np.array(beams)).cuda()]  # [N][T][2][Hkv][D]
    for i in (0, 1):
        assert torch.equal(cache[i], want[:, :, i].transpose(1, 2))
    # and the attention over them
    q = torch.from_numpy(rng.normal(0, 1, (N, Hq, D)).astype(np.float32)).bfloat16().cuda()
    out = torch.empty(N, Hq * D, device="cuda").bfloat16()
    sinks = torch.full((Hq,), -1e30, device="cuda").bfloat16()
    pos = torch.full((N,), T - 1, dtype=torch.int32, device="cuda")
    ne.attn_decode(q, cache[0], cache[1], sinks, pos, out, N, Hq, Hkv, D, T, 0)
    for b in range(N):
        for h in range(Hq):
            k, v = (want[b, :, i, h // 2].double().cpu().numpy() for i in (0, 1))
            x = k @ q[b, h].double().cpu().numpy() / 8
            p = np.exp(x - x.max())
            ref = p @ v / p.sum()
            got = out[b, h * D:(h + 1) * D].float().cpu().numpy()
            assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -12).all()
    ne.device_check()


class Calls:
    """A choice, a fork and a compaction, each from fixed inputs into outputs of its own."""

    def __init__(self, seed, B, W, vocab, n_pages, width):
        torch = torch_cuda()
        rng = np.random.default_rng(seed)
        self.W, N = W, B * W
        logits = rng.normal(0, 2.5, (N, vocab)).astype(np.float32)
        score = (-3 - rng.random(N)).astype(np.float32)
        # one sequence of each request has tokens, the others continue it
        length = np.zeros(N, np.int32)
        length[::W] = rng.integers(1, 60, B)
        table, refs = np.full((N, width), -1, np.int32), np.zeros(n_pages, np.int32)
        free = rng.permutation(n_pages)
        for b in range(0, N, W):
            k = beam_util.pages(length[b], PAGE)
            table[b, :k], free = free[:k], free[k:]
            refs[table[b, :k]] = 1
        parent = np.repeat(np.arange(0, N, W), W).astype(np.int32)
        fill = np.full((N, width), -9, np.int32)
        fork, out_of_pages = beam_util.fork(refs, table, length, PAGE, fill, parent=parent)
        assert not out_of_pages
        self.want = [*beam_util.select(logits, score, W)[:2], *fork,
                     *beam_util.compact(refs, table, length, PAGE, fill)]
        self.ins = [to_dev(x) for x in (logits, score, refs, table, length, parent)]
        self.out_score = torch.empty(N, device="cuda")
        shapes = [(N,), (N,), (n_pages,), (N, width), (N,), (N,), (N,), (N,), (n_pages,), (N, width), (n_pages,),
                  (n_pages // 2,), (n_pages // 2,)]
        self.outs = [torch.empty(s, dtype=torch.int32, device="cuda") for s in shapes]
        wb, cb = ne.pages_workspace(n_pages, N)
        self.needs = ne.beam_select_workspace(B, W, vocab, 0), wb, cb

    def __call__(self, select_ws, plan_ws, counters):
        logits, score, refs, table, length, parent = self.ins
        o = self.outs
        ne.beam_select(logits, score, self.W, o[0], o[1], self.out_score, workspace=select_ws)
        ne.pages_fork(refs, table, length, PAGE, o[2], o[3], o[4], o[5:8], parent=parent, workspace=plan_ws,
                      counters=counters)
        ne.pages_compact(refs, table, length, PAGE, *o[8:11], o[11:13], workspace=plan_ws)

    def clear(self):
        for o in self.outs:
            o.fill_(-9)

    def check(self):
        assert len(self.outs) == len(self.want)
        for i, (o, w) in enumerate(zip(self.outs, self.want)):
            assert np.array_equal(to_host(o), w), i


# (one block each, and several launches each)
SIZES = [[(3, 4, 5000, 200, 8), (7, 2, 900, 90, 5)], [(40, 8, 3000, 9000, 12), (100, 3, 20011, 30000, 7)]]


def buffers(needs):
    torch = torch_cuda()
    s, w, c = needs
    return (torch.full((s,), 0xA5, dtype=torch.uint8, device="cuda"),
            torch.full((w,), 0xA5, dtype=torch.uint8, device="cuda"),
            torch.zeros(c, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("sizes", SIZES, ids=["small", "large"])
def test_graphs_share_workspaces(sizes):
    """Two captured graphs of calls of different sizes with one set of workspaces and
    counters, replayed in turn with an eager call in between."""
    torch = torch_cuda()
    calls = [Calls(20 + i, *s) for i, s in enumerate(sizes)]
    shared = buffers([max(n) for n in zip(*(c.needs for c in calls))])
    for c in calls:
        c(*shared)
    torch.cuda.synchronize()
    graphs = []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c(*shared)
    for replay in range(5):
        say("replay", replay)
        for c in calls:
            c.clear()
        for g in graphs if replay % 2 else graphs[::-1]:
            g.replay()
        for c in calls:
            c.check()
        calls[replay % 2].clear()
        calls[replay % 2](*shared)
        calls[replay % 2].check()
    assert not shared[2].any()
    ne.device_check()


@pytest.mark.parametrize("sizes", SIZES, ids=["small", "large"])
def test_two_streams_at_once(sizes):
    """The same calls on two streams, each with workspaces and counters of its own."""
    torch = torch_cuda()
    calls = [Calls(30 + i, *s) for i, s in enumerate(sizes)]
    own = [buffers(c.needs) for c in calls]
    for c in calls:
        c.clear()
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, b, s in zip(calls, own, streams):
            with torch.cuda.stream(s):
                c(*b)
    torch.cuda.synchronize()
    for c in calls:
        c.check()
    ne.device_check()


@pytest.mark.parametrize("max_pages", [10, 9000])
@pytest.mark.parametrize("steps", [1, 2])
def test_pages_run_out_in_a_run(max_pages, steps):
    """The fork of a step needs more pages than are free; the append and the attention that
    follow, and the fork of the next step, meet the entries without one.  The check names
    the cause, once.  (max_pages: a plan of one launch, and of three.)"""
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, V, n) for n in (16, 31)]
    # 3 pages of the prompts; 4 and 3 more for the first tokens; then 4 more for the second
    s = Search(prompts, 4, 12, max_pages, [], seed=13)
    s.choose()
    s.advance(first=True)
    ne.device_check()
    assert int((s.refs == 0).sum()) == 2
    say(f"pages run out, width {max_pages}, {steps} steps")
    for _ in range(steps):
        s.choose()
        s.advance()
    with pytest.raises(ne.NeonError) as e:
        ne.device_check()
    assert e.value.status == ne.NEON_EKV_FULL
    ne.device_check()
