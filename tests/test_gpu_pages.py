"""GPU tests of neon_pages_fork, neon_pages_copy and neon_pages_compact against
their plain forms: everything is whole numbers or moved bytes, and has to be equal."""
import sys

import numpy as np
import pytest

import neonengine_amd as ne
from tests import beam_util
from tests.beam_util import Pool
from tests.gpu_util import empty_dev, to_dev, to_host, torch_cuda

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def run_fork(refs, table, length, page, B, in_place=False, counters=None, workspace=None, **seqs):
    torch = torch_cuda()
    d = [to_dev(x) for x in (refs, table, length)]
    outs = [empty_dev(len(refs), np.int32), torch.full((B, table.shape[1]), -9, dtype=torch.int32, device="cuda"),
            empty_dev(B, np.int32)]
    if in_place:
        outs = [d[0], d[1] if in_place == "all" else outs[1], d[2] if B == len(length) else outs[2]]
    copies = [torch.full((B,), 99, dtype=torch.int32, device="cuda") for _ in range(3)]
    k = {n: to_dev(np.asarray(v, np.int32)) for n, v in seqs.items() if v is not None}
    ne.pages_fork(*d, page, *outs, copies, counters=counters, workspace=workspace, **k)
    return [to_host(x) for x in (*outs, *copies)]


def check_fork(pool, B, in_place=False, full=False, counters=None, workspace=None, **seqs):
    start = np.full((B, pool.width), -9, np.int32)
    if in_place == "all":
        start = pool.table
    want, ran_out = beam_util.fork(pool.refs, pool.table, pool.length, pool.page, start, **seqs)
    full = ran_out if full is None else full  # None: as the plain form has it
    assert ran_out == full
    got = run_fork(pool.refs, pool.table, pool.length, pool.page, B, in_place, counters, workspace, **seqs)
    for name, g, w in zip(("refs", "table", "length", "src", "dst", "rows"), got, want):
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5])
    if full:
        with pytest.raises(ne.NeonError) as e:
            ne.device_check()
        assert e.value.status == ne.NEON_EKV_FULL
    ne.device_check()
    return got


def lengths(rng, n, top, page):
    x = np.exp(rng.uniform(0, np.log(top), n)).astype(int)
    x[rng.random(n) < 0.2] = page * rng.integers(0, max(1, top // page))  # page borders, and none
    return x


@pytest.mark.parametrize("B,W,page,top,spare", [
    (1, 1, 16, 40, 40), (1, 4, 16, 100, 30), (3, 4, 64, 2000, 100), (16, 4, 16, 3000, 3000),
    (9, 8, 128, 5000, 100), (100, 5, 16, 300, 6000), (2, 3, 16, 9000, 40), (4, 32, 16, 500, 400)])
@pytest.mark.parametrize("kind", ["beams", "any", "samples", "grow", "drafts", "new"])
@pytest.mark.parametrize("wide", [False, True])
def test_fork(B, W, page, top, spare, kind, wide):
    """wide: tables of more entries than the launch of one block takes."""
    rng = np.random.default_rng(B * W + top)
    lens = lengths(rng, B, top, page)
    N = B * W
    pool = Pool(rng, lens, W, page, spare + 2 * B * W * (1 + 16 // page + 4), tail=kind in ("any", "grow"),
                held=min(20, spare), width=max((top + 40) // page + 3, 65536 // N + 2 if wide else 0))
    say(f"fork {kind} B={B} W={W} page={page} top={top} pages={pool.n_pages} wide={wide}")
    if kind in ("beams", "any"):
        first = np.repeat(np.arange(B) * W, W)
        parent = first + rng.integers(0, W, N)
        if kind == "beams":
            parent = np.where(rng.random(N) < 0.6, np.arange(N), parent)
        else:  # any row of the batch, some of none
            parent = np.where(rng.random(N) < 0.3, rng.integers(-1, N, N), parent)
        check_fork(pool, N, parent=parent)
        check_fork(pool, N, parent=parent, in_place="refs")
    elif kind == "samples":  # more sequences than before
        check_fork(pool, 2 * N + 1, parent=rng.integers(0, N, 2 * N + 1))
    elif kind == "grow":
        check_fork(pool, N)
        check_fork(pool, N, in_place="all")
        check_fork(pool, N, in_place="all", add=rng.integers(0, 30, N))
    elif kind == "drafts":
        keep = np.maximum(pool.length - rng.integers(0, 20, N), 0)
        check_fork(pool, N, keep=keep, add=rng.integers(0, 9, N), in_place="all")
        check_fork(pool, N, keep=keep, parent=np.arange(N))
    else:  # some leave, new ones come
        parent = np.where(rng.random(N) < 0.5, np.arange(N), -1)
        add = np.where(parent < 0, rng.integers(0, page, N), 1)
        check_fork(pool, N, parent=parent, add=add)
        check_fork(pool, max(1, N // 2), parent=parent[:max(1, N // 2)], add=add[:max(1, N // 2)])


@pytest.mark.parametrize("n_pages,used,B", [(8192, 8000, 64), (8193, 8100, 64), (70000, 66000, 300),
                                            (200000, 150, 1500), (300000, 299000, 40)])
def test_fork_large_pools(n_pages, used, B):
    """Most of the pool held by others, the free pages anywhere in it; whole prompts and
    single tokens."""
    rng = np.random.default_rng(n_pages)
    pool = Pool(rng, np.minimum(lengths(rng, B, 60, 16), 60), 1, 16, n_pages, width=30)
    pool.n_pages = n_pages
    pool.refs = pool.refs[:n_pages].copy()
    pool.table[:] = -7
    ids = rng.permutation(n_pages)
    at = 0
    pool.refs[:] = 0
    for b, n in enumerate(pool.length):
        k = beam_util.pages(n, 16)
        pool.table[b, :k] = ids[at:at + k]
        at += k
    pool.refs[ids[:at]] = 1
    pool.refs[ids[:max(at, used)]] += 1
    parent = np.where(rng.random(B) < 0.5, np.arange(B), rng.integers(-1, B, B))
    need = np.where(rng.random(B) < 0.2, rng.integers(0, 300, B), 1)
    say(f"large pool {n_pages} used {used} B={B}")
    check_fork(pool, B, parent=parent, add=need, full=None)
    check_fork(pool, B, in_place="all", full=None)


@pytest.mark.parametrize("width", [6, 6000])
def test_fork_without_free_pages(width):
    rng = np.random.default_rng(3)
    for spare in (0, 1, 5):
        pool = Pool(rng, [32, 32, 20, 16], 3, 16, spare, held=0, width=width)
        say(f"pages run out, {spare} spare")
        check_fork(pool, 12, full=True, add=[17] * 12)
        check_fork(pool, 12, full=True, parent=np.repeat(np.arange(4) * 3, 3), add=[40] * 12)


@pytest.mark.parametrize("width", [40, 9000])
def test_fork_counters_serve_again(width):
    """One set of counters and workspace for calls of different sizes."""
    torch = torch_cuda()
    rng = np.random.default_rng(4)
    pools = [Pool(rng, lengths(rng, b, 400, 16), 4, 16, 300, width=width) for b in (30, 2, 11)]
    n = max(p.n_pages for p in pools)
    wb, cb = ne.pages_workspace(n, 200)
    ws = torch.full((wb,), 0xA5, dtype=torch.uint8, device="cuda")
    counters = torch.zeros(cb, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for p in pools:
            N = len(p.table)
            check_fork(p, N, parent=np.repeat(np.arange(N // 4) * 4, 4), counters=counters, workspace=ws)
            assert not to_host(counters).any()


@pytest.mark.parametrize("width", [6, 20000])
def test_fork_numbers_that_do_not_fit(width):
    """Such a sequence is left without tokens; the others are as they would be."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, [40, 35, 70, 16], 1, 16, 60, width=width)
    top = width * 16
    for what, seqs, good in [
            ("parent", dict(parent=[0, 4, 2, 3]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1])),
            ("parent", dict(parent=[0, -2, 2, 3]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1])),
            ("keep", dict(keep=[40, 36, 70, 16]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1])),
            ("keep", dict(keep=[40, -1, 70, 16]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1])),
            ("add", dict(add=[1, -1, 1, 1]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1])),
            ("add", dict(add=[1, top, 1, 1]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1])),
            ("add", dict(add=[1, 2 ** 31 - 1, 1, 1]), dict(parent=[0, -1, 2, 3], add=[1, 0, 1, 1]))]:
        say(f"bad {what} {seqs}")
        want, _ = beam_util.fork(pool.refs, pool.table, pool.length, 16, np.full((4, width), -9, np.int32), **good)
        got = run_fork(pool.refs, pool.table, pool.length, 16, 4, **seqs)
        for g, w in zip(got, want):
            assert np.array_equal(g, w)
        with pytest.raises(ne.NeonError) as e:
            ne.device_check()
        assert e.value.status == ne.NEON_EINVAL
        ne.device_check()
    # a length that is none: the row holds nothing
    for n in (-1, top + 1, 2 ** 31 - 1):
        length = pool.length.copy()
        length[1] = n
        say(f"bad length {n}")
        clean = length.copy()
        clean[1] = 0
        want, _ = beam_util.fork(pool.refs, pool.table, clean, 16, np.full((4, width), -9, np.int32))
        got = run_fork(pool.refs, pool.table, length, 16, 4)
        for g, w in zip(got, want):
            assert np.array_equal(g, w)
        with pytest.raises(ne.NeonError):
            ne.device_check()
    # page ids that are none are passed on and not counted
    table = pool.table.copy()
    table[2, 0], table[2, 4] = -5, pool.n_pages
    say("bad page ids")
    got = run_fork(pool.refs, table, pool.length, 16, 4)
    assert got[1][2, 0] == -5 and got[1][2, 4] == pool.n_pages and got[2].tolist() == [41, 36, 71, 17]
    with pytest.raises(ne.NeonError):
        ne.device_check()


def check_wrong_counts(refs, table, length, want, page=16, **seqs):
    """A fork whose counts are not those of the table: its outputs (entries past a row's
    pages are -9), and the error, once."""
    start = np.full_like(table, -9)
    for name, w in zip(("refs", "table", "length", "src", "dst", "rows"), want):
        if name == "table":
            for row, ids in zip(start, w):
                row[:len(ids)] = ids
    want = [w if i != 1 else start for i, w in enumerate(want)]
    got = run_fork(refs, table, length, page, len(want[2]), **seqs)
    for name, g, w in zip(("refs", "table", "length", "src", "dst", "rows"), got, want):
        assert np.array_equal(g, w), (name, g, w)
    with pytest.raises(ne.NeonError) as e:
        ne.device_check()
    assert e.value.status == ne.NEON_EINVAL
    ne.device_check()


WIDTHS = [4, 40000]  # a plan of one launch, and of three


def wide_table(rows, width):
    t = np.full((len(rows), width), -7, np.int32)
    for r, ids in zip(t, rows):
        r[:len(ids)] = ids
    return t


@pytest.mark.parametrize("width", WIDTHS)
def test_fork_counts_below_the_writers(width):
    """A page that goes on being written by more sequences than its count says: the first
    keeps it, the others get a copy, its count is 1, and the error is set."""
    i32 = lambda *x: np.array(x, np.int32)
    for count in (1, 2):
        refs = i32(0, 0, 0, 0, 0, count)
        say(f"count {count} of a page of three writers")
        check_wrong_counts(refs, wide_table([[5]] * 3, width), i32(10, 4, 7),
                           (i32(1, 1, 0, 0, 0, 1), [[5], [0], [1]], i32(11, 5, 8), i32(-1, 5, 5),
                            i32(-1, 0, 1), i32(0, 4, 7)))
    # children of one row, which the count leaves out
    say("count 0 of a page of two writers")
    check_wrong_counts(i32(0, 1, 0), wide_table([[2], [1]], width), i32(10, 16),
                       (i32(1, 0, 1), [[2], [0]], i32(11, 11), i32(-1, 2), i32(-1, 0), i32(0, 10)),
                       parent=[0, 0])
    # a writer whose page has no count at all
    say("count 0 of a page that is written")
    check_wrong_counts(i32(0, 0, 0), wide_table([[0], []], width), i32(10, 0),
                       (i32(1, 1, 0), [[0], [1]], i32(11, 5), i32(-1, -1), i32(-1, -1), i32(0, 0)),
                       add=[1, 5])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("width", WIDTHS)
def test_fork_held_pages_without_a_count(width, in_place):
    """A page that a sequence of the result holds is not handed out, whatever its count
    says: it stays with a count of 1, and the error is set."""
    torch = torch_cuda()
    i32 = lambda *x: np.array(x, np.int32)
    # the full page 0 of the first sequence was never counted; the second grows
    cases = [("never counted", i32(0, 1, 1, 0), [[0, 2], [1]], i32(20, 16), None, i32(1, 16),
              i32(1, 1, 1, 1), [[0, 2], [1, 3]], i32(21, 32)),
             # a page of two sequences that was released twice: one leaves, the other stays
             ("released twice", i32(1, 1, 0), [[0], [0, 1]], i32(16, 20), i32(0, 20), i32(0, 13),
              i32(1, 1, 1), [[], [0, 1, 2]], i32(0, 33))]
    for what, refs, rows, length, keep, add, refs_out, rows_out, len_out in cases:
        if in_place:
            table = wide_table(rows, width)
            d = [to_dev(x) for x in (refs, table, length)]
            copies = [torch.full((2,), 99, dtype=torch.int32, device="cuda") for _ in range(3)]
            ne.pages_fork(*d, 16, *d, copies, keep=None if keep is None else to_dev(keep), add=to_dev(add))
            got = [to_host(x) for x in d]
            assert np.array_equal(got[0], refs_out) and np.array_equal(got[2], len_out), (what, got)
            for row, ids in zip(got[1], rows_out):
                assert row[:len(ids)].tolist() == ids
            with pytest.raises(ne.NeonError) as e:
                ne.device_check()
            assert e.value.status == ne.NEON_EINVAL
            ne.device_check()
        else:
            check_wrong_counts(refs, wide_table(rows, width), length,
                               (refs_out, rows_out, len_out, i32(-1, -1), i32(-1, -1), i32(0, 0)),
                               keep=keep, add=add)


@pytest.mark.parametrize("n_pages,B,page,top", [(1, 1, 16, 10), (2, 1, 16, 16), (5, 2, 16, 30), (1023, 7, 16, 900),
                                                (1024, 7, 64, 900), (1025, 30, 16, 100), (5000, 300, 16, 200),
                                                (70000, 64, 16, 9000)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_compact(n_pages, B, page, top, in_place, wide):
    torch = torch_cuda()
    rng = np.random.default_rng(n_pages + B)
    lens = lengths(rng, B, top, page)
    while sum(beam_util.pages(n, page) for n in lens) > n_pages:
        lens[rng.integers(0, B)] = 0
    used = sum(beam_util.pages(n, page) for n in lens)
    for held in sorted({0, (n_pages - used) // 3, n_pages}):
        pool = Pool(rng, lens, 1, page, n_pages - used, held=held,
                    width=max(top // page + 3, 65536 // B + 2 if wide else 0))
        say(f"compact n_pages={n_pages} used={used} held={held} in place {in_place}")
        d = [to_dev(x) for x in (pool.refs, pool.table, pool.length)]
        start = pool.table if in_place else np.full_like(pool.table, -9)
        outs = d[:2] if in_place else [empty_dev(n_pages, np.int32), to_dev(start)]
        to, src, dst = (empty_dev(max(1, k), np.int32) for k in (n_pages, n_pages // 2, n_pages // 2))
        ne.pages_compact(*d, page, *outs, to, (src, dst))
        want = beam_util.compact(pool.refs, pool.table, pool.length, page, start)
        got = [to_host(x) for x in (*outs, to, src[:n_pages // 2], dst[:n_pages // 2])]
        for name, g, w in zip(("refs", "table", "map", "src", "dst"), got, want):
            assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5])
        ne.device_check()


@pytest.mark.parametrize("width", [6, 30000])
def test_compact_numbers_that_do_not_fit(width):
    rng = np.random.default_rng(6)
    pool = Pool(rng, [40, 35, 70], 1, 16, 60, width=width)
    refs, table, length = pool.refs.copy(), pool.table.copy(), pool.length.copy()
    table[0, 1] = pool.n_pages + 3
    length[1] = 16 * width + 1
    lost = table[2, 2]
    refs[lost] = 0
    d = [to_dev(x) for x in (refs, table, length)]
    to, src, dst = (empty_dev(k, np.int32) for k in (pool.n_pages, pool.n_pages // 2, pool.n_pages // 2))
    out = to_dev(np.full_like(table, -9))
    ne.pages_compact(*d, 16, empty_dev(pool.n_pages, np.int32), out, to, (src, dst))
    out, to = to_host(out), to_host(to)
    assert out[0, 1] == pool.n_pages + 3 and (out[1] == -9).all() and out[2, 2] == -1
    assert out[0, 0] == to[table[0, 0]] and out[2, 4] == to[table[2, 4]] and to[lost] == -1
    with pytest.raises(ne.NeonError):
        ne.device_check()
    ne.device_check()


def caches(rng, n_kv, n_pages, Hkv, page, D, mx):
    """Host pools and their device copies."""
    out = []
    for _ in range(n_kv):
        if mx:
            p = [rng.integers(0, 256, (n_pages, Hkv, page, w)).astype(np.uint8)
                 for w in (D // 2, D // 2, D // 32, D // 32)]
        else:
            p = [rng.integers(0, 65536, (n_pages, Hkv, page, D)).astype(np.uint16) for _ in range(2)]
        out.append((p, [to_dev(x) for x in p]))
    return out


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("n_kv,n_pages,Hkv,page,D,n", [
    (1, 4, 1, 16, 64, 1), (3, 300, 2, 16, 64, 130), (2, 41, 3, 32, 128, 20), (70, 9, 1, 16, 64, 3),
    (1, 20, 8, 256, 128, 9), (24, 140, 8, 16, 64, 64)])
def test_copy(n_kv, n_pages, Hkv, page, D, n, mx):
    rng = np.random.default_rng(n_pages + n)
    pools = caches(rng, n_kv, n_pages, Hkv, page, D, mx)
    layers = ne.paged_layers([ne.paged_kv(*d) for _, d in pools])
    ids = rng.permutation(n_pages).astype(np.int32)
    src, dst = ids[:n].copy(), ids[n_pages - n:].copy() if 2 * n <= n_pages else ids[:n].copy()
    src[rng.random(n) < 0.2] = -1
    dst[rng.random(n) < 0.2] = -1
    if n > 1:
        src[-1] = src[0]  # a page may be read twice
    rows = rng.integers(0, page + 1, n).astype(np.int32)
    for r in (rows, None):
        say(f"copy n_kv={n_kv} pages={n_pages} Hkv={Hkv} page={page} D={D} n={n} mx={mx} rows={r is not None}")
        ne.pages_copy(layers, to_dev(src), to_dev(dst), None if r is None else to_dev(r))
        for host, dev in pools:
            for h, t in zip(host, dev):
                want = h.copy()
                for i in range(n):
                    if src[i] >= 0 and dst[i] >= 0:
                        k = page if r is None else r[i]
                        want[dst[i], :, :k] = h[src[i], :, :k]
                assert np.array_equal(to_host(t), want)
                h[:] = want
    ne.device_check()


def test_copy_bad_entries_are_dropped():
    rng = np.random.default_rng(7)
    (host, dev), = caches(rng, 1, 10, 2, 16, 64, False)
    kv = ne.paged_kv(*dev)
    for src, dst, rows in (([10], [1], [4]), ([0], [10], [4]), ([-2], [1], [4]), ([0], [1], [17]),
                           ([0], [1], [-1]), ([0], [1 << 30], [3])):
        ne.pages_copy(kv, *(to_dev(np.array(x, np.int32)) for x in (src, dst, rows)))
        with pytest.raises(ne.NeonError):
            ne.device_check()
    for h, t in zip(host, dev):
        assert np.array_equal(to_host(t), h)
    ne.pages_copy(kv, *(to_dev(np.array(x, np.int32)) for x in ([], [])))
    ne.device_check()


def test_refusals_python():
    torch = torch_cuda()
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    c3 = (i(2), i(2), i(2))
    good = (i(9), i(2, 4), i(2), 16, i(9), i(2, 4), i(2), c3)
    ne.pages_fork(*good)
    for at, bad in ((0, i(9).float()), (1, i(8)), (1, i(3, 4)), (4, i(8)), (5, i(2, 5)), (5, i(8)), (6, i(1)),
                    (7, (i(2), i(1), i(2))), (2, i(2).cpu()), (0, i(9).long())):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            ne.pages_fork(*args)
    with pytest.raises(ValueError):
        ne.pages_fork(*good, keep=i(3).float())
    with pytest.raises(ne.NeonError):
        ne.pages_fork(*good, workspace=i(1))
    t = i(2, 4)
    with pytest.raises(ne.NeonError):
        ne.pages_fork(i(9), t, i(2), 16, i(9), t, i(2), c3, parent=i(2))
    comp = (i(9), i(2, 4), i(2), 16, i(9), i(2, 4), i(9), (i(4), i(4)))
    ne.pages_compact(*comp)
    for at, bad in ((6, i(8)), (7, (i(4), i(3))), (5, i(7)), (1, i(2, 4).float())):
        args = list(comp)
        args[at] = bad
        with pytest.raises(ValueError):
            ne.pages_compact(*args)
    with pytest.raises(ValueError):
        ne.paged_layers([])
    ne.device_check()


def guarded(n, dtype):
    """(the whole buffer, its middle of n elements) with a sentinel on both sides."""
    torch = torch_cuda()
    whole = torch.full((n + 128,), 0x5A5A5A5A if dtype is torch.int32 else 0x5A, dtype=dtype, device="cuda")
    return whole, whole[64:64 + n]


def untouched(whole, n):
    a = to_host(whole)
    return (a[:64] == a[0]).all() and (a[64 + n:] == a[0]).all() and a[0] in (0x5A5A5A5A, 0x5A)


@pytest.mark.parametrize("n_pages,B,W,width", [(97, 2, 3, 8), (900, 16, 4, 30), (9000, 3, 4, 40), (1100, 30, 8, 20),
                                               (2049, 1, 1, 70000)])
def test_plans_stay_inside_their_buffers(n_pages, B, W, width):
    torch = torch_cuda()
    rng = np.random.default_rng(n_pages)
    lens = np.minimum(lengths(rng, B, 100, 16), 100)
    while sum(beam_util.pages(n, 16) * W for n in lens) + 2 * B * W > n_pages:
        lens[rng.integers(0, B)] = 0
    pool = Pool(rng, lens, W, 16, n_pages, width=width)
    pool.n_pages = n_pages
    keep = pool.table[pool.table >= 0]
    remap = np.full(len(pool.refs), -1)
    used = np.unique(keep)
    remap[used] = rng.permutation(n_pages)[:len(used)]
    pool.table = np.where(pool.table >= 0, remap[np.clip(pool.table, 0, None)], -7).astype(np.int32)
    refs = np.zeros(n_pages, np.int32)
    np.add.at(refs, pool.table[pool.table >= 0], 1)
    pool.refs = refs
    N = B * W
    parent = np.repeat(np.arange(B) * W, W) + rng.integers(0, W, N)
    want, full = beam_util.fork(refs, pool.table, pool.length, 16, np.full((N, width), 0x5A5A5A5A, np.int32),
                                parent=parent)
    wb, cb = ne.pages_workspace(n_pages, N)
    i32, u8 = torch.int32, torch.uint8
    sizes = [n_pages, N * width, N, N, N, N]
    bufs = [guarded(n, i32) for n in sizes]
    ws = guarded(-(-wb // 16) * 16, u8)
    ws_mid = ws[1][:wb]
    counters = guarded(cb, u8)
    counters[1].zero_()
    d = [to_dev(x) for x in (refs, pool.table, pool.length)]
    m = [b[1] for b in bufs]
    say(f"guards n_pages={n_pages} B={B} W={W} width={width}")
    ne.pages_fork(*d, 16, m[0], m[1].view(N, width), m[2], m[3:], parent=to_dev(parent.astype(np.int32)),
                  workspace=ws_mid, counters=counters[1])
    for g, w in zip(m, want):
        assert np.array_equal(to_host(g), w.reshape(-1))
    assert all(untouched(b[0], n) for b, n in zip(bufs, sizes))
    assert untouched(ws[0], len(ws[1])) and untouched(counters[0], cb) and not to_host(counters[1]).any()
    sizes = [n_pages, N * width, n_pages, n_pages // 2, n_pages // 2]
    bufs = [guarded(n, i32) for n in sizes]
    m = [b[1] for b in bufs]
    ne.pages_compact(*d, 16, m[0], m[1].view(N, width), m[2], m[3:], workspace=ws_mid)
    want = beam_util.compact(refs, pool.table, pool.length, 16, np.full((N, width), 0x5A5A5A5A, np.int32))
    for g, w in zip(m, want):
        assert np.array_equal(to_host(g), w.reshape(-1))
    assert all(untouched(b[0], n) for b, n in zip(bufs, sizes)) and untouched(ws[0], len(ws[1]))
    ne.device_check()
