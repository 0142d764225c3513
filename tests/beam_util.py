"""Plain forms of beam search's choice, of the move of its states, and of the
plans over a cache's pages, for the tests of neon_beam_* and neon_pages_*."""
import numpy as np


def select(logits, score, W, stop=()):
    """The definition in 64 bits: token, parent, score of the next beams and of
    the ended ones, [B W] each (float64 scores)."""
    N, V = logits.shape
    stop = {int(t) for t in stop}
    token, parent, out = np.full(N, -1), np.full(N, -1), np.full(N, -np.inf)
    e_token, e_parent, e_score = np.full(N, -1), np.full(N, -1), np.full(N, -np.inf)
    for b in range(0, N, W):
        cand = []
        for w in range(W):
            s = float(score[b + w])
            x = logits[b + w].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            if not np.isfinite(s) or not x.size or not np.isfinite(x.max()):
                continue
            m = x.max()
            lse = m + np.log(np.exp(x - m).sum())
            order = np.lexsort((np.arange(V), -x))[:W + len(stop)]
            cand += [(-(s + (x[t] - lse)), w, r, int(t)) for r, t in enumerate(order) if x[t] > -np.inf]
        cand.sort()
        n = 0
        for v, w, _, t in cand[:W]:
            if t in stop:
                e_token[b + n], e_parent[b + n], e_score[b + n] = t, b + w, -v
                n += 1
        place, rest = {}, []
        for v, w, _, t in [c for c in cand if c[3] not in stop][:W]:
            if w in place:
                rest.append((t, w, -v))
            else:
                place[w] = (t, w, -v)
        for w in range(W):
            if w not in place and rest:
                place[w] = rest.pop(0)
        for w, (t, p, v) in place.items():
            token[b + w], parent[b + w], out[b + w] = t, b + p, v
    return token, parent, out, e_token, e_parent, e_score


def reorder(state, parent, length, W):
    """state [N][slabs][T][..] with row r become row parent[r] (first tokens)."""
    out = state.copy()
    for r, p in enumerate(parent):
        if p // W == r // W and p >= 0:
            n = state.shape[2] if length is None else min(max(length[p], 0), state.shape[2])
            out[r, :, :n] = state[p, :, :n]
    return out


def pages(n, page):
    return -(-int(n) // page)


def fork(refs, table, length, page, table_out, parent=None, keep=None, add=None):
    """refs, table, lengths and copies after neon_pages_fork; whether pages ran
    out.  Every number has to be one that the call takes."""
    refs = [int(r) for r in refs]
    out = table_out.copy()
    B = len(out)
    seqs = []
    for b in range(B):
        p = b if parent is None else int(parent[b])
        n = int(length[p]) if p >= 0 else 0
        k = int(keep[b]) if keep is not None and p >= 0 else n
        seqs.append((p, k, int(add[b]) if add is not None else int(n > 0)))
    for r, n in enumerate(length):
        for i in range(pages(n, page)):
            refs[table[r][i]] -= 1
    writers = {}
    for b, (p, k, a) in enumerate(seqs):
        for i in range(pages(k, page)):
            refs[table[p][i]] += 1
        if k % page and a > 0:
            writers.setdefault(int(table[p][k // page]), []).append(b)
    free = [p for p, r in enumerate(refs) if r == 0]
    full = False
    holders = list(refs)
    src, dst, cnt = [-1] * B, [-1] * B, [0] * B

    def take():
        nonlocal full
        if not free:
            full = True
            return -1
        refs[free[0]] = 1
        return free.pop(0)

    for b, (p, k, a) in enumerate(seqs):
        row = [int(table[p][i]) for i in range(pages(k, page))]
        if k % page and a > 0:
            at, all_write = row[-1], len(writers[row[-1]]) == holders[row[-1]]
            if holders[at] > 1 and not (all_write and writers[at][0] == b):
                refs[at] -= 1
                row[-1] = take()
                src[b], dst[b], cnt[b] = at, row[-1], k % page
        while len(row) < pages(k + a, page):
            row.append(take())
        out[b, :len(row)] = row
    ints = [np.array(x, np.int32) for x in (refs, [k + a for _, k, a in seqs], src, dst, cnt)]
    return (ints[0], out, *ints[1:]), full


def compact(refs, table, length, page, table_out):
    """refs, table, new ids and moves after neon_pages_compact."""
    n = len(refs)
    used = [p for p in range(n) if refs[p]]
    U = len(used)
    src = [p for p in used if p >= U]
    dst = [p for p in range(U) if not refs[p]]
    to = np.array([p if refs[p] else -1 for p in range(n)], np.int32)
    to[src] = dst
    out_refs = np.zeros(n, np.int32)
    out_refs[to[used]] = refs[used]
    out = table_out.copy()
    for b, k in enumerate(length):
        for i in range(pages(k, page)):
            out[b, i] = to[table[b, i]]
    lists = [np.array((x + [-1] * n)[:n // 2], np.int32) for x in (src, dst)]
    return (out_refs, out, to, *lists)


class Pool:
    """Sequences over randomly ordered pages of a pool: requests of W sequences
    that share their first pages (and, with `tail`, the partial one), some pages
    held by others as well.  Entries that no sequence holds are poison."""

    def __init__(self, rng, lens, W, page, spare, width=None, tail=False, held=0):
        self.page, self.W = page, W
        rows, refs = [], {}
        at = 0
        for n in lens:
            shared = pages(n, page) if tail else int(n) // page
            first = list(range(at, at + shared))
            at += shared
            for _ in range(W):
                more = pages(n, page) - shared
                rows.append(first + list(range(at, at + more)))
                at += more
        self.n_pages = at + spare
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.length = np.repeat(np.array(lens, np.int32), W)
        self.refs = np.zeros(self.n_pages, np.int32)
        self.width = width or max(1, max(len(r) for r in rows)) + 2
        self.table = np.full((len(rows), self.width), -7, np.int32)
        for b, r in enumerate(rows):
            self.table[b, :len(r)] = ids[r]
            np.add.at(self.refs, ids[r], 1)
        others = rng.choice(self.n_pages, held, replace=False)
        self.refs[others] += 1
