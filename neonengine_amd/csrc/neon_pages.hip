// neon_pages.hip -- the pages of a cache as a whole: which sequence holds which
// (forking, growing, cutting and freeing by reference counts), copying pages, and
// compacting the pool.
//
// A sequence of n tokens holds the pages 0 .. ceil(n / page) - 1 of its table row.
// refs[p] counts the holders of page p, sequences of the batch and others; 0 is a
// free page.  No free list: free pages are taken in the order of their ids, so the
// result depends on no order of threads, and there is nothing to keep in step.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "neon_common.hpp"
#include "neon_internal.hpp"

namespace neon {

constexpr int kPgChunk = 1024;    // pages of a block: 4 of a thread
constexpr int kPgSeqs = 256;      // sequences of a block of the plan
constexpr int kPgSpan = 256;      // table entries of a wave, 4 of a lane
constexpr int kPgLongest = 1 << 30;

// What sequence b of the result is made of.
struct PgSeq {
  int parent;  // row of the old table, -1: none
  int keep, add;
};
__device__ __forceinline__ bool pg_len_ok(const PagesForkArgs& a, int n) {
  return n >= 0 && n <= kPgLongest && (int64_t)n <= (int64_t)a.max_pages << a.page_log2;
}
__device__ __forceinline__ int pg_pages(int page_log2, int n) {
  return (n + (1 << page_log2) - 1) >> page_log2;
}
// tokens of an old row (0 where its length is none)
__device__ __forceinline__ int pg_len(const PagesForkArgs& a, int p) {
  const int n = a.len[p];
  return pg_len_ok(a, n) ? n : 0;
}
// Sequence b with its parent's tokens and what keep and add say (where they are given).
// ok: false where the numbers are none; the sequence is then left without tokens.
__device__ __forceinline__ int pg_parent(const PagesForkArgs& a, int b) {
  return a.parent != nullptr ? a.parent[b] : b;
}
__device__ __forceinline__ PgSeq pg_seq_of(const PagesForkArgs& a, int parent, int len, int keep, int add,
                                           bool& ok) {
  PgSeq q;
  const int n = pg_len_ok(a, len) ? len : 0;
  q.parent = parent;
  q.keep = a.keep != nullptr && parent >= 0 ? keep : n;
  q.add = a.add != nullptr ? add : n > 0 ? 1 : 0;
  ok = parent >= -1 && parent < a.B_in && pg_len_ok(a, len) && q.keep >= 0 && q.keep <= n && q.add >= 0 &&
       q.add <= kPgLongest && pg_len_ok(a, (int)min((int64_t)q.keep + q.add, (int64_t)kPgLongest + 1));
  if (!ok) {
    q.parent = -1;
    q.keep = q.add = 0;
  }
  return q;
}
__device__ __forceinline__ PgSeq pg_seq(const PagesForkArgs& a, int b, bool& ok) {
  const int parent = pg_parent(a, b), keep = a.keep != nullptr ? a.keep[b] : 0;
  const int add = a.add != nullptr ? a.add[b] : 0;
  const int len = parent >= 0 && parent < a.B_in ? a.len[parent] : 0;
  return pg_seq_of(a, parent, len, keep, add, ok);
}
// Whether the sequence goes on writing a page that holds tokens already.
__device__ __forceinline__ bool pg_writes(const PagesForkArgs& a, const PgSeq& q) {
  return (q.keep & ((1 << a.page_log2) - 1)) != 0 && q.add > 0;
}

// ---------------------------------------------------------------------------
// Fork, in three launches.
// 1. What the change adds to and takes from the counts: a sequence that goes on in its
//    own row gives up what it does not keep; another row is given up whole, and taken up
//    by its continuations.  And who writes where: per page the number of sequences that
//    will, and the first of them; and which pages are kept, so that none of them is handed
//    out if its count is wrong.
// 2. Which pages are free then (listed, a chunk of pages by a block), and what each
//    sequence needs: pages past its last, and one for the page that it would write and
//    that others hold too (if all holders write, the first keeps it).
// 3. The counts, and the new entries of the tables: free pages in order.  (What is kept is
//    in them since the first launch.)
// No order of threads reaches the result: sums, a maximum, and ranks.  Bound: the chain of
// each launch (lookups of parent, length, entries; then the lists; then a page's place):
// 1024 sequences of up to 4096 tokens, 45000 pages, 5.0 + 5.0 + 4.7 us for 1.5 MB (without
// the marks of the kept pages 4.8 + 3.9 + 4.8).
// ---------------------------------------------------------------------------
struct PgWork {  // the workspace
  int* free_in;   // [chunks] free pages of a chunk
  int* need_in;   // [plans] pages that a block's sequences need
  int* need;      // [B] of a sequence
  int* before;    // [B] needs of the sequences before it in its block
  int* keep;      // [B] as the plan has them
  int* add;
  int* copy;      // [B] page that is copied (-1: none)
  int* free_ids;  // [chunks][kPgChunk]
  int chunks, plans;
};
__host__ __device__ inline PgWork pg_work(void* ws, int n_pages, int B) {
  PgWork w;
  w.chunks = (n_pages + kPgChunk - 1) / kPgChunk;
  w.plans = (B + kPgSeqs - 1) / kPgSeqs;
  int* p = (int*)ws;
  w.free_in = p; p += w.chunks;
  w.need_in = p; p += w.plans;
  w.need = p; p += B;
  w.before = p; p += B;
  w.keep = p; p += B;
  w.add = p; p += B;
  w.copy = p; p += B;
  w.free_ids = p;
  return w;
}
// counters: [n_pages] change of the count, [n_pages] writers, [n_pages] B - first writer,
// [n_pages] bytes: 1 where a sequence of the result keeps the page
__device__ __forceinline__ int* pg_change(const PagesForkArgs& a) { return a.counters; }
__device__ __forceinline__ int* pg_writers(const PagesForkArgs& a) { return a.counters + a.n_pages; }
__device__ __forceinline__ int* pg_first(const PagesForkArgs& a) {
  return a.counters + 2 * (int64_t)a.n_pages;
}
__device__ __forceinline__ uint8_t* pg_held(const PagesForkArgs& a) {
  return reinterpret_cast<uint8_t*>(a.counters + 3 * (int64_t)a.n_pages);
}

// A row gives up page o and its new sequence takes up page p (where they do).  A page of
// both changes nothing: most of a prompt is shared by the beams of a request.  bad: an id
// that is none.
__device__ __forceinline__ void pg_change_of(const PagesForkArgs& a, int o, bool gives, int p, bool takes,
                                             int* change, bool& bad) {
  const bool is_o = (unsigned)o < (unsigned)a.n_pages, is_p = (unsigned)p < (unsigned)a.n_pages;
  bad |= (gives & !is_o) | (takes & !is_p);
  const bool same = gives & takes & (o == p);
  if (gives & is_o & !same) atomicAdd(change + o, -1);
  if (takes & is_p & !same) atomicAdd(change + p, 1);
}

// wave (row, part): what old row `row` gives up and new sequence `row` takes up
__global__ __launch_bounds__(256) void k_pages_change(PagesForkArgs a, int parts) {
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int row = (int)(id / parts), part = (int)(id % parts), lane = threadIdx.x & 63;
  const int rows = max(a.B, a.B_in);
  if (row >= rows) return;
  const int i0 = part * kPgSpan, i1 = i0 + kPgSpan;
  PgSeq q{-1, 0, 0};
  if (row < a.B) {
    bool ok;
    q = pg_seq(a, row, ok);
    if (!ok && part == 0 && lane == 0) flag_dev_err(a.err, kDevErrPagePlan);
  }
  const int kept = q.parent >= 0 ? pg_pages(a.page_log2, q.keep) : 0;
  int held = 0;
  if (row < a.B_in) {
    held = pg_pages(a.page_log2, pg_len(a, row));
    if (part == 0 && lane == 0 && !pg_len_ok(a, a.len[row])) flag_dev_err(a.err, kDevErrPagePlan);
  }
  const int32_t* old = a.table + (int64_t)min(row, a.B_in - 1) * a.max_pages;
  const int32_t* now = a.table + (int64_t)max(q.parent, 0) * a.max_pages;
  const int from = q.parent == row ? min(kept, held) : 0;
  int32_t* out = a.table_out + (int64_t)min(row, a.B - 1) * a.max_pages;
  const bool moves = now != out && kept > 0;  // the kept entries into a table of their own
  const int end = min(i1, max(held, kept));
  if (end > i0) {
    // (inside the row whatever i is: a load under a condition of its own is waited for)
    int o[kPgSpan / 64], p[kPgSpan / 64];
#pragma unroll
    for (int u = 0; u < kPgSpan / 64; ++u) {
      const int i = min(i0 + 64 * u + lane, a.max_pages - 1);
      o[u] = old[i];
      p[u] = now[i];
    }
    if (moves) {
#pragma unroll
      for (int u = 0; u < kPgSpan / 64; ++u)
        if (i0 + 64 * u + lane < min(end, kept)) out[i0 + 64 * u + lane] = p[u];
    }
#pragma unroll
    for (int u = 0; u < kPgSpan / 64; ++u)
      if (i0 + 64 * u + lane < min(end, kept) && (unsigned)p[u] < (unsigned)a.n_pages) pg_held(a)[p[u]] = 1;
    if (from < end) {
      bool bad = false;
#pragma unroll
      for (int u = 0; u < kPgSpan / 64; ++u) {
        const int i = i0 + 64 * u + lane;
        pg_change_of(a, o[u], (i >= from) & (i < min(end, held)), p[u],
                     (i < min(end, kept)) & (q.parent != row), pg_change(a), bad);
      }
      if (bad) flag_dev_err(a.err, kDevErrPageId);
    }
  }
  if (q.parent >= 0 && pg_writes(a, q) && part == 0 && lane == 0) {
    const int p = now[kept - 1];
    if ((unsigned)p < (unsigned)a.n_pages) {
      atomicAdd(pg_writers(a) + p, 1);
      atomicMax(pg_first(a) + p, a.B - row);
    } else {
      flag_dev_err(a.err, kDevErrPageId);
    }
  }
}

// sums over the wave's lanes up to and with each
template <int CTRL, int ROWS>
__device__ __forceinline__ int pg_add_from(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int pg_wave_scan(int x) {
  x = pg_add_from<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
  x = pg_add_from<0x112, 0xF>(x);
  x = pg_add_from<0x114, 0xF>(x);
  x = pg_add_from<0x118, 0xF>(x);
  x = pg_add_from<0x142, 0xA>(x);     // a row's last lane into the next row
  return pg_add_from<0x143, 0xC>(x);  // lane 31 into the upper half
}
// Before every flag j of a thread, how many are set: the order is j, then the thread (so
// page j blockDim + thread: loads and stores of a j lie side by side).  Gives the number of
// all.  sums: LDS, 128 of them, not in use before.
template <int J, int WAVES>
__device__ __forceinline__ int pg_ranks(const bool (&is)[J], int (&rank)[J], int* sums) {
  static_assert(J * WAVES <= 128, "two of a lane");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint64_t in = __ballot(is[j]);
    rank[j] = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
    if (lane == 0) sums[j * WAVES + wave] = __builtin_popcountll(in);
  }
  __syncthreads();
  const int a = 2 * lane < J * WAVES ? sums[2 * lane] : 0, b = 2 * lane + 1 < J * WAVES ? sums[2 * lane + 1] : 0;
  const int to = pg_wave_scan(a + b);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int at = j * WAVES + wave;
    const int before = __builtin_amdgcn_ds_bpermute(4 * (at >> 1), to - b - ((at & 1) == 0 ? a : 0));
    rank[j] += before;
  }
  return __builtin_amdgcn_readlane(to, 63);
}
// exclusive sum over the block of WAVES waves; all: the total.  sums: LDS, WAVES of them
template <int WAVES>
__device__ __forceinline__ int pg_block_scan(int v, int* sums, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = pg_wave_scan(v);
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  const int to = pg_wave_scan(lane < WAVES ? sums[lane] : 0);
  all = __builtin_amdgcn_readlane(to, 63);
  const int before = __builtin_amdgcn_readlane(to, __builtin_amdgcn_readfirstlane(max(wave - 1, 0)));
  return (wave > 0 ? before : 0) + x - v;
}

// A page's holders: its count after the change, and no fewer than go on writing it, or than
// one that keeps it (a count that says less is wrong: the page is neither free nor written
// by two).  Of these `least` are known.
__device__ __forceinline__ int pg_least(int writers, int held) { return max(writers, held); }
__device__ __forceinline__ int pg_holders(int count, int least) {
  return least > 0 ? max(count, least) : count;
}

__global__ __launch_bounds__(256) void k_pages_plan(PagesForkArgs a) {
  __shared__ int waves[4];
  const PgWork w = pg_work(a.workspace, a.n_pages, a.B);
  int all;
  if ((int)blockIdx.x < w.chunks) {
    // the chunk's free pages, in order
    __shared__ int sums[16];
    bool is[4];
    int rank[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = blockIdx.x * kPgChunk + 256 * j + threadIdx.x;
      const int r = p < a.n_pages ? a.refs[p] + pg_change(a)[p] : 1;
      const int least = p < a.n_pages ? pg_least(pg_writers(a)[p], pg_held(a)[p]) : 0;
      if (r < least) flag_dev_err(a.err, kDevErrPagePlan);
      is[j] = pg_holders(r, least) == 0;
    }
    all = pg_ranks<4, 4>(is, rank, sums);
    int* ids = w.free_ids + (int64_t)blockIdx.x * kPgChunk;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is[j]) ids[rank[j]] = blockIdx.x * kPgChunk + 256 * j + threadIdx.x;
    if (threadIdx.x == 0) w.free_in[blockIdx.x] = all;
    return;
  }
  const int plan = blockIdx.x - w.chunks;
  const int b = plan * kPgSeqs + threadIdx.x;
  int need = 0;
  if (b < a.B) {
    bool ok;
    const PgSeq q = pg_seq(a, b, ok);
    const int kept = pg_pages(a.page_log2, q.keep);
    need = pg_pages(a.page_log2, q.keep + q.add) - kept;
    int copy = -1;
    if (pg_writes(a, q)) {
      const int p = a.table[(int64_t)q.parent * a.max_pages + kept - 1];
      if ((unsigned)p < (unsigned)a.n_pages) {
        const int k = pg_writers(a)[p], r = pg_holders(a.refs[p] + pg_change(a)[p], k);
        const bool mine = r == k && pg_first(a)[p] == a.B - b;
        if (r > 1 && !mine) {
          copy = p;
          ++need;
        }
      }
    }
    w.need[b] = need;
    w.keep[b] = q.keep;
    w.add[b] = q.add;
    w.copy[b] = copy;
  }
  const int before = pg_block_scan<4>(need, waves, all);
  if (b < a.B) w.before[b] = before;
  if (threadIdx.x == 0) w.need_in[plan] = all;
}

// sum of n numbers, by the wave (of pages or of table entries: 32 bits)
__device__ __forceinline__ int pg_wave_total(const int* v, int n) {
  const int lane = threadIdx.x & 63;
  int s = 0;
  for (int i = lane; i < n; i += 64) s += v[i];
  return __builtin_amdgcn_readlane(pg_wave_scan(s), 63);
}

// What the count of a page of r holders becomes: `rank` is the place of a free one, k
// sequences would go on writing it, and all that get a copy leave.
__device__ __forceinline__ int pg_count(int r, int rank, int taken, int k) {
  if (r == 0) return rank < taken ? 1 : 0;
  return k > 0 && r > 1 ? r - (r == k ? k - 1 : k) : r;
}
// blocks 0 .. chunks - 1: the counts; then waves (sequence, part of its row): the new
// entries
__global__ __launch_bounds__(256) void k_pages_apply(PagesForkArgs a, int parts) {
  const PgWork w = pg_work(a.workspace, a.n_pages, a.B);
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x < w.chunks) {
    __shared__ int sums[16];
    const int taken = pg_wave_total(w.need_in, w.plans);
    const int before = pg_wave_total(w.free_in, blockIdx.x);
    int r[4], k[4], rank[4];
    bool is[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = blockIdx.x * kPgChunk + 256 * j + threadIdx.x;
      k[j] = p < a.n_pages ? pg_writers(a)[p] : 0;
      r[j] = p < a.n_pages ? pg_holders(a.refs[p] + pg_change(a)[p], pg_least(k[j], pg_held(a)[p])) : 1;
      is[j] = r[j] == 0;
    }
    pg_ranks<4, 4>(is, rank, sums);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = blockIdx.x * kPgChunk + 256 * j + threadIdx.x;
      if (p >= a.n_pages) break;
      a.refs_out[p] = pg_count(r[j], before + rank[j], taken, k[j]);
      pg_change(a)[p] = 0;
      pg_writers(a)[p] = 0;
      pg_first(a)[p] = 0;
      pg_held(a)[p] = 0;
    }
    return;
  }
  const int64_t id = ((int64_t)blockIdx.x - w.chunks) * 4 + (threadIdx.x >> 6);
  const int b = (int)(id / parts), part = (int)(id % parts);
  if (b >= a.B) return;
  const int keep = w.keep[b], add = w.add[b], copy = w.copy[b];
  const int goal = pg_pages(a.page_log2, keep + add);
  const int old_end = pg_pages(a.page_log2, keep) - (copy >= 0 ? 1 : 0);
  int32_t* out = a.table_out + (int64_t)b * a.max_pages;
  const int i0 = part * kPgSpan, i1 = min(i0 + kPgSpan, goal);
  if (part == 0 && lane == 0) {
    a.len_out[b] = keep + add;
    a.copy_src[b] = copy;
    a.copy_rows[b] = copy >= 0 ? keep & ((1 << a.page_log2) - 1) : 0;
    if (copy < 0) a.copy_dst[b] = -1;
  }
  if (i1 <= old_end || i0 >= goal) return;
  const int first = pg_wave_total(w.need_in, b / kPgSeqs) + w.before[b];
  const int n_free = pg_wave_total(w.free_in, w.chunks);
  for (int ib = max(i0, old_end); ib < i1; ib += 64) {
    const int i = ib + lane;
    const int j = first + (i - old_end);
    // the chunk that holds the j-th free page, chunks 64 at a time
    int id2 = -1;
    const bool mine = i < i1 && j < n_free;
    int from = 0;
    for (int c0 = 0; c0 < w.chunks && __any(mine && j >= from); c0 += 64) {
      const int in = c0 + lane < w.chunks ? w.free_in[c0 + lane] : 0;
      const int to = pg_wave_scan(in), all = __builtin_amdgcn_readlane(to, 63);
      const bool now = mine && j >= from && j < from + all;
      const int want = now ? j - from : 0;
      int c = 0;  // the first of the 64 sums above it
#pragma unroll
      for (int step = 32; step > 0; step >>= 1) {
        const int upto = __builtin_amdgcn_ds_bpermute(4 * (c + step - 1), to);
        c += upto <= want ? step : 0;
      }
      const int before = __builtin_amdgcn_ds_bpermute(4 * c, to - in);
      if (now) id2 = w.free_ids[(int64_t)(c0 + c) * kPgChunk + want - before];
      from += all;
    }
    if (i < i1) {
      if (!mine) flag_dev_err(a.err, kDevErrPagesFull);
      out[i] = id2;
      if (copy >= 0 && i == old_end) a.copy_dst[b] = id2;
    }
  }
}

// ---------------------------------------------------------------------------
// The same for small pools and few sequences in one launch of one block: counts, writers
// and free pages in LDS, a thread per sequence and eight pages a thread.
// Bound: the chain of loads of a row, a wave's four rows in two pairs one after another (4.6
// us of the 9.6 that 64 beams of up to 8192 tokens take), and the host: in a graph 4 / 64 /
// 128 / 256 rows take 5.8 / 9.9 to 10.5 / 15 / 24 us against 8.2 / 10.4 to 11.4 / 11.6 / 11.7
// in three launches, and a call is enqueued in 9 us against 13.  (64 rows of 4003 tokens grown
// in place: 8.8; their kept entries are read only so that no page among them is handed out,
// 6.8 without.)
// ---------------------------------------------------------------------------
constexpr int kPgOneThreads = 1024;
constexpr int kPgOnePages = 8 * kPgOneThreads;
constexpr int kPgOneEntries = 65536;  // table entries: B max_pages at most
constexpr int kPgOneRows = 64;        // of the fork
constexpr int kPcOneRows = 256;       // of the compaction

__global__ __launch_bounds__(kPgOneThreads) void k_pages_fork_one(PagesForkArgs a) {
  __shared__ int count[kPgOnePages], writers[kPgOnePages], first[kPgOnePages];
  __shared__ uint16_t free_ids[kPgOnePages];
  __shared__ uint8_t keeps[kPgOnePages];  // 1 where a sequence of the result keeps the page
  __shared__ int s_parent[kPgOneThreads], s_kept[kPgOneThreads], s_held[kPgOneThreads];
  __shared__ int s_goal[kPgOneThreads], s_before[kPgOneThreads];
  __shared__ int sums[2][128];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = tid;
  // all that depends on nothing, in one round trip
  int r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = 1024 * j + tid < a.n_pages ? a.refs[1024 * j + tid] : 1;
  const int len = b < a.B_in ? a.len[b] : 0;
  const int parent = b < a.B ? pg_parent(a, b) : -1;
  const int keep = b < a.B && a.keep != nullptr ? a.keep[b] : 0;
  const int add = b < a.B && a.add != nullptr ? a.add[b] : 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (1024 * j + tid < a.n_pages) {
      count[1024 * j + tid] = r[j];
      writers[1024 * j + tid] = first[1024 * j + tid] = 0;
      keeps[1024 * j + tid] = 0;
    }
  s_held[tid] = len;
  __syncthreads();
  PgSeq q{-1, 0, 0};
  if (b < a.B) {
    bool ok;
    q = pg_seq_of(a, parent, parent >= 0 && parent < a.B_in ? s_held[parent] : 0, keep, add, ok);
    if (!ok) flag_dev_err(a.err, kDevErrPagePlan);
  }
  if (!pg_len_ok(a, len)) flag_dev_err(a.err, kDevErrPagePlan);
  const int kept = q.parent >= 0 ? pg_pages(a.page_log2, q.keep) : 0;
  s_parent[tid] = q.parent;
  s_kept[tid] = kept;
  __syncthreads();  // (lengths are read)
  s_held[tid] = pg_len_ok(a, len) ? pg_pages(a.page_log2, len) : 0;
  __syncthreads();
  const bool writes = q.parent >= 0 && pg_writes(a, q);
  int page = writes ? a.table[(int64_t)q.parent * a.max_pages + kept - 1] : -1;
  // a wave takes two rows at a time: their changes, and the kept entries into the new table
  const int rows = max(a.B, a.B_in);
  bool bad = false;
  struct Row {
    const int32_t *old, *now;
    int32_t* out;
    int k, held, from, i0, end;
    bool moves, own;
    int o[4], p[4];
  };
  auto open_row = [&](Row& w, int row) {
    const bool has = row < rows;
    const int par = has ? __builtin_amdgcn_readfirstlane(s_parent[row]) : -1;
    w.k = has ? __builtin_amdgcn_readfirstlane(s_kept[row]) : 0;
    w.held = has ? __builtin_amdgcn_readfirstlane(s_held[row]) : 0;
    w.old = a.table + (int64_t)min(row, a.B_in - 1) * a.max_pages;
    w.now = a.table + (int64_t)max(par, 0) * a.max_pages;
    w.out = a.table_out + (int64_t)min(row, a.B - 1) * a.max_pages;
    w.own = par == row;
    w.from = w.own ? min(w.k, w.held) : 0;
    w.moves = w.now != w.out && w.k > 0;
    w.i0 = 0;
    w.end = max(w.held, w.k);
  };
  auto load = [&](Row& w) {
    // (inside the row whatever i is: a load under a condition of its own is waited for)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(w.i0 + 64 * u + lane, a.max_pages - 1);
      w.o[u] = w.old[i];
      w.p[u] = w.now[i];
    }
  };
  auto use = [&](Row& w) {
    if (w.moves) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (w.i0 + 64 * u + lane < w.k) w.out[w.i0 + 64 * u + lane] = w.p[u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (w.i0 + 64 * u + lane < w.k && (unsigned)w.p[u] < (unsigned)a.n_pages) keeps[w.p[u]] = 1;
    if (w.from < w.end) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = w.i0 + 64 * u + lane;
        pg_change_of(a, w.o[u], (i >= w.from) & (i < w.held), w.p[u], (i < w.k) & !w.own, count, bad);
      }
    }
    w.i0 += 256;
  };
  for (int row = wave; row < rows; row += 2 * (kPgOneThreads / 64)) {
    Row x, y;
    open_row(x, row);
    open_row(y, row + kPgOneThreads / 64);
    while (x.i0 < x.end || y.i0 < y.end) {
      if (x.i0 < x.end) load(x);
      if (y.i0 < y.end) load(y);
      if (x.i0 < x.end) use(x);
      if (y.i0 < y.end) use(y);
    }
  }
  if (writes && (unsigned)page >= (unsigned)a.n_pages) {
    bad = true;
    page = -1;
  }
  if (bad) flag_dev_err(a.err, kDevErrPageId);
  if (page >= 0) {
    atomicAdd(&writers[page], 1);
    atomicMax(&first[page], a.B - b);
  }
  __syncthreads();
  // free pages in order
  bool is[8];
  int rank[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = 1024 * j + tid;
    if (p < a.n_pages) {
      const int least = pg_least(writers[p], keeps[p]);
      if (count[p] < least) flag_dev_err(a.err, kDevErrPagePlan);
      r[j] = pg_holders(count[p], least);
    }
    is[j] = r[j] == 0;
  }
  const int n_free = pg_ranks<8, 16>(is, rank, sums[0]);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (is[j]) free_ids[rank[j]] = (uint16_t)(1024 * j + tid);
  // needs
  const int goal = pg_pages(a.page_log2, q.keep + q.add);
  int copy = -1, taken;
  if (page >= 0) {
    const int holders = pg_holders(count[page], writers[page]);
    if (holders > 1 && !(holders == writers[page] && first[page] == a.B - b)) copy = page;
  }
  const int old_end = kept - (copy >= 0 ? 1 : 0);
  const int before = pg_block_scan<16>(goal - old_end, sums[1], taken);
  s_goal[tid] = goal;
  s_before[tid] = before;
  s_kept[tid] = old_end;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = 1024 * j + tid;
    if (p < a.n_pages) a.refs_out[p] = pg_count(r[j], rank[j], taken, writers[p]);
  }
  if (b < a.B) {
    a.len_out[b] = q.keep + q.add;
    a.copy_src[b] = copy;
    a.copy_rows[b] = copy >= 0 ? q.keep & ((1 << a.page_log2) - 1) : 0;
    a.copy_dst[b] = copy >= 0 && before < n_free ? free_ids[before] : -1;
  }
  // the new entries: a wave's rows side by side while they are few
  for (int row0 = 64 * wave; row0 < a.B; row0 += kPgOneThreads) {
    const int row = row0 + lane, end = row < a.B ? s_goal[row] : 0, at = row < a.B ? s_kept[row] : 0;
    const int base = row < a.B ? s_before[row] : 0;
    uint64_t some = __ballot(end > at);
    const bool few = __ballot(end - at > 4) == 0;
    auto put = [&](int64_t r64, int i, int j) {
      int id = -1;
      if (j < n_free) id = free_ids[j];
      else flag_dev_err(a.err, kDevErrPagesFull);
      a.table_out[r64 * a.max_pages + i] = id;
    };
    if (few) {
      for (int i = at; i < end; ++i) put(row, i, base + i - at);
      continue;
    }
    for (; some != 0; some &= some - 1) {
      const int l = __builtin_ctzll(some);
      const int e = __builtin_amdgcn_readlane(end, l), f = __builtin_amdgcn_readlane(at, l);
      const int bs = __builtin_amdgcn_readlane(base, l);
      for (int i = f + lane; i < e; i += 64) put(row0 + l, i, bs + i - f);
    }
  }
}

static bool pages_one(int n_pages, int B, int most, int max_pages) {
  return n_pages <= kPgOnePages && B <= most && (int64_t)B * max_pages <= kPgOneEntries;
}
size_t pages_counters(int n_pages) { return (size_t)n_pages * 12 + ((size_t)n_pages + 3) / 4 * 4; }
static int64_t pages_parts(int max_pages) { return ((int64_t)max_pages + kPgSpan - 1) / kPgSpan; }
// All entries of a table count in 32 bits (what the sequences need is summed), and then
// the grids hold them too.
bool pages_fits(int B, int max_pages) { return (int64_t)B * max_pages < (int64_t)1 << 31; }
void launch_pages_fork(const PagesForkArgs& a, hipStream_t st) {
  const int parts = (int)pages_parts(a.max_pages);
  const int rows = a.B > a.B_in ? a.B : a.B_in;
  if (pages_one(a.n_pages, rows, kPgOneRows, a.max_pages)) {
    hipLaunchKernelGGL(k_pages_fork_one, dim3(1), dim3(kPgOneThreads), 0, st, a);
    return;
  }
  const int chunks = (a.n_pages + kPgChunk - 1) / kPgChunk, plans = (a.B + kPgSeqs - 1) / kPgSeqs;
  hipLaunchKernelGGL(k_pages_change, dim3((unsigned)(((int64_t)rows * parts + 3) / 4)), dim3(256), 0, st,
                     a, parts);
  hipLaunchKernelGGL(k_pages_plan, dim3((unsigned)(chunks + plans)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_pages_apply, dim3((unsigned)(chunks + ((int64_t)a.B * parts + 3) / 4)), dim3(256),
                     0, st, a, parts);
}

// ---------------------------------------------------------------------------
// Compaction, in three launches: with U pages in use, the used ones from id U on move
// to the free ids below U, both in their order, so that no page is read and written.
// 1. used pages of each chunk; 2. the lists, and what becomes of every page; 3. the
// counts and the tables.
// Bound: the chain of each launch: 131072 pages, 512 sequences, 2.4 + 5.0 + 5.6 us for
// 2.4 MB.
// ---------------------------------------------------------------------------
struct PcWork {
  int* used_in;   // [chunks]
  int* sums;      // U, and the used pages below id U
  int* high_ref;  // counts of the pages that move
  int* fate;      // [n_pages] kPcFree, kPcStays, or the number of its move
  int chunks;
};
constexpr int kPcFree = -1, kPcStays = -2;
__host__ __device__ inline PcWork pc_work(void* ws, int n_pages) {
  PcWork w;
  w.chunks = (n_pages + kPgChunk - 1) / kPgChunk;
  int* p = (int*)ws;
  w.sums = p; p += 2;
  w.used_in = p; p += w.chunks;
  w.high_ref = p; p += n_pages / 2;
  w.fate = p;
  return w;
}
static size_t pc_bytes(int n_pages) {
  return 4 * (2 + ((size_t)n_pages + kPgChunk - 1) / kPgChunk + (size_t)n_pages / 2 + (size_t)n_pages);
}

// the thread's four counts of a chunk (0 past the end), and which are of used pages
__device__ __forceinline__ void pc_load(const int32_t* refs, int n_pages, int chunk, int (&r)[4],
                                        bool (&is)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = chunk * kPgChunk + 256 * j + threadIdx.x;
    r[j] = p < n_pages ? refs[p] : 0;
    is[j] = r[j] != 0;
  }
}

__global__ __launch_bounds__(256) void k_pages_used(PagesCompactArgs a) {
  __shared__ int sums[16];
  const PcWork w = pc_work(a.workspace, a.n_pages);
  int r[4], rank[4];
  bool is[4];
  pc_load(a.refs, a.n_pages, blockIdx.x, r, is);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (r[j] < 0) flag_dev_err(a.err, kDevErrPagePlan);
  const int all = pg_ranks<4, 4>(is, rank, sums);
  if (threadIdx.x == 0) w.used_in[blockIdx.x] = all;
}

__global__ __launch_bounds__(256) void k_pages_lists(PagesCompactArgs a) {
  __shared__ int sums[16], sums2[16];
  const PcWork w = pc_work(a.workspace, a.n_pages);
  int r[4], u[4], rank[4], rank2[4];
  bool is[4], low_is[4];
  pc_load(a.refs, a.n_pages, blockIdx.x, r, is);
  const int before = pg_wave_total(w.used_in, blockIdx.x);
  const int U = pg_wave_total(w.used_in, w.chunks);
  // used pages below U: whole chunks, and those of U's own
  const int cu = U / kPgChunk;
  pc_load(a.refs, a.n_pages, cu, u, low_is);
#pragma unroll
  for (int j = 0; j < 4; ++j) low_is[j] &= cu * kPgChunk + 256 * j + (int)threadIdx.x < U;
  pg_ranks<4, 4>(is, rank, sums);
  const int low = pg_wave_total(w.used_in, cu) + pg_ranks<4, 4>(low_is, rank2, sums2);
  const int moves = U - low;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    w.sums[0] = U;
    w.sums[1] = low;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = blockIdx.x * kPgChunk + 256 * j + threadIdx.x;
    if (p >= a.n_pages) break;
    const int at = before + rank[j];  // used pages before it
    int fate = kPcFree;
    if (is[j]) {
      fate = p < U ? kPcStays : at - low;
      if (p >= U) {
        a.copy_src[fate] = p;
        w.high_ref[fate] = r[j];
      }
    } else if (p < U) {
      a.copy_dst[p - at] = p;  // as many free pages before it
    }
    w.fate[p] = fate;
    if (p >= moves && p < a.n_pages / 2) {
      a.copy_src[p] = -1;
      a.copy_dst[p] = -1;
    }
  }
}

// blocks 0 .. chunks - 1: the counts; then waves (sequence, part of its row)
__global__ __launch_bounds__(256) void k_pages_map(PagesCompactArgs a, int parts) {
  const PcWork w = pc_work(a.workspace, a.n_pages);
  if ((int)blockIdx.x < w.chunks) {
    __shared__ int sums[16];
    int r[4], rank[4];
    bool is[4];
    pc_load(a.refs, a.n_pages, blockIdx.x, r, is);
    const int U = w.sums[0];
    const int before = pg_wave_total(w.used_in, blockIdx.x);
    pg_ranks<4, 4>(is, rank, sums);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = blockIdx.x * kPgChunk + 256 * j + threadIdx.x;
      if (p >= a.n_pages) break;
      const int f = w.fate[p];
      a.moved_to[p] = f == kPcFree ? -1 : f == kPcStays ? p : a.copy_dst[f];
      a.refs_out[p] = p >= U ? 0 : is[j] ? r[j] : w.high_ref[p - before - rank[j]];
    }
    return;
  }
  const int64_t id = ((int64_t)blockIdx.x - w.chunks) * 4 + (threadIdx.x >> 6);
  const int b = (int)(id / parts), part = (int)(id % parts), lane = threadIdx.x & 63;
  if (b >= a.B) return;
  const int len = a.len[b];
  if (len < 0 || len > kPgLongest || (int64_t)len > (int64_t)a.max_pages << a.page_log2) {
    if (part == 0 && lane == 0) flag_dev_err(a.err, kDevErrPagePlan);
    return;
  }
  const int i0 = part * kPgSpan, i1 = min(i0 + kPgSpan, pg_pages(a.page_log2, len));
  for (int i = i0 + lane; i < i1; i += 64) {
    const int64_t at = (int64_t)b * a.max_pages + i;
    const int p = a.table[at];
    int to = p;
    if ((unsigned)p >= (unsigned)a.n_pages) {
      flag_dev_err(a.err, kDevErrPageId);
    } else {
      const int f = w.fate[p];
      if (f == kPcFree) flag_dev_err(a.err, kDevErrPagePlan);
      to = f == kPcFree ? -1 : f == kPcStays ? p : a.copy_dst[f];
    }
    a.table_out[at] = to;
  }
}

// The same for small pools and few sequences, in one launch of one block: in a graph 4 /
// 64 / 250 / 1000 sequences take 3.9 / 6.2 to 7.6 / 9.4 / 19 us against 7.1 / 10 to 11 /
// 9.5 / 9.5 in three launches, and a call is enqueued in 7.2 us against 12.
__global__ __launch_bounds__(kPgOneThreads) void k_pages_compact_one(PagesCompactArgs a) {
  __shared__ int fate[kPgOnePages];                                 // new id, -1: free
  __shared__ uint16_t high[kPgOnePages / 2], low[kPgOnePages / 2];  // ids that move, and where to
  __shared__ int high_ref[kPgOnePages / 2];
  __shared__ int held[kPgOneThreads];
  __shared__ int sums[2][128];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int r[8], rank[8];
  bool is[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = 1024 * j + tid < a.n_pages ? a.refs[1024 * j + tid] : 0;
  const int len = tid < a.B ? a.len[tid] : 0;
  const bool fits = len >= 0 && len <= kPgLongest && (int64_t)len <= (int64_t)a.max_pages << a.page_log2;
  if (!fits) flag_dev_err(a.err, kDevErrPagePlan);
  held[tid] = fits ? pg_pages(a.page_log2, len) : 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (r[j] < 0) flag_dev_err(a.err, kDevErrPagePlan);
    is[j] = r[j] != 0;
  }
  const int U = pg_ranks<8, 16>(is, rank, sums[0]);
  int below = 0, n_low;
#pragma unroll
  for (int j = 0; j < 8; ++j) below += is[j] && 1024 * j + tid < U;
  pg_block_scan<16>(below, sums[1], n_low);
  const int moves = U - n_low;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = 1024 * j + tid;
    if (p >= a.n_pages) break;
    if (is[j] && p >= U) {
      high[rank[j] - n_low] = (uint16_t)p;
      high_ref[rank[j] - n_low] = r[j];
    }
    if (!is[j] && p < U) low[p - rank[j]] = (uint16_t)p;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = 1024 * j + tid;
    if (p >= a.n_pages) break;
    const int to = !is[j] ? -1 : p < U ? p : low[rank[j] - n_low];
    fate[p] = to;
    a.moved_to[p] = to;
    a.refs_out[p] = p >= U ? 0 : is[j] ? r[j] : high_ref[p - rank[j]];
  }
  for (int i = tid; i < a.n_pages / 2; i += kPgOneThreads) {
    a.copy_src[i] = i < moves ? high[i] : -1;
    a.copy_dst[i] = i < moves ? low[i] : -1;
  }
  __syncthreads();
  for (int row = wave; row < a.B; row += kPgOneThreads / 64) {
    const int64_t at = (int64_t)row * a.max_pages;
    const int end = __builtin_amdgcn_readfirstlane(held[row]);
    for (int i0 = 0; i0 < end; i0 += 256) {
      int p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = a.table[at + min(i0 + 64 * u + lane, end - 1)];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i0 + 64 * u + lane >= end) break;
        int to = p[u];
        if ((unsigned)to >= (unsigned)a.n_pages) {
          flag_dev_err(a.err, kDevErrPageId);
        } else {
          to = fate[to];
          if (to < 0) flag_dev_err(a.err, kDevErrPagePlan);
        }
        a.table_out[at + i0 + 64 * u + lane] = to;
      }
    }
  }
}

void launch_pages_compact(const PagesCompactArgs& a, hipStream_t st) {
  if (pages_one(a.n_pages, a.B, kPcOneRows, a.max_pages)) {
    hipLaunchKernelGGL(k_pages_compact_one, dim3(1), dim3(kPgOneThreads), 0, st, a);
    return;
  }
  const int parts = (int)pages_parts(a.max_pages);
  const unsigned chunks = (unsigned)((a.n_pages + kPgChunk - 1) / kPgChunk);
  hipLaunchKernelGGL(k_pages_used, dim3(chunks), dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_pages_lists, dim3(chunks), dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_pages_map, dim3((unsigned)(chunks + ((int64_t)a.B * parts + 3) / 4)), dim3(256), 0,
                     st, a, parts);
}

size_t pages_workspace(int n_pages, int B) {
  const size_t chunks = ((size_t)n_pages + kPgChunk - 1) / kPgChunk;
  const size_t plans = ((size_t)B + kPgSeqs - 1) / kPgSeqs;
  const size_t fork = 4 * (chunks + plans + 5 * (size_t)B + chunks * kPgChunk);
  return fork > pc_bytes(n_pages) ? fork : pc_bytes(n_pages);
}

// ---------------------------------------------------------------------------
// Copy.  A block takes one 16-byte unit per thread of a page, in one pool, for 64
// entries of the list: the entries that are none cost a load and a ballot.  One launch
// serves up to 64 caches.
// Bound: the bytes read and written: 600 pages of 256 KB in two layers, 1.26 GB, 257 us,
// 4.89 TB/s; the first rows of 20 pages in 24 layers, 77 MB, 17 us.
// ---------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ void pg_copy_units(const PagesCopyArgs& a, uint8_t* pool, int64_t page_units,
                                              int row_units, int64_t unit, uint64_t has, int src, int dst,
                                              int rows) {
  T* p = reinterpret_cast<T*>(pool) + unit;
  const bool in = unit < page_units;
  const int row = in ? (int)(unit / row_units) & ((1 << a.kv.page_log2) - 1) : 0;
  while (has != 0) {
    const int e = __builtin_ctzll(has);
    has &= has - 1;
    const int s = __builtin_amdgcn_readlane(src, e), d = __builtin_amdgcn_readlane(dst, e);
    const int n = __builtin_amdgcn_readlane(rows, e);
    if (in && row < n) stream_store(p + (int64_t)d * page_units, p[(int64_t)s * page_units]);
  }
}

constexpr int kPgList = 64;  // entries of a block
__global__ __launch_bounds__(256) void k_pages_copy(PagesCopyArgs a, int n_kv, int parts, int scale_parts) {
  const int per = 2 * (parts + scale_parts);  // blocks of a cache and 64 entries
  int id = blockIdx.x;
  const int sub = id % per;
  id /= per;
  const int layer = id % n_kv, e0 = id / n_kv * kPgList;
  const int lane = threadIdx.x & 63, e = e0 + lane, page = 1 << a.kv.page_log2;
  int src = -1, dst = -1, rows = 0;
  if (e < a.n) {
    src = a.src[e];
    dst = a.dst[e];
    rows = a.rows != nullptr ? a.rows[e] : page;
    const bool none = src == -1 || dst == -1;
    const bool bad = (unsigned)src >= (unsigned)a.kv.n_pages || (unsigned)dst >= (unsigned)a.kv.n_pages ||
                     rows < 0 || rows > page;
    if (bad && !none && layer == 0 && sub == 0 && threadIdx.x < 64) flag_dev_err(a.err, kDevErrPageId);
    if (bad || none) rows = 0;
  }
  const uint64_t has = __ballot(rows > 0);
  if (has == 0) return;
  const bool scale = sub >= 2 * parts;
  const int x = scale ? 2 + (sub - 2 * parts) / scale_parts : sub / parts;
  const int part = scale ? (sub - 2 * parts) % scale_parts : sub % parts;
  const int64_t unit = (int64_t)part * 256 + threadIdx.x;
  const int64_t head_rows = (int64_t)a.kv.Hkv << a.kv.page_log2;
  uint8_t* pool = a.pool[layer][x];
  if (!scale) {
    const int row_units = (a.kv.ks != nullptr ? a.kv.D / 2 : a.kv.D * 2) / 16;
    pg_copy_units<uint4>(a, pool, head_rows * row_units, row_units, unit, has, src, dst, rows);
  } else if (a.kv.D == 64) {
    pg_copy_units<uint16_t>(a, pool, head_rows, 1, unit, has, src, dst, rows);
  } else {
    pg_copy_units<uint32_t>(a, pool, head_rows, 1, unit, has, src, dst, rows);
  }
}

static void copy_parts(const PagedKv& kv, int64_t& parts, int64_t& scale_parts) {
  const int64_t rows = (int64_t)kv.Hkv << kv.page_log2;
  const bool f4 = kv.ks != nullptr;
  parts = (rows * ((f4 ? kv.D / 2 : kv.D * 2) / 16) + 255) / 256;
  scale_parts = f4 ? (rows + 255) / 256 : 0;
}
bool pages_copy_fits(const PagedKv& kv, int n) {
  int64_t parts, scale_parts;
  copy_parts(kv, parts, scale_parts);
  return 2 * (parts + scale_parts) * (((int64_t)n + kPgList - 1) / kPgList) < 1 << 24;
}
void launch_pages_copy(PagesCopyArgs a, const PagedKv* kv, int n_kv, hipStream_t st) {
  int64_t parts, scale_parts;
  copy_parts(kv[0], parts, scale_parts);
  a.kv = kv[0];
  const int64_t blocks = 2 * (parts + scale_parts) * (((int64_t)a.n + kPgList - 1) / kPgList);  // of a cache
  const int most = (int)std::min<int64_t>(kPagesLayers, ((1 << 24) - 1) / blocks);
  for (int x0 = 0, m; x0 < n_kv; x0 += m) {
    m = std::min(n_kv - x0, most);
    for (int x = 0; x < m; ++x) {
      a.pool[x][0] = kv[x0 + x].k; a.pool[x][1] = kv[x0 + x].v;
      a.pool[x][2] = kv[x0 + x].ks; a.pool[x][3] = kv[x0 + x].vs;
    }
    hipLaunchKernelGGL(k_pages_copy, dim3((unsigned)(blocks * m)), dim3(256), 0, st, a, m, (int)parts,
                       (int)scale_parts);
  }
}

}  // namespace neon
