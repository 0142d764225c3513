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
// ok: false where the numbers are none; the sequence is then left without tokens
__device__ __forceinline__ PgSeq pg_seq(const PagesForkArgs& a, int b, bool& ok) {
  PgSeq q;
  ok = true;
  q.parent = a.parent != nullptr ? a.parent[b] : b;
  if (q.parent < -1 || q.parent >= a.B_in) {
    ok = false;
    q.parent = -1;
  }
  const int raw = q.parent >= 0 ? a.len[q.parent] : 0;
  ok &= pg_len_ok(a, raw);
  const int n = pg_len_ok(a, raw) ? raw : 0;
  q.keep = a.keep != nullptr && q.parent >= 0 ? a.keep[b] : n;
  q.add = a.add != nullptr ? a.add[b] : n > 0 ? 1 : 0;
  ok &= q.keep >= 0 && q.keep <= n && q.add >= 0 && q.add <= kPgLongest &&
        pg_len_ok(a, (int)min((int64_t)q.keep + q.add, (int64_t)kPgLongest + 1));
  if (!ok) {
    q.parent = -1;
    q.keep = q.add = 0;
  }
  return q;
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
//    will, and the first of them.
// 2. Which pages are free then (listed, a chunk of pages by a block), and what each
//    sequence needs: pages past its last, and one for the page that it would write and
//    that others hold too (if all holders write, the first keeps it).
// 3. The counts; the tables: what is kept, then free pages in order.
// ---------------------------------------------------------------------------
struct PgWork {  // the workspace
  int* free_in;   // [chunks] free pages of a chunk
  int* need_in;   // [plans] pages that a block's sequences need
  int* need;      // [B] of a sequence
  int* before;    // [B] needs of the sequences before it in its block
  int* keep;      // [B] as the plan has them
  int* add;
  int* parent;
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
  w.parent = p; p += B;
  w.copy = p; p += B;
  w.free_ids = p;
  return w;
}
// counters: [n_pages] change of the count, [n_pages] writers, [n_pages] B - first writer
__device__ __forceinline__ int* pg_change(const PagesForkArgs& a) { return a.counters; }
__device__ __forceinline__ int* pg_writers(const PagesForkArgs& a) { return a.counters + a.n_pages; }
__device__ __forceinline__ int* pg_first(const PagesForkArgs& a) {
  return a.counters + 2 * (int64_t)a.n_pages;
}

// wave (row, part): entries of old row `row` given up, then of new sequence `row` taken up
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
  const int kept = pg_pages(a.page_log2, q.keep);
  if (row < a.B_in) {
    const int held = pg_pages(a.page_log2, pg_len(a, row));
    const int from = q.parent == row ? kept : 0;
    if (part == 0 && lane == 0 && !pg_len_ok(a, a.len[row])) flag_dev_err(a.err, kDevErrPagePlan);
    for (int i = max(i0, from) + lane; i < min(i1, held); i += 64) {
      const int p = a.table[(int64_t)row * a.max_pages + i];
      if ((unsigned)p < (unsigned)a.n_pages) atomicAdd(pg_change(a) + p, -1);
      else flag_dev_err(a.err, kDevErrPageId);
    }
  }
  if (q.parent >= 0) {
    const int32_t* t = a.table + (int64_t)q.parent * a.max_pages;
    if (q.parent != row)
      for (int i = i0 + lane; i < min(i1, kept); i += 64) {
        const int p = t[i];
        if ((unsigned)p < (unsigned)a.n_pages) atomicAdd(pg_change(a) + p, 1);
        else flag_dev_err(a.err, kDevErrPageId);
      }
    if (pg_writes(a, q) && part == 0 && lane == 0) {
      const int p = t[kept - 1];
      if ((unsigned)p < (unsigned)a.n_pages) {
        atomicAdd(pg_writers(a) + p, 1);
        atomicMax(pg_first(a) + p, a.B - row);
      } else {
        flag_dev_err(a.err, kDevErrPageId);
      }
    }
  }
}

// exclusive sum over the block's 256 threads; all: the total
__device__ __forceinline__ int pg_block_scan(int v, int* waves, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) base += waves[w];
    all += waves[w];
  }
  return base + x - v;
}

__global__ __launch_bounds__(256) void k_pages_plan(PagesForkArgs a) {
  __shared__ int waves[4];
  const PgWork w = pg_work(a.workspace, a.n_pages, a.B);
  int all;
  if ((int)blockIdx.x < w.chunks) {
    // the chunk's free pages, in order
    const int p0 = blockIdx.x * kPgChunk + 4 * threadIdx.x;
    bool is[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + j;
      const int r = p < a.n_pages ? a.refs[p] + pg_change(a)[p] : 1;
      if (r < 0) flag_dev_err(a.err, kDevErrPagePlan);
      is[j] = r == 0;
      n += is[j];
    }
    int at = pg_block_scan(n, waves, all);
    int* ids = w.free_ids + (int64_t)blockIdx.x * kPgChunk;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is[j]) ids[at++] = p0 + j;
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
        const int r = a.refs[p] + pg_change(a)[p];
        const bool mine = r == pg_writers(a)[p] && pg_first(a)[p] == a.B - b;
        if (r > 1 && !mine) {
          copy = p;
          ++need;
        }
      }
    }
    w.need[b] = need;
    w.keep[b] = q.keep;
    w.add[b] = q.add;
    w.parent[b] = q.parent;
    w.copy[b] = copy;
  }
  const int before = pg_block_scan(need, waves, all);
  if (b < a.B) w.before[b] = before;
  if (threadIdx.x == 0) w.need_in[plan] = all;
}

// sum of n numbers, by the wave
__device__ __forceinline__ int64_t pg_wave_total(const int* v, int n) {
  const int lane = threadIdx.x & 63;
  int64_t s = 0;
  for (int i = lane; i < n; i += 64) s += v[i];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  return s;
}

// blocks 0 .. chunks - 1: the counts; then waves (sequence, part of its row)
__global__ __launch_bounds__(256) void k_pages_apply(PagesForkArgs a, int parts) {
  const PgWork w = pg_work(a.workspace, a.n_pages, a.B);
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x < w.chunks) {
    __shared__ int waves[4];
    const int64_t taken = pg_wave_total(w.need_in, w.plans);
    const int64_t free_before = pg_wave_total(w.free_in, blockIdx.x);
    const int p0 = blockIdx.x * kPgChunk + 4 * threadIdx.x;
    int r[4], n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + j;
      r[j] = p < a.n_pages ? a.refs[p] + pg_change(a)[p] : 1;
      n += r[j] == 0;
    }
    int all;
    int64_t at = free_before + pg_block_scan(n, waves, all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + j;
      if (p >= a.n_pages) break;
      const int k = pg_writers(a)[p];
      int out = r[j];
      if (r[j] == 0) out = at++ < taken ? 1 : 0;
      else if (k > 0 && r[j] > 1) out -= r[j] == k ? k - 1 : k;  // those that get a copy
      a.refs_out[p] = out;
      pg_change(a)[p] = 0;
      pg_writers(a)[p] = 0;
      pg_first(a)[p] = 0;
    }
    return;
  }
  const int64_t id = ((int64_t)blockIdx.x - w.chunks) * 4 + (threadIdx.x >> 6);
  const int b = (int)(id / parts), part = (int)(id % parts);
  if (b >= a.B) return;
  const int keep = w.keep[b], add = w.add[b], parent = w.parent[b], copy = w.copy[b];
  const int goal = pg_pages(a.page_log2, keep + add);
  const int old_end = pg_pages(a.page_log2, keep) - (copy >= 0 ? 1 : 0);
  int32_t* out = a.table_out + (int64_t)b * a.max_pages;
  const int i0 = part * kPgSpan, i1 = min(i0 + kPgSpan, goal);
  if (i0 < old_end && parent >= 0) {
    const int32_t* t = a.table + (int64_t)parent * a.max_pages;
    if (t != out)
      for (int i = i0 + lane; i < min(i1, old_end); i += 64) out[i] = t[i];
  }
  // (a sequence without an entry of its own in this part is done)
  if (part == 0 && lane == 0) {
    a.len_out[b] = keep + add;
    a.copy_src[b] = copy;
    a.copy_rows[b] = copy >= 0 ? keep & ((1 << a.page_log2) - 1) : 0;
    if (copy < 0) a.copy_dst[b] = -1;
  }
  if (i1 <= old_end || i0 >= goal) return;
  const int64_t first = pg_wave_total(w.need_in, b / kPgSeqs) + w.before[b];
  const int64_t n_free = pg_wave_total(w.free_in, w.chunks);
  for (int i = max(i0, old_end) + lane; i < i1; i += 64) {
    const int64_t j = first + i - old_end;
    int id2 = -1;
    if (j < n_free) {
      int64_t rest = j;
      int c = 0;
      while (rest >= w.free_in[c]) rest -= w.free_in[c++];
      id2 = w.free_ids[(int64_t)c * kPgChunk + rest];
    } else {
      flag_dev_err(a.err, kDevErrPagesFull);
    }
    out[i] = id2;
    if (copy >= 0 && i == old_end) a.copy_dst[b] = id2;
  }
}

// ---------------------------------------------------------------------------
// The same for small pools in one launch of one block: counts, writers and free pages in
// LDS, a thread per sequence and eight pages a thread.
// ---------------------------------------------------------------------------
constexpr int kPgOneThreads = 1024;
constexpr int kPgOnePages = 8 * kPgOneThreads;
constexpr int kPgOneEntries = 65536;  // table entries: B max_pages at most

// exclusive sum over a block of 1024 threads
__device__ __forceinline__ int pg_scan_one(int v, int* waves, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  const int w = waves[lane & 15];
  int base = lane < 16 && lane < wave ? w : 0;
  all = lane < 16 ? w : 0;
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) {
    base += __shfl_xor(base, d);
    all += __shfl_xor(all, d);
  }
  base = __builtin_amdgcn_readfirstlane(base);
  all = __builtin_amdgcn_readfirstlane(all);
  return base + x - v;
}
// eight counts of a thread
__device__ __forceinline__ void pg_load8(const int32_t* refs, int n_pages, int p0, int past, int (&r)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = p0 + j < n_pages ? refs[p0 + j] : past;
}

__global__ __launch_bounds__(kPgOneThreads) void k_pages_fork_one(PagesForkArgs a) {
  __shared__ int change[kPgOnePages], writers[kPgOnePages], first[kPgOnePages];
  __shared__ uint16_t free_ids[kPgOnePages];
  __shared__ int s_parent[kPgOneThreads], s_keep[kPgOneThreads], s_goal[kPgOneThreads];
  __shared__ int s_before[kPgOneThreads], s_copy[kPgOneThreads];
  __shared__ int waves[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int p0 = 8 * tid, b = tid;
  int r[8];
  pg_load8(a.refs, a.n_pages, p0, 1, r);
  for (int i = tid; i < a.n_pages; i += kPgOneThreads) change[i] = writers[i] = first[i] = 0;
  PgSeq q{-1, 0, 0};
  int held = 0;
  if (b < a.B) {
    bool ok;
    q = pg_seq(a, b, ok);
    if (!ok) flag_dev_err(a.err, kDevErrPagePlan);
  }
  if (b < a.B_in) {
    const int n = a.len[b];
    if (!pg_len_ok(a, n)) flag_dev_err(a.err, kDevErrPagePlan);
    held = pg_len_ok(a, n) ? pg_pages(a.page_log2, n) : 0;
  }
  const int kept = pg_pages(a.page_log2, q.keep);
  int page = -1;  // that the sequence goes on writing
  if (pg_writes(a, q)) page = a.table[(int64_t)q.parent * a.max_pages + kept - 1];
  if (q.parent >= 0 && pg_writes(a, q) && (unsigned)page >= (unsigned)a.n_pages) {
    flag_dev_err(a.err, kDevErrPageId);
    page = -1;
  }
  __syncthreads();
  if (page >= 0) {
    atomicAdd(&writers[page], 1);
    atomicMax(&first[page], a.B - b);
  }
  // a wave takes its 64 rows one after another, those with something to change
  auto count = [&](int row, int i0, int i1, int by) {
    const int32_t* t = a.table + (int64_t)row * a.max_pages;
    for (int i = i0 + lane; i < i1; i += 64) {
      const int p = t[i];
      if ((unsigned)p < (unsigned)a.n_pages) atomicAdd(&change[p], by);
      else flag_dev_err(a.err, kDevErrPageId);
    }
  };
  s_parent[tid] = q.parent;
  s_keep[tid] = kept;
  s_goal[tid] = held;
  __syncthreads();
  const int rows = max(a.B, a.B_in);
  for (int row = wave; row < rows; row += kPgOneThreads / 64) {
    const int par = s_parent[row], k = s_keep[row], h = s_goal[row];
    count(row, par == row ? k : 0, h, -1);
    if (par >= 0 && par != row) count(par, 0, k, 1);
  }
  __syncthreads();
  // free pages in order
  int n = 0, n_free;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (p0 + j < a.n_pages) r[j] += change[p0 + j];
    if (r[j] < 0) flag_dev_err(a.err, kDevErrPagePlan);
    n += r[j] == 0;
  }
  int at = pg_scan_one(n, waves[0], n_free);
  const int free_before = at;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (r[j] == 0) free_ids[at++] = (uint16_t)(p0 + j);
  // needs
  const int goal = pg_pages(a.page_log2, q.keep + q.add);
  int copy = -1, taken;
  if (page >= 0) {
    const int holders = a.refs[page] + change[page];
    if (holders > 1 && !(holders == writers[page] && first[page] == a.B - b)) copy = page;
  }
  const int before = pg_scan_one(goal - kept + (copy >= 0), waves[1], taken);
  s_goal[tid] = goal;
  s_before[tid] = before;
  s_copy[tid] = copy;
  __syncthreads();
  at = free_before;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = p0 + j;
    if (p >= a.n_pages) break;
    const int k = writers[p];
    int out = r[j];
    if (r[j] == 0) out = at++ < taken ? 1 : 0;
    else if (k > 0 && r[j] > 1) out -= r[j] == k ? k - 1 : k;
    a.refs_out[p] = out;
  }
  if (b < a.B) {
    a.len_out[b] = q.keep + q.add;
    a.copy_src[b] = copy;
    a.copy_rows[b] = copy >= 0 ? q.keep & ((1 << a.page_log2) - 1) : 0;
    a.copy_dst[b] = copy >= 0 && before < n_free ? free_ids[before] : -1;
  }
  for (int row = wave; row < a.B; row += kPgOneThreads / 64) {
    const int par = s_parent[row], end = s_goal[row], cp = s_copy[row], base = s_before[row];
    const int old_end = s_keep[row] - (cp >= 0 ? 1 : 0);
    int32_t* out = a.table_out + (int64_t)row * a.max_pages;
    const int32_t* t = a.table + (int64_t)max(par, 0) * a.max_pages;
    for (int i = (t == out ? old_end : 0) + lane; i < end; i += 64) {
      int id = -1;
      if (i < old_end) id = t[i];
      else if (base + i - old_end < n_free) id = free_ids[base + i - old_end];
      else flag_dev_err(a.err, kDevErrPagesFull);
      out[i] = id;
    }
  }
}

static bool pages_one(int n_pages, int B, int max_pages) {
  return n_pages <= kPgOnePages && B <= kPgOneThreads && (int64_t)B * max_pages <= kPgOneEntries;
}
size_t pages_counters(int n_pages) { return (size_t)n_pages * 12; }
static int64_t pages_parts(int max_pages) { return ((int64_t)max_pages + kPgSpan - 1) / kPgSpan; }
bool pages_fits(int B, int max_pages) {
  return pages_parts(max_pages) * B / 4 + (kPagesMax / kPgChunk) + 2 < 1 << 24;
}
void launch_pages_fork(const PagesForkArgs& a, hipStream_t st) {
  const int parts = (int)pages_parts(a.max_pages);
  const int rows = a.B > a.B_in ? a.B : a.B_in;
  if (pages_one(a.n_pages, rows, a.max_pages)) {
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

// the thread's four pages' counts (0 past the end)
__device__ __forceinline__ int pc_load(const int32_t* refs, int n_pages, int p0, int (&r)[4]) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[j] = p0 + j < n_pages ? refs[p0 + j] : 0;
    n += r[j] != 0;
  }
  return n;
}

__global__ __launch_bounds__(256) void k_pages_used(PagesCompactArgs a) {
  __shared__ int waves[4];
  const PcWork w = pc_work(a.workspace, a.n_pages);
  int r[4], all;
  const int n = pc_load(a.refs, a.n_pages, blockIdx.x * kPgChunk + 4 * threadIdx.x, r);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (r[j] < 0) flag_dev_err(a.err, kDevErrPagePlan);
  pg_block_scan(n, waves, all);
  if (threadIdx.x == 0) w.used_in[blockIdx.x] = all;
}

__global__ __launch_bounds__(256) void k_pages_lists(PagesCompactArgs a) {
  __shared__ int waves[4], waves2[4];
  const PcWork w = pc_work(a.workspace, a.n_pages);
  const int64_t before = pg_wave_total(w.used_in, blockIdx.x);
  const int U = (int)pg_wave_total(w.used_in, w.chunks);
  const int p0 = blockIdx.x * kPgChunk + 4 * threadIdx.x;
  int r[4], u[4], all;
  const int n = pc_load(a.refs, a.n_pages, p0, r);
  int rank = (int)before + pg_block_scan(n, waves, all);  // used pages before p0
  // used pages below U: whole chunks, and those of U's own
  const int cu = U / kPgChunk, q0 = cu * kPgChunk + 4 * threadIdx.x;
  pc_load(a.refs, a.n_pages, q0, u);
  int mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) mine += u[j] != 0 && q0 + j < U;
  pg_block_scan(mine, waves2, all);
  const int low = (int)pg_wave_total(w.used_in, cu) + all, moves = U - low;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    w.sums[0] = U;
    w.sums[1] = low;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = p0 + j;
    if (p >= a.n_pages) break;
    int fate = kPcFree;
    if (r[j] != 0) {
      fate = p < U ? kPcStays : rank - low;
      if (p >= U) {
        a.copy_src[fate] = p;
        w.high_ref[fate] = r[j];
      }
    } else if (p < U) {
      a.copy_dst[p - rank] = p;  // p - rank free pages before it
    }
    w.fate[p] = fate;
    if (p >= moves && p < a.n_pages / 2) {
      a.copy_src[p] = -1;
      a.copy_dst[p] = -1;
    }
    rank += r[j] != 0;
  }
}

// blocks 0 .. chunks - 1: the counts; then waves (sequence, part of its row)
__global__ __launch_bounds__(256) void k_pages_map(PagesCompactArgs a, int parts) {
  const PcWork w = pc_work(a.workspace, a.n_pages);
  if ((int)blockIdx.x < w.chunks) {
    __shared__ int waves[4];
    const int U = w.sums[0];
    const int p0 = blockIdx.x * kPgChunk + 4 * threadIdx.x;
    int r[4], all;
    const int n = pc_load(a.refs, a.n_pages, p0, r);
    int rank = (int)pg_wave_total(w.used_in, blockIdx.x) + pg_block_scan(n, waves, all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + j;
      if (p >= a.n_pages) break;
      const int f = w.fate[p];
      a.moved_to[p] = f == kPcFree ? -1 : f == kPcStays ? p : a.copy_dst[f];
      a.refs_out[p] = p >= U ? 0 : r[j] != 0 ? r[j] : w.high_ref[p - rank];
      rank += r[j] != 0;
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

// The same for small pools, in one launch of one block.
__global__ __launch_bounds__(kPgOneThreads) void k_pages_compact_one(PagesCompactArgs a) {
  __shared__ int fate[kPgOnePages];                                   // new id, -1: free
  __shared__ uint16_t high[kPgOnePages / 2], low[kPgOnePages / 2];    // ids that move, and where to
  __shared__ int high_ref[kPgOnePages / 2];
  __shared__ int waves[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, p0 = 8 * tid;
  int r[8], n = 0, U, below = 0, n_low;
  pg_load8(a.refs, a.n_pages, p0, 0, r);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (r[j] < 0) flag_dev_err(a.err, kDevErrPagePlan);
    n += r[j] != 0;
  }
  const int first = pg_scan_one(n, waves[0], U);
#pragma unroll
  for (int j = 0; j < 8; ++j) below += r[j] != 0 && p0 + j < U;
  pg_scan_one(below, waves[1], n_low);
  const int moves = U - n_low;
  int rank = first;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = p0 + j;
    if (p < a.n_pages) {
      if (r[j] != 0 && p >= U) {
        high[rank - n_low] = (uint16_t)p;
        high_ref[rank - n_low] = r[j];
      }
      if (r[j] == 0 && p < U) low[p - rank] = (uint16_t)p;
    }
    rank += r[j] != 0;
  }
  __syncthreads();
  rank = first;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = p0 + j;
    if (p < a.n_pages) {
      const int to = r[j] == 0 ? -1 : p < U ? p : low[rank - n_low];
      fate[p] = to;
      a.moved_to[p] = to;
      a.refs_out[p] = p >= U ? 0 : r[j] != 0 ? r[j] : high_ref[p - rank];
    }
    rank += r[j] != 0;
  }
  for (int i = tid; i < a.n_pages / 2; i += kPgOneThreads) {
    a.copy_src[i] = i < moves ? high[i] : -1;
    a.copy_dst[i] = i < moves ? low[i] : -1;
  }
  __syncthreads();
  for (int b = wave; b < a.B; b += kPgOneThreads / 64) {
    const int len = a.len[b];
    if (len < 0 || len > kPgLongest || (int64_t)len > (int64_t)a.max_pages << a.page_log2) {
      if (lane == 0) flag_dev_err(a.err, kDevErrPagePlan);
      continue;
    }
    const int end = pg_pages(a.page_log2, len);
    for (int i = lane; i < end; i += 64) {
      const int64_t at = (int64_t)b * a.max_pages + i;
      const int p = a.table[at];
      int to = p;
      if ((unsigned)p >= (unsigned)a.n_pages) {
        flag_dev_err(a.err, kDevErrPageId);
      } else {
        to = fate[p];
        if (to < 0) flag_dev_err(a.err, kDevErrPagePlan);
      }
      a.table_out[at] = to;
    }
  }
}

void launch_pages_compact(const PagesCompactArgs& a, hipStream_t st) {
  if (pages_one(a.n_pages, a.B, a.max_pages)) {
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
  const size_t fork = 4 * (chunks + plans + 6 * (size_t)B + chunks * kPgChunk);
  return fork > pc_bytes(n_pages) ? fork : pc_bytes(n_pages);
}

// ---------------------------------------------------------------------------
// Copy.  A block takes one 16-byte unit per thread of a page, in one pool, for 64
// entries of the list: the entries that are none cost a load and a ballot.
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
