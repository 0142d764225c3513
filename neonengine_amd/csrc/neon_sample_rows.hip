// neon_sample_rows.hip -- sampling with temperature, top-k, top-p, min-p and a
// given random number per row.
//
// For a row l with maximum m:  w_i = exp((l_i - m) / T) in 64 bits.  Tokens are
// ordered by (l descending, index ascending).  Kept are the first top_k; of
// these the shortest prefix whose mass reaches top_p times theirs; of these the
// ones with w_i >= min_p.  The draw is the lowest kept index whose running sum,
// in index order, exceeds u times the kept mass.
//
// Masses are integers, round(w 2^S) with V 2^S <= 2^62: sums are exact, so no
// order of threads or atomics changes a draw.  A token more than 31.2 below the
// maximum (in units of T; 45 ln 2, less past 2^18 tokens, where S is smaller) has
// mass 0 and cannot be drawn; its share is under 2^-45 of the most probable token's,
// below the 2^-24 steps of u.
#include <hip/hip_runtime.h>

#include "neon_common.hpp"
#include "neon_internal.hpp"

namespace neon {

typedef unsigned long long u64;

// Order of a logit as an integer: larger logit, larger key; both zeros are
// one; NaN counts as minus infinity.
__device__ __forceinline__ uint32_t sr_key(float l) {
  if (l != l) l = -INFINITY;
  const uint32_t b = __float_as_uint(l + 0.0f);  // -0 + 0 = +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kSrNone = 0x007FFFFFu;  // key of minus infinity

// ---------------------------------------------------------------------------
// A row is cut into chunks of one block each.  The order is searched in bins of
// 1/16 of T below the maximum (512 of them; what lies further down has mass 0):
//   k_sr_max    chunk maxima
//   k_sr_hist   adds the chunk's count and mass of every bin to the row's
//   k_sr_pick   finds the bins that the top_k-th token and the token at top_p's goal
//               can lie in (every block for itself), then per chunk the mass of the
//               bins above those, which is kept whatever the exact places are, and
//               the tokens of those bins (the candidates); the row's last block
//               finds the two places among the candidates, then the part that holds
//               the draw, then the token in it
// A row of one chunk is one launch with the same steps.  Nothing but the chunks'
// partial results crosses launches, at agent scope, so that the last block reads
// what the others wrote without a launch in between.
// Bound: for many rows three reads of the logits (64 x 201088: 10.5 us each at the
// rate of a large copy), k_sr_hist's 64-bit exponentials (vector units 75% busy) and
// the last blocks; for few rows the chain of dependent steps, about 10 us of it in
// the last block of k_sr_pick (sort 4.5, draw 3.5).
// Candidates are some hundreds of 201088 normal logits at a deviation of 2.5 T (sorted,
// up to 512), up to 4096 at 1.3 T (selected by digits: 34 us for one row), and more
// where the row is flatter: then the last block reads the row again for each step, and
// one row of deviation T takes 520 us, 64 of them 960.
// Kernel times, us (max + hist + pick): 1 x 201088 3 + 5 + 16, 64 x 201088 10.5 +
// 22.5 + 37, 7 x 32003 3 + 4.5 + 18; one block per row, 8 bits of the key at a time,
// took 585, 1030 and 206.
// ---------------------------------------------------------------------------
constexpr int kSrThreads = 512;
constexpr int kSrBins = 512;   // one per thread in the scan
constexpr int kSrCap = 4096;   // candidates of a row that are listed
constexpr int kSrPart = 8 * kSrThreads;  // tokens whose kept mass is held apart
constexpr int kSrMaxChunk = 65536;
constexpr int kSrMaxParts = kSrMaxChunk / kSrPart;
constexpr float kSrBinsPerT = 16.0f;

// A row's parameters as the kernels use them.
struct SrRow {
  const float* l;
  int V;
  float m;       // the maximum
  float bin_t;   // bins per unit of the logits
  double m_d;    // the same
  double to_t;   // 64 log2(e) / T
  double scale;  // 2^S
  const double* table;
  double min_p, p, u;
  int k;         // 0: all
  uint64_t best; // key and ~index of the maximum
};
// exp((l - m) / T) by table (P.T.P. Tang's method): with t = 64 log2(e) (l - m)
// / T and n the nearest integer, 2^(n / 64) = 2^(n >> 6) table[n & 63] and the
// rest 2^(x / 64), |x| <= 1/2, is a Taylor sum in x: with y = x ln 2 / 64 its
// next term y^6 / 720 < 2^-53.  t is below 64 x 46.2 where a mass is not 0, so
// its rounding costs 2^-48.  About 20 instructions; exp() and a conversion to
// 64 bits are 50, which bound k_sr_hist (64 x 201088: 37.6 -> 29.2 us then).  For
// tokens in a bin only: no overflow; both infinite give t = NaN, which is 0 here.
constexpr int kSrTable = 64;
__device__ __forceinline__ void sr_table(double* table) {
  if (threadIdx.x < kSrTable) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / kSrTable));
}
__device__ __forceinline__ double sr_weight(const SrRow& r, float l) {
  constexpr double L = 0.69314718055994530942 / kSrTable;
  const double t = fmin(((double)l - r.m_d) * r.to_t, 0.0);
  const double n = __builtin_rint(t), x = t - n;
  const int i = (int)n;
  double e = __builtin_fma(x, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
  e = __builtin_fma(x, e, L * L * L / 6.0);
  e = __builtin_fma(x, e, L * L / 2.0);
  e = __builtin_fma(x, e, L);
  e = __builtin_fma(x, e, 1.0);
  return __builtin_ldexp(r.table[i & (kSrTable - 1)] * e, i >> 6);
}
// round(w 2^S) for w 2^S <= 2^44: the low bits of w 2^S + 2^52
__device__ __forceinline__ u64 sr_units(const SrRow& r, double w) {
  return (u64)__builtin_bit_cast(int64_t, __builtin_fma(w, r.scale, 0x1p52)) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ u64 sr_mass(const SrRow& r, float l) { return sr_units(r, sr_weight(r, l)); }
// mass under min_p's limit: 0 below it
__device__ __forceinline__ u64 sr_kept_mass(const SrRow& r, float l) {
  const double w = sr_weight(r, l);
  return w >= r.min_p ? sr_units(r, w) : 0;
}
// The first bin whose weights all lie below min_p (w <= exp(-bin / 16), the
// 1 + 2^-10 covers the rounding of the bins and of the logarithm).
__device__ __forceinline__ int sr_min_bin(const SrRow& r) {
  if (!(r.min_p > 0.0)) return kSrBins;
  return (int)fminf(-__logf((float)r.min_p) * (kSrBinsPerT * (1.0f + 0x1p-10f)) + 2.0f,
                    (float)kSrBins);
}
// Falls with l, never rises: each step rounds monotonically.
__device__ __forceinline__ int sr_bin(const SrRow& r, float l) {
  if (l == r.m) return 0;
  const float x = (r.m - l) * r.bin_t;
  return x < (float)kSrBins ? (int)x : kSrBins;  // a NaN goes to the end
}
__device__ __forceinline__ float sr_clean(float l) { return l != l ? -INFINITY : l + 0.0f; }
// unique, and in the order of the tokens: larger logit, then lower index
__device__ __forceinline__ u64 sr_place(float l, int i) {
  return ((u64)sr_key(l) << 32) | (uint32_t)~i;
}

__device__ __forceinline__ double sr_scale(int V) {
  const int lg = V > 1 ? 32 - __builtin_clz((unsigned)(V - 1)) : 0;
  return lg <= 18 ? 0x1p44 : __builtin_ldexp(1.0, 62 - lg);
}

__device__ __forceinline__ u64 sr_get(const u64* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void sr_put(u64* p, u64 v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int J>
__device__ __forceinline__ u64 sr_xor_lane(u64 x) {
  return (u64)(uint32_t)xor_lane_i<J>((int)(uint32_t)x) |
         (u64)(uint32_t)xor_lane_i<J>((int)(x >> 32)) << 32;
}
template <int J = 32>
__device__ __forceinline__ u64 sr_wave_sum(u64 v) {
  v += sr_xor_lane<J>(v);
  if constexpr (J > 1) return sr_wave_sum<J / 2>(v);
  else return v;
}
template <int J = 32>
__device__ __forceinline__ u64 sr_wave_max(u64 v) {
  const u64 x = sr_xor_lane<J>(v);
  v = x > v ? x : v;
  if constexpr (J > 1) return sr_wave_max<J / 2>(v);
  else return v;
}
// v plus that of the lane that CTRL names, where ROWS has the lane's row (DPP)
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 sr_add_from(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
  return v + ((u64)hi << 32 | lo);
}
// sum of the lanes up to this one
__device__ __forceinline__ u64 sr_wave_scan(u64 v) {
  v = sr_add_from<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = sr_add_from<0x112, 0xF>(v);
  v = sr_add_from<0x114, 0xF>(v);
  v = sr_add_from<0x118, 0xF>(v);
  v = sr_add_from<0x142, 0xA>(v);  // a row's last lane into the next row
  return sr_add_from<0x143, 0xC>(v);  // lane 31 into the upper half
}
__device__ __forceinline__ u64 sr_block_sum(u64 v, u64* red) {
  v = sr_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int w = 0; w < kSrThreads / 64; ++w) t += red[w];
  return t;
}
__device__ __forceinline__ u64 sr_block_max(u64 v, u64* red) {
  v = sr_wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSrThreads / 64; ++w) v = red[w] > v ? red[w] : v;
  return v;
}
// sum of the threads before this one; `all`: of the block's
__device__ __forceinline__ u64 sr_block_before(u64 v, u64* red, u64& all) {
  u64 x = sr_wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = x;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kSrThreads / 64; ++w) {
    const u64 y = red[w];
    all += y;
    if (w < (int)(threadIdx.x >> 6)) x += y;
  }
  return x - v;
}
__device__ __forceinline__ u64 sr_block_before(u64 v, u64* red) {
  u64 all;
  return sr_block_before(v, red, all);
}

// What the scan of the bins finds.
struct SrFound {
  int lo, hi;     // bins that top_p's token can lie in: everything before lo is kept
  int bin_k;      // bin of the top_k-th token, kSrBins where none is cut
  u64 base;       // mass before lo
  u64 before_k;   // mass before bin_k
  u64 mass_k;     // mass of the top_k tokens, where bin_k cuts none
  u64 need_k;     // tokens of bin_k that are among the top_k
};

struct SrHistShared {
  u64 red[16];
  double table[kSrTable];
  u64 mass[kSrBins];
  uint32_t count[kSrBins];
  SrFound found;
  u64 s_u64[2];
  int s_int[4];
};
struct SrShared : SrHistShared {
  u64 any[256];
  u64 list[kSrCap];
  float queue[kSrThreads / 64][512];       // per wave: the tokens of eight that matter,
  uint16_t queued[kSrThreads / 64][512];   // and which they are
};

// Reads row b's parameters; false where one is out of range.
__device__ __forceinline__ bool sr_params(const SampleRowsArgs& a, int b, double* table, SrRow& r,
                                          bool& greedy) {
  const float t = a.temperature != nullptr ? a.temperature[b] : 1.0f;
  const float p = a.top_p != nullptr ? a.top_p[b] : 1.0f;
  const float mp = a.min_p != nullptr ? a.min_p[b] : 0.0f;
  const float u = a.u[b];
  const int k = a.top_k != nullptr ? a.top_k[b] : 0;
  sr_table(table);  // a barrier follows with the row's maximum
  r.table = table;
  r.l = a.logits + (int64_t)b * a.stride;
  r.V = a.V;
  r.k = k > 0 && k < a.V ? k : 0;
  r.p = (double)p;
  r.min_p = (double)mp;
  r.u = (double)u;
  r.to_t = 64.0 * 1.44269504088896340736 / (double)t;
  r.bin_t = (float)(1.0 / (double)t) * kSrBinsPerT;
  r.scale = sr_scale(a.V);
  greedy = t == 0.0f;
  return t >= 0.0f && t < INFINITY && p > 0.0f && p <= 1.0f && mp >= 0.0f && mp <= 1.0f &&
         u >= 0.0f && u < 1.0f;
}
__device__ __forceinline__ void sr_set_best(SrRow& r, u64 best) {
  r.best = best;
  const uint32_t key = (uint32_t)(best >> 32);
  r.m = __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
  r.m_d = (double)r.m;
}
__device__ __forceinline__ int sr_best_id(u64 best) { return (int)~(uint32_t)best; }

// fn(logits, index of the first) for tokens [i0, i1), i0 a multiple of kSrPart: a
// thread's eight of a part are 512 apart.  The next part's are requested before
// these are used; the last, incomplete part has minus infinity past i1.
// The first part (`first`) may be requested before work that its use waits for.
struct SrPart {
  float v[8];
};
__device__ __forceinline__ SrPart sr_part(const float* l, int i, int i1) {
  SrPart p;
  if (i + kSrPart <= i1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) p.v[j] = (l + i + j * kSrThreads)[threadIdx.x];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) p.v[j] = l[min(i + (int)threadIdx.x + j * kSrThreads, i1 - 1)];
  }
  return p;
}
template <class F>
__device__ __forceinline__ void sr_tokens(const float* l, int i0, int i1, SrPart next, F fn) {
  const int tid = threadIdx.x;
  for (int i = i0; i < i1; i += kSrPart) {
    SrPart p = next;
    if (i + kSrPart < i1) next = sr_part(l, i + kSrPart, i1);
    if (i + kSrPart > i1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) p.v[j] = i + tid + j * kSrThreads < i1 ? p.v[j] : -INFINITY;
    }
    fn(p.v, i + tid);
  }
}

__device__ __forceinline__ u64 sr_chunk_max(const float* l, int i0, int i1, u64* red) {
  float best = -INFINITY;  // of equal ones the first; a NaN is never larger
  int at = i0;
  sr_tokens(l, i0, i1, sr_part(l, i0, i1), [&](const float (&v)[8], int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      at = v[j] > best ? i + j * kSrThreads : at;
      best = v[j] > best ? v[j] : best;
    }
  });
  return sr_block_max(sr_place(best, at), red);
}

// counts (for top_k) and masses (for top_p) of the chunk's bins into sh.count /
// sh.mass
template <class SH>
__device__ __forceinline__ void sr_chunk_hist(const SrRow& r, int i0, int i1, const SrPart& first, SH& sh) {
  sh.mass[threadIdx.x] = 0;
  sh.count[threadIdx.x] = 0;
  __syncthreads();
  sr_tokens(r.l, i0, i1, first, [&](const float (&v)[8], int) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int bin = sr_bin(r, v[j]);
      if (bin < kSrBins) {
        if (r.k > 0) atomicAdd(&sh.count[bin], 1u);
        if (r.p < 1.0) atomicAdd(&sh.mass[bin], sr_mass(r, v[j]));
      }
    }
  });
  __syncthreads();
}

// The bins to look into, from the row's counts and masses (thread = bin).
template <class SH>
__device__ __forceinline__ void sr_scan(const SrRow& r, u64 count, u64 mass, SH& sh) {
  const int bin = threadIdx.x;
  const u64 c0 = sr_block_before(count, sh.red), m0 = sr_block_before(mass, sh.red);
  const u64 c1 = c0 + count, m1 = m0 + mass;
  SrFound& f = sh.found;
  if (bin == 0) {
    f.bin_k = kSrBins;
    f.lo = f.hi = kSrBins;
    f.base = f.before_k = f.need_k = 0;
  }
  if (bin == kSrBins - 1) f.mass_k = m1;
  __syncthreads();
  const u64 k = (u64)r.k;
  if (r.k > 0 && c0 < k && c1 >= k) {
    if (c1 == k) {  // the bins up to this one are the top_k
      f.mass_k = m1;
      f.lo = bin + 1;  // where top_p is off: no candidates
      f.hi = bin;
    } else {
      f.bin_k = bin;
      f.before_k = m0;
      f.need_k = k - c0;
      f.lo = f.hi = bin;
      f.mass_k = m1;  // an upper bound
    }
  }
  __syncthreads();
  if (r.p < 1.0) {
    const bool cut = f.bin_k < kSrBins;
    const double g0 = r.p * (double)(cut ? f.before_k : f.mass_k), g1 = r.p * (double)f.mass_k;
    __syncthreads();
    // the first bins whose running mass reaches the goal (the last bin reaches
    // any); with g0 = 0, no bin does better than the first
    if ((double)m1 >= g0 && (bin == 0 || (double)m0 < g0)) f.lo = bin;
    if ((double)m1 >= g1 && (bin == 0 || (double)m0 < g1)) f.hi = bin;
    __syncthreads();
    if (bin == f.lo) f.base = m0;
  }
  __syncthreads();
}

__device__ __forceinline__ bool sr_candidate(const SrFound& f, int bin) {
  return (bin >= f.lo && bin <= f.hi && bin < kSrBins) || bin == f.bin_k;
}

// The kept mass of the sure bins of each part of tokens [i0, i1) (i0 a multiple
// of kSrPart) into sh.mass[0 ..], thread = part for the result; the candidates
// into sh.list (as many as fit; sh.s_int[0] counts all).
__device__ __forceinline__ u64 sr_collect(const SrRow& r, const SrFound& f, int i0, int i1,
                                          const SrPart& first, SrShared& sh) {
  __syncthreads();
  if (threadIdx.x == 0) sh.s_int[0] = 0;
  if (threadIdx.x < kSrMaxParts) sh.mass[threadIdx.x] = 0;
  __syncthreads();
  const int keep = min(min(f.lo, kSrBins), sr_min_bin(r));
  // Mostly a few of a hundred tokens matter: those of the first bins, up to
  // `keep`, and those of the candidates' bins.  Logits that bound them from outside:
  auto edge = [&](int bin, double out) {
    const double below = bin / (double)r.bin_t;
    const float x = (float)(r.m_d - below + out * (fabs(r.m_d) + below) * 1e-6);
    return x == x ? x : (float)-INFINITY;
  };
  const int c_lo = min(f.lo, f.bin_k), c_hi = max(f.hi < kSrBins ? f.hi : -1, f.bin_k < kSrBins ? f.bin_k : -1);
  const float from = keep > 0 ? edge(keep, -1.0) : INFINITY;
  const float c_from = c_hi >= 0 ? edge(c_hi + 1, -1.0) : INFINITY;
  const float c_to = c_lo > 0 ? edge(c_lo, 1.0) : INFINITY;
  sr_tokens(r.l, i0, i1, first, [&](const float (&v)[8], int i) {
    // gathered first: a wave pays an exponential for all its lanes if one needs it
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = v[j] >= from || (v[j] >= c_from && v[j] <= c_to);
      const u64 who = __ballot(in);
      if (in) {
        const int to = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                                     __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        sh.queue[wave][to] = v[j];
        sh.queued[wave][to] = (uint16_t)(j * kSrThreads + lane);
      }
      n += __builtin_popcountll(who);
    }
    wave_lds_sync();
    u64 sure = 0;
    for (int q = lane; q < n; q += 64) {
      const float l = sh.queue[wave][q];
      const int bin = sr_bin(r, l);
      if (bin < keep) {
        sure += sr_kept_mass(r, l);
      } else if (bin >= f.lo && bin < kSrBins && sr_candidate(f, bin)) {
        const int to = atomicAdd(&sh.s_int[0], 1);
        if (to < kSrCap) sh.list[to] = sr_place(l, i - lane + (int)sh.queued[wave][q]);
      }
    }
    wave_lds_sync();  // read before the next eight are written
    if (__any(sure > 0)) {  // 64 lanes on one address would be done one by one
      sure = sr_wave_sum(sure);
      if ((threadIdx.x & 63) == 0) atomicAdd(&sh.mass[(i - i0) / kSrPart], sure);
    }
  });
  __syncthreads();
  return threadIdx.x < kSrMaxParts ? sh.mass[threadIdx.x] : 0;
}

__device__ __forceinline__ float sr_place_logit(u64 place) {
  const uint32_t key = (uint32_t)(place >> 32);
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Calls fn(place) for every candidate at or above `from` in the bins [lo, hi]:
// of the list, or of the row where the list did not hold them all.
template <class F>
__device__ __forceinline__ void sr_each(const SrRow& r, const SrShared& sh, int n, int lo, int hi,
                                        u64 from, F fn) {
  if (n <= kSrCap) {
    for (int j = threadIdx.x; j < n; j += kSrThreads) {
      const u64 x = sh.list[j];
      if (x < from) continue;
      const int bin = sr_bin(r, sr_place_logit(x));
      if (bin >= lo && bin <= hi) fn(x);
    }
  } else {
    for (int i = threadIdx.x; i < r.V; i += kSrThreads) {
      const float l = sr_clean(r.l[i]);
      const int bin = sr_bin(r, l);
      if (bin < lo || bin > hi || bin >= kSrBins) continue;
      const u64 x = sr_place(l, i);
      if (x >= from) fn(x);
    }
  }
}

// The place of the candidate at which the running count (or mass), in order and
// starting at `base`, reaches `goal`; the last one where none does.  `upto`: the
// running value including it.  Searched by 8 bits of the place at a time,
// beginning at the highest bit in which the candidates differ.
template <bool MASS>
__device__ __forceinline__ u64 sr_select(const SrRow& r, SrShared& sh, int n, int lo, int hi, u64 from,
                                         u64 base, double goal, u64& upto) {
  const int tid = threadIdx.x;
  u64 mx = 0, mn = 0;  // of the places, and of their complements
  sr_each(r, sh, n, lo, hi, from, [&](u64 x) {
    mx = x > mx ? x : mx;
    mn = ~x > mn ? ~x : mn;
  });
  mx = sr_block_max(mx, sh.red);
  mn = ~sr_block_max(mn, sh.red);
  int top = mx == mn ? 0 : 64 - __builtin_clzll(mx ^ mn);  // bits to decide
  u64 prefix = top < 64 ? mx >> top : 0;
  u64 run = base;
  while (true) {
    const int shift = top > 8 ? top - 8 : 0;
    const int digits = 1 << (top - shift);
    __syncthreads();
    if (tid < 256) {
      sh.mass[tid] = 0;
      sh.count[tid] = 0;
    }
    __syncthreads();
    sr_each(r, sh, n, lo, hi, from, [&](u64 x) {
      if (top < 64 && (x >> top) != prefix) return;
      const int d = (int)(x >> shift) & (digits - 1);
      if (MASS) atomicAdd(&sh.mass[d], sr_mass(r, sr_place_logit(x)));
      atomicAdd(&sh.count[d], 1u);
      sh.any[d] = x;
    });
    __syncthreads();
    if (tid < 64) {  // four digits a lane, from the largest down
      u64 c[4], v[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = 255 - (4 * tid + j);
        c[j] = d < digits ? sh.count[d] : 0;
        v[j] = MASS ? (d < digits ? sh.mass[d] : 0) : c[j];
        sum += v[j];
      }
      const u64 x = sr_wave_scan(sum);
      u64 at = run + x - sum;
      // the first digit that reaches the goal, else the last that is there
      int hit = -1, last = -1;
      u64 hit_at = 0, last_at = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c[j] > 0) {
          last = 4 * tid + j;
          last_at = at;
          if (hit < 0 && (double)(at + v[j]) >= goal) {
            hit = last;
            hit_at = at;
          }
        }
        at += v[j];
      }
      const u64 hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
      const int lane = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(lasts | 1);
      if (tid == lane) {
        sh.s_int[1] = 255 - (hits ? hit : last);
        sh.s_u64[0] = hits ? hit_at : last_at;
      }
    }
    __syncthreads();
    const int d = sh.s_int[1];
    run = sh.s_u64[0];
    if (sh.count[d] == 1 || shift == 0) {
      upto = run + (MASS ? sh.mass[d] : sh.count[d]);
      return sh.any[d];
    }
    prefix = (prefix << (top - shift)) | (u64)d;
    top = shift;
  }
}

// Bitonic sort, descending, of the threads' x; those from n on hold 0.  Loops:
// unrolled, the 45 steps are fetched once each, which takes longer than they do.
template <int J>
__device__ __forceinline__ u64 sr_sort_lanes(u64 x, int K) {
  if (J < K) {
    const u64 y = sr_xor_lane<J>(x);
    const bool larger = ((threadIdx.x & K) == 0) == ((threadIdx.x & J) == 0);
    x = (x > y) == larger ? x : y;
  }
  if constexpr (J > 1) return sr_sort_lanes<J / 2>(x, K);
  else return x;
}
__device__ __forceinline__ u64 sr_sort(u64 x, u64* buf, int n) {
  const int tid = threadIdx.x;
  const bool in = (tid & ~63) < 1 << (32 - __builtin_clz(max(n - 1, 1)));
#pragma unroll 1
  for (int K = 2; K < 2 * n && K <= kSrThreads; K *= 2) {  // runs of K, distance J
#pragma unroll 1
    for (int J = K / 2; J >= 64; J /= 2) {
      __syncthreads();
      buf[tid] = x;
      __syncthreads();
      const u64 y = buf[tid ^ J];
      const bool larger = ((tid & K) == 0) == ((tid & J) == 0);
      x = (x > y) == larger ? x : y;
    }
    if (in) x = sr_sort_lanes<32>(x, K);  // the other waves hold zeros only
  }
  return x;
}

// sr_cut for up to one candidate per thread: sorted, the places are positions.
// A selection by digits takes about two passes for each of the two places, each
// with a histogram, its sum and six barriers: 10 us where this takes 4.
__device__ __forceinline__ u64 sr_cut_sorted(const SrRow& r, SrShared& sh, int n) {
  const int tid = threadIdx.x;
  const SrFound f = sh.found;
  u64 x = tid < n ? sh.list[tid] : 0;
  x = sr_sort(x, sh.list, n);
  __syncthreads();
  sh.list[tid] = x;
  const bool has = tid < n;
  const float l = sr_place_logit(x);
  const int bin = has ? sr_bin(r, l) : kSrBins;
  u64 mass_k = f.mass_k, cut = 0;
  const u64 mass = has && r.p < 1.0 ? sr_mass(r, l) : 0;
  bool in = has;  // among the top_k
  if (f.bin_k < kSrBins) {
    const int first = __syncthreads_count(bin < f.bin_k);
    in = has && tid < first + (int)f.need_k;
    cut = sh.list[min(first + (int)f.need_k, n) - 1];
    if (r.p < 1.0) mass_k = f.before_k + sr_block_sum(in && bin == f.bin_k ? mass : 0, sh.red);
  }
  __syncthreads();  // the sorted list is there
  if (r.p < 1.0 && f.lo < kSrBins) {
    const bool mine = in && bin >= f.lo && bin <= f.hi;
    const u64 own = mine ? mass : 0;
    const u64 upto = f.base + sr_block_before(own, sh.red) + own;
    // the first of them that reaches the goal, else the last of them
    const int all = __syncthreads_count(mine);
    const int short_of = __syncthreads_count(mine && (double)upto < r.p * (double)mass_k);
    cut = sh.list[max(min(short_of, all - 1), 0)];
  }
  return cut;
}

// The last place that is kept, from the row's n candidates.
__device__ __forceinline__ u64 sr_cut(const SrRow& r, SrShared& sh, int n) {
  if (n <= kSrThreads) return sr_cut_sorted(r, sh, n);
  const SrFound f = sh.found;
  u64 cut = 0, mass_k = f.mass_k, upto;
  if (f.bin_k < kSrBins) {
    cut = sr_select<false>(r, sh, n, f.bin_k, f.bin_k, 0, 0, (double)f.need_k, upto);
    if (r.p < 1.0) {
      u64 in = 0;
      sr_each(r, sh, n, f.bin_k, f.bin_k, cut, [&](u64 x) { in += sr_mass(r, sr_place_logit(x)); });
      mass_k = f.before_k + sr_block_sum(in, sh.red);
    }
  }
  if (r.p < 1.0 && f.lo < kSrBins)
    cut = sr_select<true>(r, sh, n, f.lo, f.hi, cut, f.base, r.p * (double)mass_k, upto);
  return cut;
}

// Whether the token is kept before min_p: bins before lo are, the others from
// the cut on.
__device__ __forceinline__ bool sr_in(const SrFound& f, u64 cut, int bin, u64 place) {
  return bin < f.lo ? bin < kSrBins : sr_candidate(f, bin) && place >= cut;
}

// The token of the part [i0, i1) (up to kSrPart of them) at which the kept
// running mass, starting at `before`, exceeds the target; the row's best where
// rounding leaves none.  A thread holds the tokens tid + 512 j, so a wave's 64
// for one j are in order: their masses add up in a segment each.
__device__ __forceinline__ int sr_walk(const SrRow& r, SrShared& sh, u64 cut, int i0, int i1, u64 before,
                                       double target) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const SrFound f = sh.found;
  const int limit = sr_min_bin(r);
  __syncthreads();
  if (tid < 64) sh.mass[tid] = 0;
  if (tid == 0) sh.s_int[2] = sr_best_id(r.best);
  __syncthreads();
  u64 m[8];
  uint32_t todo = 0;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    m[j] = 0;
    v[j] = r.l[min(i0 + tid + j * kSrThreads, i1 - 1)];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = i0 + tid + j * kSrThreads;
    v[j] = sr_clean(v[j]);
    const int bin = sr_bin(r, v[j]);
    if (i < i1 && bin < limit && sr_in(f, cut, bin, sr_place(v[j], i))) todo |= 1u << j;
  }
  // each turn takes every lane's next one: a wave pays an exponential for all its
  // lanes if one needs it
  while (__any(todo != 0)) {
    const int at = __builtin_ctz(todo | 0x80000000u);
    float l = v[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) l = at == j ? v[j] : l;
    const u64 x = todo != 0 ? sr_kept_mass(r, l) : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = at == j ? x : m[j];
    if (x > 0) atomicAdd(&sh.mass[8 * at + wave], x);
    todo &= todo - 1;
  }
  __syncthreads();
  if (tid < 64) {
    const u64 own = sh.mass[tid];
    const u64 x = sr_wave_scan(own) + before;
    const u64 hit = __ballot(own > 0 && (double)x > target);
    if (tid == (hit ? __builtin_ctzll(hit) : 0)) {
      sh.s_int[1] = hit ? tid : -1;
      sh.s_u64[0] = x - own;
    }
  }
  __syncthreads();
  const int seg = sh.s_int[1];
  if (seg >= 0 && wave == (seg & 7)) {
    const int j = seg >> 3, lane = tid & 63;
    u64 own = m[0];
#pragma unroll
    for (int q = 1; q < 8; ++q) own = j == q ? m[q] : own;
    const u64 x = sr_wave_scan(own);
    const u64 hit = __ballot(own > 0 && (double)(x + sh.s_u64[0]) > target);
    if (hit && lane == __builtin_ctzll(hit)) sh.s_int[2] = i0 + tid + j * kSrThreads;
  }
  __syncthreads();
  return sh.s_int[2];
}

// The draw, from the parts' kept masses: part_mass(p0) gives the thread's of 512
// parts from p0 on.
template <class F>
__device__ __forceinline__ int sr_draw(const SrRow& r, SrShared& sh, u64 cut, F part_mass) {
  const int tid = threadIdx.x, parts = (r.V + kSrPart - 1) / kSrPart;
  u64 total = 0, own = 0, run = 0, all = 0;
  for (int p0 = 0; p0 < parts; p0 += kSrThreads) {
    own = part_mass(p0);
    run = sr_block_before(own, sh.red, all);
    total += all;
  }
  const double target = r.u * (double)total;
  u64 before = 0;
  for (int p0 = 0; p0 < parts; p0 += kSrThreads) {
    if (parts > kSrThreads) {
      own = part_mass(p0);
      run = before + sr_block_before(own, sh.red, all);
      before += all;
    }
    if (tid == 0) sh.s_int[3] = -1;
    __syncthreads();
    if (own > 0 && (double)run <= target && (double)(run + own) > target) {
      sh.s_int[3] = p0 + tid;
      sh.s_u64[1] = run;
    }
    __syncthreads();
    if (sh.s_int[3] >= 0) break;
  }
  const int hit = sh.s_int[3];
  const u64 start = sh.s_u64[1];
  return hit < 0 ? sr_best_id(r.best)
                 : sr_walk(r, sh, cut, hit * kSrPart, min((hit + 1) * kSrPart, r.V), start, target);
}

// Adds the kept candidates of 512 parts from p0 on to the thread's `sure` mass.
__device__ __forceinline__ u64 sr_part_mass(const SrRow& r, SrShared& sh, u64 cut, int n, int p0,
                                            u64 sure) {
  const SrFound f = sh.found;
  __syncthreads();
  sh.mass[threadIdx.x] = sure;
  __syncthreads();
  sr_each(r, sh, n, f.lo, kSrBins - 1, 0, [&](u64 x) {
    const float l = sr_place_logit(x);
    const int part = (int)~(uint32_t)x / kSrPart - p0;
    if (part >= 0 && part < kSrThreads && sr_in(f, cut, sr_bin(r, l), x))
      atomicAdd(&sh.mass[part], sr_kept_mass(r, l));
  });
  __syncthreads();
  return sh.mass[threadIdx.x];
}

// A row's place in the workspace: C chunks.
struct SrSpace {
  u64 *best, *sure, *list;  // [C], [parts], [kSrCap]
  u64 *mass, *count;        // [kSrBins]
  int32_t* n;               // candidates, arrivals
};
__host__ __device__ inline size_t sr_space_bytes(int C, int V) {
  const size_t b = (size_t)C * 8 + (size_t)((V + kSrPart - 1) / kSrPart) * 8 + kSrCap * 8 + 64 +
                   kSrBins * 16;
  return (b + 255) & ~(size_t)255;
}
__device__ __forceinline__ SrSpace sr_space(const SampleRowsArgs& a, int b) {
  SrSpace s;
  const int C = a.chunks;
  u64* p = reinterpret_cast<u64*>(reinterpret_cast<char*>(a.workspace) + (size_t)b * sr_space_bytes(C, a.V));
  s.best = p;
  s.sure = p + C;
  s.list = s.sure + (a.V + kSrPart - 1) / kSrPart;
  s.n = reinterpret_cast<int32_t*>(s.list + kSrCap);
  s.mass = s.list + kSrCap + 8;
  s.count = s.mass + kSrBins;
  return s;
}

__global__ __launch_bounds__(kSrThreads) void k_sr_max(SampleRowsArgs a) {
  __shared__ u64 red[16];
  const int c = blockIdx.x, b = blockIdx.y;
  const SrSpace s = sr_space(a, b);
  const u64 best = sr_chunk_max(a.logits + (int64_t)b * a.stride, c * a.chunk,
                                min((c + 1) * a.chunk, a.V), red);
  if (threadIdx.x == 0) s.best[c] = best;
  if (c == 0) {  // for the next launches
    if (threadIdx.x < 2) s.n[threadIdx.x] = 0;
    s.mass[threadIdx.x] = 0;
    s.count[threadIdx.x] = 0;
  }
}

// The row's parameters and maximum from the chunks'; false (the answer written
// by the row's first block) where there is nothing to search.
__device__ __forceinline__ bool sr_begin(const SampleRowsArgs& a, const SrSpace& s, int b, SrRow& r,
                                         SrHistShared& sh, bool answer) {
  bool greedy;
  const bool ok = sr_params(a, b, sh.table, r, greedy);
  u64 best = 0;
  for (int c = threadIdx.x; c < a.chunks; c += kSrThreads) best = s.best[c] > best ? s.best[c] : best;
  best = sr_block_max(best, sh.red);
  sr_set_best(r, best);
  const bool none = (uint32_t)(best >> 32) <= kSrNone;
  if (ok && !none && !greedy) return true;
  if (answer && blockIdx.x == 0 && threadIdx.x == 0) {
    a.ids[b] = ok && !none ? sr_best_id(best) : -1;
    if (!ok) flag_dev_err(a.err, kDevErrSampleParam);
  }
  return false;
}

__global__ __launch_bounds__(kSrThreads) void k_sr_hist(SampleRowsArgs a) {
  __shared__ SrHistShared sh;
  const int c = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int i0 = c * a.chunk, i1 = min(i0 + a.chunk, a.V);
  const SrSpace s = sr_space(a, b);
  const SrPart first = sr_part(a.logits + (int64_t)b * a.stride, i0, i1);
  SrRow r;
  if (!sr_begin(a, s, b, r, sh, false)) return;
  if (r.k == 0 && r.p >= 1.0) return;  // every bin is kept
  sr_chunk_hist(r, i0, i1, first, sh);
  // integers: no order changes the sums
  if (sh.mass[tid] > 0)
    __hip_atomic_fetch_add(s.mass + tid, sh.mass[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (sh.count[tid] > 0)
    __hip_atomic_fetch_add(s.count + tid, (u64)sh.count[tid], __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void sr_no_cut(SrFound& f) {
  if (threadIdx.x == 0) {
    f.lo = f.hi = f.bin_k = kSrBins;
    f.base = f.before_k = f.mass_k = f.need_k = 0;
  }
  __syncthreads();
}

__global__ __launch_bounds__(kSrThreads) void k_sr_pick(SampleRowsArgs a) {
  __shared__ SrShared sh;
  const int c = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int i0 = c * a.chunk, i1 = min(i0 + a.chunk, a.V);
  const SrSpace s = sr_space(a, b);
  const SrPart first = sr_part(a.logits + (int64_t)b * a.stride, i0, i1);
  const u64 count = s.count[tid], mass = s.mass[tid];
  SrRow r;
  if (!sr_begin(a, s, b, r, sh, true)) return;
  // every block for itself: an arrival in k_sr_hist and a scan by the row's last
  // block there made a row of 201088 1.5 us slower
  if (r.k > 0 || r.p < 1.0) sr_scan(r, count, mass, sh);
  else sr_no_cut(sh.found);
  const u64 sure = sr_collect(r, sh.found, i0, i1, first, sh);
  const int mine = sh.s_int[0];
  const int part = c * (a.chunk / kSrPart) + tid;
  if (tid < a.chunk / kSrPart && (int64_t)part * kSrPart < a.V) sr_put(s.sure + part, sure);
  if (tid == 0)
    sh.s_int[1] = mine > 0 ? __hip_atomic_fetch_add(s.n, mine, __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_AGENT) : 0;
  __syncthreads();
  const int at = sh.s_int[1];
  for (int j = tid; j < min(mine, kSrCap) && at + j < kSrCap; j += kSrThreads)
    sr_put(s.list + at + j, sh.list[j]);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores have completed
  __syncthreads();
  if (tid == 0) {
    sh.s_int[3] = __hip_atomic_fetch_add(s.n + 1, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (sh.s_int[3] != a.chunks - 1) return;
  // the row's last block; what it reads is requested together
  const int parts = (a.V + kSrPart - 1) / kSrPart;
  const int n = __hip_atomic_load(s.n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const u64 place = sr_get(s.list + tid), part_sure = tid < parts ? sr_get(s.sure + tid) : 0;
  if (tid < n) sh.list[tid] = place;
  for (int j = tid + kSrThreads; j < min(n, kSrCap); j += kSrThreads) sh.list[j] = sr_get(s.list + j);
  __syncthreads();
  const u64 cut = sr_cut(r, sh, n);
  const int id = sr_draw(r, sh, cut, [&](int p0) {
    const u64 own = p0 == 0 ? part_sure : p0 + tid < parts ? sr_get(s.sure + p0 + tid) : 0;
    return sr_part_mass(r, sh, cut, n, p0, own);
  });
  if (tid == 0) a.ids[b] = id;
}

// A row of one chunk: the same steps in one block.
__global__ __launch_bounds__(kSrThreads) void k_sr_one(SampleRowsArgs a) {
  __shared__ SrShared sh;
  const int b = blockIdx.x, tid = threadIdx.x;
  SrRow r;
  bool greedy;
  const bool ok = sr_params(a, b, sh.table, r, greedy);
  const u64 best = sr_chunk_max(r.l, 0, a.V, sh.red);
  sr_set_best(r, best);
  const bool none = (uint32_t)(best >> 32) <= kSrNone;
  if (!ok || none || greedy) {
    if (tid == 0) {
      a.ids[b] = ok && !none ? sr_best_id(best) : -1;
      if (!ok) flag_dev_err(a.err, kDevErrSampleParam);
    }
    return;
  }
  u64 cut = 0;
  if (r.k > 0 || r.p < 1.0) {
    sr_chunk_hist(r, 0, a.V, sr_part(r.l, 0, a.V), sh);
    sr_scan(r, sh.count[tid], sh.mass[tid], sh);
  } else {
    sr_no_cut(sh.found);
  }
  const u64 sure = sr_collect(r, sh.found, 0, a.V, sr_part(r.l, 0, a.V), sh);
  const int n = sh.s_int[0];
  if (r.k > 0 || r.p < 1.0) cut = sr_cut(r, sh, n);
  const int id = sr_draw(r, sh, cut, [&](int p0) { return sr_part_mass(r, sh, cut, n, p0, sure); });
  if (tid == 0) a.ids[b] = id;
}

// Tokens of a chunk, a multiple of kSrPart: as many chunks as k_sr_pick has places
// on the chip at once (two blocks of a CU; a second round would double it), of a
// part at least.
static int sr_chunk(int B, int V) {
  const int per_row = B < 512 ? 512 / B : 1;
  const int64_t chunk = (((int64_t)V + per_row - 1) / per_row + kSrPart - 1) / kSrPart * kSrPart;
  return chunk < kSrMaxChunk ? (int)chunk : kSrMaxChunk;
}

size_t sample_rows_needs(int B, int V) {
  const int C = (V + sr_chunk(B, V) - 1) / sr_chunk(B, V);
  return C == 1 ? 0 : (size_t)B * sr_space_bytes(C, V);
}
// The most that a batch of up to B rows needs: fewer rows are cut into more chunks
// each.  A chunk depends on 512 / B alone, so of the batches with the same quotient
// the largest needs the most.
size_t sample_rows_workspace(int B, int V) {
  size_t most = sample_rows_needs(B, V);
  for (int b = B < 512 ? B : 511; b >= 1; b = 512 / (512 / b + 1)) {
    const size_t n = sample_rows_needs(b, V);
    most = n > most ? n : most;
  }
  return most;
}

void launch_sample_rows(SampleRowsArgs a, hipStream_t st) {
  a.chunk = sr_chunk(a.B, a.V);
  a.chunks = (a.V + a.chunk - 1) / a.chunk;
  if (a.chunks == 1) {
    hipLaunchKernelGGL(k_sr_one, dim3(a.B), dim3(kSrThreads), 0, st, a);
    return;
  }
  const dim3 grid(a.chunks, a.B);
  hipLaunchKernelGGL(k_sr_max, grid, dim3(kSrThreads), 0, st, a);
  if (a.top_k != nullptr || a.top_p != nullptr)
    hipLaunchKernelGGL(k_sr_hist, grid, dim3(kSrThreads), 0, st, a);
  hipLaunchKernelGGL(k_sr_pick, grid, dim3(kSrThreads), 0, st, a);
}

}  // namespace neon
