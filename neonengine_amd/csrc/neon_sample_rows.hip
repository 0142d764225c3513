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
// order of threads or atomics changes a draw.  A token more than 31 below the
// maximum (in units of T) has mass 0 and cannot be drawn; its share is under
// 2^-44 of the most probable token's, below the 2^-24 steps of u.
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
__device__ __forceinline__ float sr_logit(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
constexpr uint32_t kSrNone = 0x007FFFFFu;  // key of minus infinity

struct SrRow {
  float m;       // the row's maximum
  double inv_t;  // 1 / T
  double scale;  // 2^S
  double min_p;
};
__device__ __forceinline__ double sr_weight(const SrRow& r, uint32_t key) {
  const float l = sr_logit(key);
  if (l == r.m) return 1.0;  // also where both are infinite
  return exp(((double)l - (double)r.m) * r.inv_t);
}
__device__ __forceinline__ u64 sr_mass(const SrRow& r, uint32_t key) {
  return (u64)__builtin_rint(sr_weight(r, key) * r.scale);
}

__device__ __forceinline__ double sr_scale(int V) {
  const int lg = V > 1 ? 32 - __builtin_clz((unsigned)(V - 1)) : 0;
  return lg <= 18 ? 0x1p44 : __builtin_ldexp(1.0, 62 - lg);
}

__device__ __forceinline__ u64 sr_block_sum(u64 v, u64* red) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) t += red[w];
  return t;
}
// sums of the threads before this one
__device__ __forceinline__ u64 sr_block_before(u64 v, u64* red) {
  u64 x = v;
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_up(x, o);
    if ((int)(threadIdx.x & 63) >= o) x += y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = x;
  __syncthreads();
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) x += red[w];
  return x - v;
}

// A row's parameters; false (flagged) where one is out of range.
__device__ __forceinline__ bool sr_params(const SampleRowsArgs& a, int b, float& t, int& k, float& p,
                                          float& mp, float& u) {
  t = a.temperature != nullptr ? a.temperature[b] : 1.0f;
  k = a.top_k != nullptr ? a.top_k[b] : 0;
  p = a.top_p != nullptr ? a.top_p[b] : 1.0f;
  mp = a.min_p != nullptr ? a.min_p[b] : 0.0f;
  u = a.u[b];
  return t >= 0.0f && t < INFINITY && p > 0.0f && p <= 1.0f && mp >= 0.0f && mp <= 1.0f &&
         u >= 0.0f && u < 1.0f;
}

// One block per row; the order is searched by 8 bits of the key at a time over
// the whole row (counts for top_k, masses for top_p).
__global__ __launch_bounds__(1024) void k_sample_rows(SampleRowsArgs a) {
  __shared__ u64 red[16], hist[256];
  __shared__ uint32_t s_key;
  __shared__ u64 s_above;
  __shared__ int s_id;
  const int b = blockIdx.x, tid = threadIdx.x;
  const float* l = a.logits + (int64_t)b * a.stride;
  const int V = a.V;
  float t, p, mp, u;
  int k;
  if (!sr_params(a, b, t, k, p, mp, u)) {
    if (tid == 0) {
      flag_dev_err(a.err, kDevErrSampleParam);
      a.ids[b] = -1;
    }
    return;
  }
  // the maximum, lowest index first
  u64 best = 0;
  for (int i = tid; i < V; i += 1024) {
    const u64 x = ((u64)sr_key(l[i]) << 32) | (uint32_t)~i;
    best = x > best ? x : best;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const u64 x = __shfl_xor(best, o);
    best = x > best ? x : best;
  }
  if ((tid & 63) == 0) red[tid >> 6] = best;
  __syncthreads();
  for (int w = 0; w < 16; ++w) best = red[w] > best ? red[w] : best;
  const uint32_t top = (uint32_t)(best >> 32);
  if (top == kSrNone || t == 0.0f) {  // nothing to choose from, or greedy
    if (tid == 0) a.ids[b] = top == kSrNone ? -1 : (int32_t)~(uint32_t)best;
    return;
  }
  SrRow r;
  r.m = sr_logit(top);
  r.inv_t = 1.0 / (double)t;
  r.scale = sr_scale(V);
  r.min_p = (double)mp;

  // The largest key whose elements and those above it reach `goal`, in
  // elements (by = false) or mass; `above`: what the larger keys have.
  auto search = [&](bool by_mass, double goal, uint32_t floor_key, u64& above) {
    uint32_t prefix = 0;
    u64 before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += 1024) {
        const uint32_t x = sr_key(l[i]);
        if (x < floor_key || (shift < 24 && (x >> (shift + 8)) != prefix)) continue;
        const u64 w = by_mass ? sr_mass(r, x) : 1;
        if (w) atomicAdd(&hist[(x >> shift) & 255], w);
      }
      __syncthreads();
      if (tid == 0) {
        u64 run = before;
        int d = 255;
        for (; d > 0; --d) {
          if ((double)(run + hist[d]) >= goal) break;
          run += hist[d];
        }
        s_key = d;
        s_above = run;
      }
      __syncthreads();
      prefix = (prefix << 8) | s_key;
      before = s_above;
    }
    above = before;
    return prefix;
  };
  auto total = [&](uint32_t key, bool by_mass) {  // of larger keys' elements
    u64 n = 0;
    for (int i = tid; i < V; i += 1024) {
      const uint32_t x = sr_key(l[i]);
      if (x > key) n += by_mass ? sr_mass(r, x) : 1;
    }
    return sr_block_sum(n, red);
  };

  // kept: keys above `key`, and the first `ties` indexes with the key itself
  uint32_t key = 0;
  u64 ties = ~0ull;
  if (k > 0 && k < V) {
    u64 above;
    key = search(false, (double)k, 0, above);
    ties = k - above;
  }
  if (p < 1.0f) {
    u64 above, kept = total(key, true);
    if (ties != ~0ull) kept += ties * sr_mass(r, key);
    const double goal = (double)p * (double)kept;
    const uint32_t pk = search(true, goal, key, above);
    const u64 w = sr_mass(r, pk);
    const u64 cap = pk == key ? ties : ~0ull;
    if (w > 0) {
      u64 n = (u64)ceil((goal - (double)above) / (double)w);
      if (n < 1) n = 1;
      ties = n < cap ? n : cap;
      key = pk;
    }
  }
  // the draw, in index order: thread tid owns a contiguous slice
  const int C = (V + 1023) / 1024, i0 = min(tid * C, V), i1 = min(i0 + C, V);
  const u64 tie_mass = key != 0 && sr_weight(r, key) >= r.min_p ? sr_mass(r, key) : 0;
  u64 gt = 0, eq = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t x = sr_key(l[i]);
    if (x > key && sr_weight(r, x) >= r.min_p) gt += sr_mass(r, x);
    eq += x == key;
  }
  const u64 eq_before = sr_block_before(eq, red);
  const u64 eq_kept = eq_before >= ties ? 0 : (eq < ties - eq_before ? eq : ties - eq_before);
  const u64 own = gt + eq_kept * tie_mass;
  const u64 before = sr_block_before(own, red);
  const double target = (double)u * (double)sr_block_sum(own, red);
  if (tid == 0) s_id = (int)~(uint32_t)best;
  __syncthreads();
  if (own > 0 && (double)before <= target && (double)(before + own) > target) {
    u64 run = before, seen = eq_before;
    for (int i = i0; i < i1; ++i) {
      const uint32_t x = sr_key(l[i]);
      if (x == key) {
        if (seen < ties) run += tie_mass;
        ++seen;
      } else if (x > key && sr_weight(r, x) >= r.min_p) {
        run += sr_mass(r, x);
      }
      if ((double)run > target) {
        s_id = i;
        break;
      }
    }
  }
  __syncthreads();
  if (tid == 0) a.ids[b] = s_id;
}

void launch_sample_rows(const SampleRowsArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(k_sample_rows, dim3(a.B), dim3(1024), 0, st, a);
}

}  // namespace neon
