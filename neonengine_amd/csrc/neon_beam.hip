// neon_beam.hip -- beam search: the choice of the next beams from the logits, and
// the move of the beams' states in place.
//
// Choice.  For request b, place w, token t:  v = s_w + l_wt - lse_w, with
// lse_w = m + log(sum_t exp(l_wt - m)), all in 64 bits.  Candidates are ordered by
// (v descending, place ascending, token ascending).  Stop tokens among the W best
// end; the W best others go on.  The best child of a beam takes its place, the
// other children the free places, in their order.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "neon_common.hpp"
#include "neon_internal.hpp"

namespace neon {

typedef unsigned long long u64;
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---------------------------------------------------------------------------
// The K best of what a wave sees.  The K-th largest of the lanes' maxima is a bound (K
// lanes hold something at least as large): what reaches it goes into a list in LDS, and its
// order is found by counting.  Few others reach it where the lanes see alike.  They do in a
// row's tokens; in the join lane i reads keys 64 h + i of ordered lists of K, so where K
// divides 64 a lane sees one rank of all lists and the bound is loose (2 requests of 32
// beams, 88480 tokens: 62 us with K = 32, 43 with 33; one of 16, 201088: 25.5 with 16,
// 19.7 with 17).
// ---------------------------------------------------------------------------
__device__ __forceinline__ u64 bm_lane_key(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)v, lane) |
         (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32;
}
// The largest x, of the upper 16 bits, that K of the wave's values reach; 0 where fewer
// than K lanes have a value.  Two bits at a time: the three counts of a step do not wait
// for each other.
__device__ __forceinline__ uint32_t bm_kth(uint32_t v, int K) {
  uint32_t x = 0;
#pragma unroll
  for (int bit = 30; bit >= 16; bit -= 2) {
    const uint32_t y1 = x | 1u << bit, y2 = x | 2u << bit, y3 = x | 3u << bit;
    const int n1 = __builtin_popcountll(__ballot(v >= y1));
    const int n2 = __builtin_popcountll(__ballot(v >= y2));
    const int n3 = __builtin_popcountll(__ballot(v >= y3));
    x = n3 >= K ? y3 : n2 >= K ? y2 : n1 >= K ? y1 : x;
  }
  return x;
}
// this lane's place among the set lanes of a mask
__device__ __forceinline__ int bm_rank(u64 mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// A wave's list of the best keys so far (unique; 0: none).
constexpr int kBmFull = 128;           // with more than these it is cut down to K
constexpr int kBmList = kBmFull + 64;  // 64 at most are added at once
struct BmList {
  u64* key;           // LDS, kBmList of the wave's own
  int n = 0;
  uint32_t least = 0x00800000u;  // upper halves below it are not among the K best (all logits
                                 // above minus infinity reach this one)
  u64 last = 0;        // nor are keys up to this one
  __device__ __forceinline__ explicit BmList(u64* p) : key(p) {}
  // a bound from the lanes' maxima of something that is added next
  __device__ __forceinline__ void bound(uint32_t top, int K) { least = max(least, bm_kth(top, K)); }
  // (n is at most kBmFull)
  __device__ __forceinline__ void add(u64 k) {
    const bool is = (uint32_t)(k >> 32) >= least && k > last;
    const u64 in = __ballot(is);
    if (is) key[n + bm_rank(in)] = k;
    n += __builtin_popcountll(in);
  }
  // the K best, in order
  __device__ __forceinline__ void cut(int K) {
    const int lane = threadIdx.x & 63;
    wave_lds_sync();
    u64 k[3];
#pragma unroll
    for (int h = 0; h < 3; ++h) k[h] = 64 * h + lane < n ? key[64 * h + lane] : 0;
    bound((uint32_t)(max(max(k[0], k[1]), k[2]) >> 32), K);
    wave_lds_sync();
#pragma unroll
    for (int h = 0; h < 3; ++h) {
      u64 in = __ballot((uint32_t)(k[h] >> 32) >= least);
      while (in != 0) {
        const int j = __builtin_ctzll(in);
        in &= in - 1;
        const u64 x = bm_lane_key(k[h], j);
        const int at = __builtin_popcountll(__ballot(k[0] > x)) + __builtin_popcountll(__ballot(k[1] > x)) +
                       __builtin_popcountll(__ballot(k[2] > x));
        if (at < K && lane == j) key[at] = x;
      }
    }
    wave_lds_sync();
    if (n >= K) last = max(last, key[K - 1]);
    n = min(n, K);
  }
};

// Keys of a list that come before `mine`: every lane reads the same ones, so nothing goes
// through scalar registers.  Entries from n to the next multiple of 8 are read: `pad` gives
// them 0, by one wave, before a barrier.
__device__ __forceinline__ void bm_pad(u64* key, int n) {
  const int lane = threadIdx.x & 63;
  if (lane < 8) key[n + lane] = 0;
}
__device__ __forceinline__ int bm_before(const u64* key, int n, u64 mine) {
  int p = 0;
  for (int j = 0; j < n; j += 8)
#pragma unroll
    for (int i = 0; i < 8; ++i) p += key[j + i] > mine;
  return p;
}

// x[e] for a lane's own e, N a power of two: a choice by each bit of e, as bit masks (a
// condition on array elements would put the array into memory)
template <int N>
__device__ __forceinline__ uint32_t bm_pick(const uint32_t (&x)[N], int e) {
  if constexpr (N == 1) {
    return x[0];
  } else {
    const uint32_t odd = -(uint32_t)(e & 1);
    uint32_t y[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) y[i] = (x[2 * i + 1] & odd) | (x[2 * i] & ~odd);
    return bm_pick<N / 2>(y, e >> 1);
  }
}

// Order of a logit as an integer: larger logit, larger key; both zeros are one, and
// minus infinity is 0 (no candidate).
__device__ __forceinline__ uint32_t bm_ordered(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);  // -0 + 0 = +0
  return l == -INFINITY ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bm_logit(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// unique, and in the order of the tokens: larger logit, then lower token
__device__ __forceinline__ u64 bm_key(float l, int token) {
  const uint32_t o = bm_ordered(l);
  return o == 0 ? 0 : (u64)o << 32 | (uint32_t)~token;
}
// the order of a 64-bit value above minus infinity
__device__ __forceinline__ u64 bm_ordered64(double v) {
  const u64 b = __builtin_bit_cast(u64, v + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double bm_value64(u64 k) {
  return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

// exp(x) for x up to kBmAbove: 2^f by a polynomial of degree 9 on [-1/2, 1/2]
// (interpolated at the Chebyshev points, 1.9e-14), the exponent added as an integer.  x / ln 2
// is rounded, so the error is 1.9e-14 + |x| 2^-53 of the value: 2^-45 near the largest, whose
// sum this is for, under 1e-13 at -700.  2^-1020 stands for all below it; what comes of larger x
// (past the exponents, garbage) is not used.  The coefficients stay in scalar registers: as
// literals each would be moved into vector registers first.
struct BmExp {
  double c[10];
  __device__ __forceinline__ BmExp()
      : c{0x1.000000000003dp+0,  0x1.62e42fefa39f7p-1,  0x1.ebfbdff8149f2p-3,  0x1.c6b08d7044117p-5,
          0x1.3b2ab72b175e1p-7,  0x1.5d87fe908fb19p-10, 0x1.43088e2580989p-13, 0x1.ffcb767842e11p-17,
          0x1.63ef9699120e2p-20, 0x1.b6571e229927fp-24} {
#pragma unroll
    for (int i = 0; i < 10; ++i) asm("" : "+s"(c[i]));
  }
  __device__ __forceinline__ double operator()(double x) const {
    constexpr double kMagic = 0x1.8p52;  // its sum's low bits are the nearest integer
    const double t = fmax(x * 1.4426950408889634074, -1020.0);
    const double r = t + kMagic;
    const double f = t - (r - kMagic);
    double p = c[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) p = __builtin_fma(p, f, c[i]);
    const u64 b = __builtin_bit_cast(u64, p);
    const uint32_t n = (uint32_t)__builtin_bit_cast(u64, r);
    return __builtin_bit_cast(double, b + ((u64)(n << 20) << 32));
  }
};

template <int OFF = 32>
__device__ __forceinline__ double bm_wave_sum(double v) {
  const u64 b = __builtin_bit_cast(u64, v);
  const uint32_t lo = (uint32_t)xor_lane_i<OFF>((int)(uint32_t)b);
  const uint32_t hi = (uint32_t)xor_lane_i<OFF>((int)(uint32_t)(b >> 32));
  v += __builtin_bit_cast(double, (u64)lo | (u64)hi << 32);
  if constexpr (OFF > 1) return bm_wave_sum<OFF / 2>(v);
  return v;
}

// A beam that has a score to go on from.
__device__ __forceinline__ bool bm_alive(float score) { return score > -INFINITY && score < INFINITY; }

// ---------------------------------------------------------------------------
// A chunk of a row: the sum of exponentials and its K = W + n_stop best tokens (of
// W + n_stop at least W are no stop tokens, and a stop token that is not among them has W
// better ones in its own row).  A wave requests all its tokens at once, up to kBmGroups
// groups of 256 (4 of a lane), and takes the exponentials of a group as it comes: relative
// to the maximum of the first one, and only where a later one is more than 64 above are
// they taken again (the sum is as exact).  Then the maxima of the block's lanes give the
// bound of its list, which about K of its tokens reach.
// Bound: the vector units beside the reads.  64 rows of 201088: 19.5 us, 51.5 MB, floor
// 10.3; 500 vector instructions for 1024 tokens of a wave, 307 of them the exponentials
// (19 each, 64-bit ones at one in 4 cycles), are 12 us of all SIMDs.  Without the exponentials it takes 16, without the list 16.5, without both
// 12.  4, 5, 7, 8, 10 and 13 groups, in places for as many blocks as run at once, came to
// 18 to 21 us; two steps of 1024 with the next on its way to 22.  4 rows: 5.3 us (0.3 until
// the tokens are there, 0.9 exponentials, 0.5 the bound, 0.3 the list, 0.9 the rest).
// ---------------------------------------------------------------------------
constexpr int kBmGroups = 8;  // (4 kBmGroups bits of a word)
constexpr float kBmAbove = 64.0f;
struct __align__(16) BmSum {
  double s;  // sum of exp(l - m)
  float m;   // -inf: no token, +inf: a logit of it
  float pad;
};

// Group k of a wave: lane i has the tokens t0 + 256 k + 4 i .. + 3.  A row begins at any
// multiple of 4 bytes; which lane takes a token does not depend on it, so equal rows have
// equal sums, and equal beams are ordered by their places.  Tokens past the end are minus
// infinity, groups past the wave's the last one again (a load under a condition of its own
// is waited for where the paths join).
typedef float bm_f4 __attribute__((ext_vector_type(4), aligned(4)));
template <int NG>
__device__ __forceinline__ void bm_load(const float* row, int V, int t0, int groups, int lane,
                                        float (&x)[4 * NG]) {
  if (t0 + 256 * groups <= V) {
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const bm_f4 v = *reinterpret_cast<const bm_f4*>(row + t0 + 256 * min(k, groups - 1) + 4u * lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * k + j] = v[j];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4 * NG; ++e) {
      const int t = t0 + 256 * min(e >> 2, groups - 1) + 4 * lane + (e & 3);
      const float v = row[(uint32_t)min(t, V - 1)];
      x[e] = t < V ? v : -INFINITY;
    }
  }
}

template <int NG>
__global__ __launch_bounds__(256) void k_beam_part(BeamSelectArgs a) {
  __shared__ u64 keys[4][kBmList];
  __shared__ double sums[4][64];
  __shared__ float tops[4][64];
  __shared__ u64 joint[4 * 64 + 8];
  __shared__ int total;
  __shared__ float ms[4];
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  if (!bm_alive(a.score[row])) return;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int K = a.K;
  const int first = (chunk * 4 + wave) * a.groups * 256;
  const int groups = first < a.V ? min(a.groups, (a.V - first + 255) >> 8) : 0;
  const BmExp exp_of;
  float x[4 * NG], top = -INFINITY, m = -INFINITY;
  double s[2];
  if (groups > 0) {
    bm_load<NG>(a.logits + (int64_t)row * a.stride, a.V, first, groups, lane, x);
    // a NaN is a quiet one from here on: maxima pass it over, comparisons fail
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __builtin_canonicalizef(x[j]);
    m = wave_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), -INFINITY));
    for (bool again = true; again;) {
      const double md = m == -INFINITY ? 0.0 : (double)m;
      s[0] = s[1] = 0.0;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        if (k < groups) {
          float* y = x + 4 * k;
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = __builtin_canonicalizef(y[j]);
          top = fmaxf(top, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
#pragma unroll
          for (int j = 0; j < 4; ++j) s[j & 1] += exp_of((double)y[j] - md);
        }
      }
      again = __any((top > m + kBmAbove) | ((m == -INFINITY) & (top > m)));
      if (again) m = wave_max(top);
    }
  }
  tops[wave][lane] = top;
  for (int i = threadIdx.x; i < 4 * 64 + 8; i += 256) joint[i] = 0;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const float all4 = fmaxf(fmaxf(tops[0][lane], tops[1][lane]), fmaxf(tops[2][lane], tops[3][lane]));
  BmList list(keys[wave]);
  list.bound(bm_ordered(all4), K);
  const float least = bm_logit(list.least);
  // which of the lane's logits reach the bound: bit e
  uint32_t reach = 0;
  if (groups > 0) {
#pragma unroll
    for (int e = 4 * NG - 1; e >= 0; --e) reach = reach + reach + (x[e] >= least ? 1u : 0u);
    if (groups < NG) reach &= (1u << 4 * groups) - 1;
  }
  while (__any(reach != 0)) {  // every lane its next one
    const int e = __builtin_ctz(reach | 1u << 31);
    uint32_t bits[4 * NG];
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i) bits[i] = __float_as_uint(x[i]);
    const float v = __uint_as_float(bm_pick<4 * NG>(bits, e));
    list.add(reach != 0 ? bm_key(v, first + 256 * (e >> 2) + 4 * lane + (e & 3)) : 0);
    reach &= reach - 1;
    if (list.n > kBmFull) list.cut(K);
  }
  if (list.n > 64) list.cut(K);
  sums[wave][lane] = groups > 0 && m != -INFINITY ? s[0] + s[1] : 0.0;
  // the waves' lists as one, in any order
  int base = 0;
  if (lane == 0) {
    base = atomicAdd(&total, list.n);
    ms[wave] = m;
  }
  base = uni(base);
  wave_lds_sync();  // the list's keys are other lanes'
  if (lane < list.n) joint[base + lane] = keys[wave][lane];
  __syncthreads();
  const int all = total, i = threadIdx.x;
  const int64_t at = (int64_t)row * a.chunks + chunk;
  if (i < all) {
    const u64 mine = joint[i];
    const int place = bm_before(joint, all, mine);
    if (place < K) a.keys[at * K + place] = mine;
  }
  if (i >= all && i < K) a.keys[at * K + i] = 0;
  if (wave == 3) {
    const float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const double f = ms[w] == -INFINITY ? 0.0 : exp_of((double)ms[w] - (double)M);
      sum += sums[w][lane] * f;
    }
    sum = bm_wave_sum(sum);
    if (lane == 0) {
      a.sums[at].s = sum;
      a.sums[at].m = M;
    }
  }
}

// ---------------------------------------------------------------------------
// A request: the K best of each row (a wave each), then the W best that go on and the
// stop tokens among the W best.
// Bound: a chain of dependent steps of one block (4 beams 5.4 us: 1 until the chunks'
// results are there, 0.6 the sum, 0.5 the bound, 0.9 the list and its order, 0.8 the places
// among all, 0.8 the rest, the launch), and from 8 beams on the instructions of four waves
// a SIMD (16 beams 8.6 us).  A step that goes through scalar registers costs some 40 ns:
// orders are counted from LDS broadcasts (5 keys put in their places one after another
// took 1.4 us).
// ---------------------------------------------------------------------------
constexpr int kBmMaxK = kBeamMaxW + kBeamMaxStop;
constexpr int kBmJoinWaves = 16;
constexpr int kBmOpen = kBeamMaxW * kBmMaxK;
// AHEAD: keys of a lane that are requested at once, 4 where all of a row are so (16 beams
// 8.6 us, with 8 9.1; 4 beams of 25 chunks 5.7 and 5.8).
template <int AHEAD>
__global__ __launch_bounds__(64 * kBmJoinWaves) void k_beam_join(BeamSelectArgs a) {
  __shared__ u64 lists[kBmJoinWaves][kBmList + 8];
  __shared__ u64 value[kBmOpen];  // of (place, rank), ordered; 0: none
  __shared__ int token[kBmOpen];  // | place << 24, negative: a stop token
  __shared__ u64 key_all[kBmOpen + 8], key_live[kBmOpen + 8];
  __shared__ int from[kBmOpen], total;
  __shared__ uint32_t bound;
  __shared__ float best;
  __shared__ int stop[kBeamMaxStop];
  __shared__ int next[kBeamMaxW], over[kBeamMaxW], to_free[kBeamMaxW], child[kBeamMaxW];
  const int b = blockIdx.x, W = a.W, K = a.K, waves = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const BmExp exp_of;
  if ((int)threadIdx.x < a.n_stop) stop[threadIdx.x] = a.stop[threadIdx.x];
  if (threadIdx.x < kBeamMaxW) {
    next[threadIdx.x] = over[threadIdx.x] = -1;
    child[threadIdx.x] = kBeamMaxW;  // the first child of the beam in this place
  }
  for (int i = threadIdx.x; i < W * K + 8; i += blockDim.x) key_all[i] = key_live[i] = 0;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  for (int w = wave; w < W; w += waves) {
    const int row = b * W + w, all = a.chunks * K;
    const BmSum* sums = a.sums + (int64_t)row * a.chunks;
    const u64* keys = a.keys + (int64_t)row * all;
    // what the row's chunks left, on its way at once (a row without a beam has nothing
    // there that is used)
    const float score = a.score[row];
    BmSum sum = sums[min(lane, a.chunks - 1)];
    u64 k[AHEAD];
#pragma unroll
    for (int h = 0; h < AHEAD; ++h) k[h] = keys[min(64 * h + lane, all - 1)];
    bool alive = bm_alive(score);
    if (lane == 0 && (score != score || score == INFINITY)) flag_dev_err(a.err, kDevErrBeam);
    double lse = 0.0;
    BmList list(lists[wave]);
    if (alive) {
      float m = lane < a.chunks ? sum.m : -INFINITY;
      for (int c = 64 + lane; c < a.chunks; c += 64) m = fmaxf(m, sums[c].m);
      m = wave_max(m);
      double s = 0.0;
      for (int c = lane; c < a.chunks; c += 64) {
        if (c != lane) sum = sums[c];
        if (sum.m != -INFINITY) s += sum.s * exp_of((double)sum.m - (double)m);
      }
      s = bm_wave_sum(s);
      if (lane == 0 && m == INFINITY) flag_dev_err(a.err, kDevErrBeam);
      alive = m > -INFINITY && m < INFINITY;
      lse = (double)m + log(s);
    }
    if (alive) {
      for (int i0 = 0; i0 < all; i0 += 64 * AHEAD) {
        if (i0 > 0)
#pragma unroll
          for (int h = 0; h < AHEAD; ++h) k[h] = keys[min(i0 + 64 * h + lane, all - 1)];
        u64 top = 0;
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
          k[h] = i0 + 64 * h + lane < all ? k[h] : 0;
          top = max(top, k[h]);
        }
        list.bound((uint32_t)(top >> 32), K);
        uint32_t reach = 0;  // bit h: the lane's k[h] does (past the keys: 0, which does not)
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) reach |= (uint32_t)((uint32_t)(k[h] >> 32) >= list.least) << h;
        while (__any(reach != 0)) {  // every lane its next one
          uint32_t lo[AHEAD], hi[AHEAD];
#pragma unroll
          for (int h = 0; h < AHEAD; ++h) {
            lo[h] = (uint32_t)k[h];
            hi[h] = (uint32_t)(k[h] >> 32);
          }
          const int h = __builtin_ctz(reach | 1u << 31);
          list.add(reach != 0 ? (u64)bm_pick(hi, h) << 32 | bm_pick(lo, h) : 0);
          reach &= reach - 1;
          if (list.n > kBmFull) list.cut(K);
        }
      }
      if (list.n > 64) list.cut(K);
    }
    bm_pad(lists[wave], list.n);
    wave_lds_sync();
    const u64 mine = lane < list.n ? lists[wave][lane] : 0;
    const int place = bm_before(lists[wave], list.n, mine);
    if (lane < list.n && place < K) {
      const int t = (int)~(uint32_t)mine;
      const double v = (double)score + ((double)bm_logit((uint32_t)(mine >> 32)) - lse);
      value[w * K + place] = bm_ordered64(v);
      bool is = false;
      for (int j = 0; j < a.n_stop; ++j) is |= t == stop[j];
      token[w * K + place] = t | w << 24 | (is ? 1 << 31 : 0);
    }
    if (lane < K && lane >= list.n) value[w * K + lane] = 0;
    wave_lds_sync();  // the list is free
  }
  __syncthreads();
  // every candidate's place among all, if it is a stop token, or among those that are
  // none: larger values before it, and equal ones of a lower index.  Of more than 64, those
  // that cannot be among the W best are left out first.
  const int all = W * K;
  // (as distances from the best, whose upper 16 bits are fine near it)
  auto near = [&](u64 v) { return v == 0 ? 0u : bm_ordered((float)(bm_value64(v) - (double)best)); };
  if (all > 64) {
    if (wave == 0) {
      u64 top = 0;
      for (int i = lane; i < all; i += 64) top = max(top, token[i] < 0 ? 0 : value[i]);
      const float x = wave_max(top == 0 ? -INFINITY : (float)bm_value64(top));
      if (lane == 0) best = x;
      wave_lds_sync();
      const uint32_t y = bm_kth(near(top), W);
      if (lane == 0) bound = y;
    }
    __syncthreads();
  }
  const uint32_t least = all > 64 ? bound : 0;
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const u64 v = value[i];
    if (v == 0 || (least != 0 && near(v) < least)) continue;
    const int at = atomicAdd(&total, 1);
    key_all[at] = v;
    key_live[at] = token[i] < 0 ? 0 : v;
    from[at] = i;
  }
  __syncthreads();
  const int n = total;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const u64 v = key_all[c];
    const bool is = key_live[c] == 0;
    const u64* among = is ? key_all : key_live;
    int more = 0, as_much = 0;
    for (int j = 0; j < n; j += 8)
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const u64 x = among[j + g];
        more += x > v;
        as_much += x >= v;
      }
    if (as_much - more > 1)  // (itself, and equal ones)
      for (int j = 0; j < n; ++j) more += among[j] == v && from[j] < from[c];
    if (more < W) (is ? over : next)[more] = from[c];
  }
  __syncthreads();
  if (wave > 1) return;
  const int i = lane < W ? (wave == 0 ? next : over)[lane] : -1;
  const int tok = i >= 0 ? token[i] & 0xFFFFFF : -1, place = i >= 0 ? token[i] >> 24 & 31 : -1;
  const float v = i >= 0 ? (float)bm_value64(value[i]) : -INFINITY;
  if (wave == 1) {  // (places between stop tokens are empty)
    if (a.end_token == nullptr) return;
    const u64 in = __ballot(i >= 0);
    const int n_in = __builtin_popcountll(in);
    if (lane < W) {
      const int at = b * W + (i >= 0 ? bm_rank(in) : n_in + bm_rank(~in));
      a.end_token[at] = tok;
      a.end_parent[at] = i >= 0 ? b * W + place : -1;
      a.end_score[at] = v;
    }
    return;
  }
  // the first child of a beam keeps its place; the others take the free ones in order
  if (i >= 0) atomicMin(&child[place], lane);
  wave_lds_sync();
  const bool keeps = i >= 0 && child[place] == lane;
  const u64 taken = __ballot(lane < W && child[min(lane, W - 1)] < W);
  const u64 open = __ballot(lane < W && !(taken >> lane & 1));
  if (open >> lane & 1) to_free[bm_rank(open)] = lane;
  const u64 movers = __ballot(lane < W && !keeps);
  wave_lds_sync();
  if (lane < W) {
    const int to = b * W + (keeps ? place : to_free[bm_rank(movers)]);
    a.token[to] = tok;
    a.parent[to] = i >= 0 ? b * W + place : -1;
    a.out_score[to] = v;
  }
}

// Groups of a wave: about as many blocks as run at once, where there are enough tokens, 6
// of each CU (k_beam_part<4> in 64 registers has 8 places there, <8> in 87 5: 16 requests of 4
// beams, 201088 tokens, take 24.9 us in a graph with 1280 as with 1536, 2 of 32 beams, 88480
// tokens, 53.5 and 62.3); no fewer than 4 groups, since the join takes the chunks' keys one
// row after another.
constexpr int64_t kBmPlaces = 1536;
static int beam_groups(int64_t rows, int V) {
  const int64_t chunks = std::max<int64_t>(1, kBmPlaces / rows);
  const int64_t groups = ((int64_t)V + 1024 * chunks - 1) / (1024 * chunks);
  return (int)std::min<int64_t>(std::max<int64_t>(groups, 4), kBmGroups);
}
static int beam_chunks(int V, int groups) {
  const int64_t per = 1024 * (int64_t)groups;
  return (int)(((int64_t)V + per - 1) / per);
}
constexpr int64_t kBmMaxBlocks = 1 << 24;  // of 256 threads: a launch holds fewer than 2^32
bool beam_select_fits(int B, int W, int V) {
  const int64_t rows = (int64_t)B * W;
  return rows * beam_chunks(V, beam_groups(rows, V)) < kBmMaxBlocks;
}
static size_t beam_chunk_bytes(int K) { return (size_t)K * 8 + sizeof(BmSum); }
size_t beam_select_needs(int B, int W, int V, int n_stop) {
  const int64_t rows = (int64_t)B * W;
  return (size_t)rows * beam_chunks(V, beam_groups(rows, V)) * beam_chunk_bytes(W + n_stop);
}
// Fewer rows may be cut into more chunks, but into no more than run at once, or than
// those of the most groups.
size_t beam_select_workspace(int B, int W, int V, int n_stop) {
  const int64_t rows = (int64_t)B * W;
  const int64_t chunks = std::min(rows * beam_chunks(V, 4),
                                  std::max(kBmPlaces + rows, rows * beam_chunks(V, kBmGroups)));
  return (size_t)chunks * beam_chunk_bytes(W + n_stop);
}
void launch_beam_select(BeamSelectArgs a, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.W;
  a.groups = beam_groups(rows, a.V);
  a.chunks = beam_chunks(a.V, a.groups);
  a.K = a.W + a.n_stop;
  a.sums = (BmSum*)a.workspace;
  a.keys = (u64*)(a.sums + (size_t)rows * a.chunks);
  const dim3 grid((unsigned)(rows * a.chunks));
  if (a.groups > 4) hipLaunchKernelGGL(k_beam_part<kBmGroups>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(k_beam_part<4>, grid, dim3(256), 0, st, a);
  const int waves = std::min(std::max(a.W, 2), kBmJoinWaves);
  const dim3 requests((unsigned)a.B), threads(64 * waves);
  if (a.chunks * a.K > 256) hipLaunchKernelGGL(k_beam_join<8>, requests, threads, 0, st, a);
  else hipLaunchKernelGGL(k_beam_join<4>, requests, threads, 0, st, a);
}

constexpr int kReorderUnits = 4;  // 1, 2, 4, 8: 24, 22.6, 22.6, 31 us (136 MB, see below)
// ---------------------------------------------------------------------------
// Moving states.  A block takes the same part of a slab in all beams of a request, U
// units of a thread.  Where no beam that moves is also one that others continue (beams
// that go on keep their places), each is copied for itself; otherwise a thread reads all
// that move to its places before it writes any, so the move is in place whatever the
// parents are (a permutation too).
// Bound: the bytes read and written (11 of 32 beams of up to 2000 tokens in four states,
// 136 MB: 22.5 us, 6.0 TB/s, part of what is read being in the last-level cache; a large
// copy 4.98).
// ---------------------------------------------------------------------------
template <class T, int WMAX>
__global__ __launch_bounds__(256) void k_beam_reorder(BeamReorderArgs a) {
  constexpr int U = kReorderUnits;
  // block: (state, request, slab, part of the slab)
  int id = blockIdx.x;
  const int part = id % a.parts;
  id /= a.parts;
  const int slab = id % a.slabs;
  id /= a.slabs;
  const int g = id % a.groups, x = id / a.groups;
  const int lane = threadIdx.x & 63;
  // lane = place: where its row comes from, and how many units of it
  int p = -1;
  int64_t n = 0;
  if (lane < a.W) {
    p = a.parent[g * a.W + lane] - g * a.W;
    if ((unsigned)p >= (unsigned)a.W) {
      if (p != -1 - g * a.W && threadIdx.x < 64 && part == 0 && slab == 0 && x == 0)
        flag_dev_err(a.err, kDevErrBeam);
      p = -1;
    }
    if (p == lane) p = -1;
    if (p >= 0) n = (int64_t)(a.len != nullptr ? min(max(a.len[g * a.W + p], 0), a.T) : a.T) * a.per;
  }
  const int64_t i0 = (int64_t)part * (256 * U);
  uint64_t moved = __ballot(p >= 0 && n > i0);
  if (moved == 0) return;
  bool clash = false;
  for (uint64_t in = moved; in != 0; in &= in - 1)
    clash |= (moved >> __builtin_amdgcn_readlane(p, __builtin_ctzll(in)) & 1) != 0;
  T* base = reinterpret_cast<T*>(a.state[x]) + (int64_t)g * a.W * a.seq + slab * a.slab;
  auto from = [&](int w) { return base + (int64_t)__builtin_amdgcn_readlane(p, w) * a.seq; };
  auto units = [&](int w) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)n, w) |
           (int64_t)__builtin_amdgcn_readlane((int)(n >> 32), w) << 32;
  };
  if (!clash) {
    for (; moved != 0; moved &= moved - 1) {
      const int w = __builtin_ctzll(moved);
      const T* src = from(w);
      T* dst = base + (int64_t)w * a.seq;
      const int64_t end = units(w);
      T v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * 256 + threadIdx.x < end) v[u] = src[i0 + u * 256 + threadIdx.x];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * 256 + threadIdx.x < end) stream_store(dst + i0 + u * 256 + threadIdx.x, v[u]);
    }
    return;
  }
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * 256 + threadIdx.x;
    T v[WMAX];
#pragma unroll
    for (int w = 0; w < WMAX; ++w)
      if ((moved >> w & 1) != 0 && i < units(w)) v[w] = from(w)[i];
#pragma unroll
    for (int w = 0; w < WMAX; ++w)
      if ((moved >> w & 1) != 0 && i < units(w)) stream_store(base + (int64_t)w * a.seq + i, v[w]);
  }
}

static int64_t reorder_units(const BeamReorderArgs& a) {  // of a slab
  return (int64_t)a.T * (a.row_bytes % 16 == 0 ? a.row_bytes / 16 : a.row_bytes / 4);
}
bool beam_reorder_fits(const BeamReorderArgs& a) {
  const int64_t parts = (reorder_units(a) + 256 * kReorderUnits - 1) / (256 * kReorderUnits);
  return parts < kBmMaxBlocks && parts * a.slabs < kBmMaxBlocks &&
         parts * a.slabs * a.groups < kBmMaxBlocks;
}
void launch_beam_reorder(BeamReorderArgs a, void* const* states, int n_states, hipStream_t st) {
  const bool wide = a.row_bytes % 16 == 0;
  a.per = wide ? a.row_bytes / 16 : a.row_bytes / 4;
  a.slab = (int64_t)a.T * a.per;
  a.seq = a.slab * a.slabs;
  a.parts = (int)((a.slab + 256 * kReorderUnits - 1) / (256 * kReorderUnits));
  const int64_t blocks = (int64_t)a.parts * a.slabs * a.groups;  // of a state
  const int most = (int)std::min<int64_t>(kBeamStates, (kBmMaxBlocks - 1) / blocks);
  for (int x0 = 0, n; x0 < n_states; x0 += n) {
    n = std::min(n_states - x0, most);
    for (int x = 0; x < n; ++x) a.state[x] = states[x0 + x];
    const dim3 grid((unsigned)(blocks * n));
#define BREO(T, WM) hipLaunchKernelGGL((k_beam_reorder<T, WM>), grid, dim3(256), 0, st, a)
#define BREO_W(T)                                    \
  do {                                               \
    if (a.W <= 4) BREO(T, 4);                        \
    else if (a.W <= 8) BREO(T, 8);                   \
    else if (a.W <= 16) BREO(T, 16);                 \
    else BREO(T, 32);                                \
  } while (0)
    if (wide) BREO_W(uint4);
    else BREO_W(uint32_t);
#undef BREO_W
#undef BREO
  }
}

}  // namespace neon
