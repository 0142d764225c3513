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

// ---------------------------------------------------------------------------
// The K best of what a wave's lanes hold.  The K-th largest of the lanes' maxima is a
// bound that few others reach (K lanes hold something at least as large), so what
// reaches it is listed in LDS, and its order is found by counting.
// ---------------------------------------------------------------------------
constexpr int kBmList = 128;  // entries of a wave's list
__device__ __forceinline__ u64 bm_lane_key(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)v, lane) |
         (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32;
}
// The largest x, of the upper 18 bits, that K of the wave's values reach; 0 where fewer
// than K lanes have a value.  Two bits at a time: the three counts of a step do not wait
// for each other.
__device__ __forceinline__ uint32_t bm_kth(uint32_t v, int K) {
  uint32_t x = 0;
#pragma unroll
  for (int bit = 30; bit >= 14; bit -= 2) {
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

// Where more than kBmList reach the bound (rows of equal logits, orders that put
// all large ones into few lanes): lane i holds the i-th best key, and each candidate is
// put in its place.  Of equal keys the earlier one offered is the better.
__device__ __forceinline__ uint32_t bm_before(uint32_t v) {  // the lane before's (lane 0: 0)
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x138, 0xF, 0xF, false);  // wave_shr 1
}
struct BmBest {
  u64 key = 0;       // 0: none
  uint32_t what = 0;  // that belongs to it
  u64 last = 0;      // the K-th best (uniform)
  // the lane's k (0: none) and what belongs to it: first + lane
  __device__ __forceinline__ void offer(u64 k, uint32_t first, int K) {
    const int lane = threadIdx.x & 63;
    u64 in = __ballot(k > last);
    while (in != 0) {
      const int from = __builtin_ctzll(in);
      const u64 x = bm_lane_key(k, from);
      const int at = __builtin_popcountll(__ballot(key >= x));
      const u64 kb = (u64)bm_before((uint32_t)key) | (u64)bm_before((uint32_t)(key >> 32)) << 32;
      const uint32_t wb = bm_before(what);
      key = lane > at ? kb : lane == at ? x : key;
      what = lane > at ? wb : lane == at ? first + from : what;
      last = bm_lane_key(key, K - 1);
      in &= (~1ull << from) & __ballot(k > last);
    }
  }
};

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

// exp(x) for x <= 0, to 2^-45: 2^f by a polynomial of degree 9 on [-1/2, 1/2]
// (interpolated at the Chebyshev points, 1.9e-14), the exponent added as an integer.
// 2^-1020 stands for all below it.  The coefficients stay in scalar registers: as
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
// A chunk of a row: its maximum, the sum of exponentials and its K = W + n_stop best
// tokens (of W + n_stop at least W are no stop tokens, and a stop token that is not
// among them has W better ones in its own row).  A wave holds 1024 NB tokens, 16 NB of a
// lane.
// ---------------------------------------------------------------------------
struct __align__(16) BmSum {
  double s;
  float m;
  float pad;
};

// 16 logits of a lane: elements 4 k + j are the tokens t0 + 256 k + 4 lane + j.  A row
// begins at any multiple of 4 bytes; which lane takes a token does not depend on it, so
// equal rows have equal sums, and equal beams are ordered by their places.  Tokens past
// the end and NaNs are minus infinity.
typedef float bm_f4 __attribute__((ext_vector_type(4), aligned(4)));
template <int N>
__device__ __forceinline__ void bm_load(const float* row, int V, int t0, int lane, float (&x)[N]) {
  if (t0 + 64 * N <= V) {  // the whole wave's
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const bm_f4 v = *reinterpret_cast<const bm_f4*>(row + t0 + 256 * k + 4 * lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * k + j] = v[j];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int t = t0 + 256 * (e >> 2) + 4 * lane + (e & 3);
      const float v = row[min(t, V - 1)];
      x[e] = t < V ? v : -INFINITY;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = x[e] != x[e] ? -INFINITY : x[e];
}

template <int NB>
__global__ __launch_bounds__(256) void k_beam_part(BeamSelectArgs a) {
  constexpr int N = 16 * NB;
  __shared__ u64 list[4][kBmList];
  __shared__ int count[4];
  __shared__ float ms[4];
  __shared__ double ss[4];
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  if (!bm_alive(a.score[row])) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int K = a.K;
  const int t0 = (chunk * 4 + wave) * 64 * N;
  const BmExp exp_of;
  float m = -INFINITY;
  double s = 0.0;
  int n = 0;
  if (t0 < a.V) {
    float x[N], top4[N / 4], top;
    bm_load<N>(a.logits + (int64_t)row * a.stride, a.V, t0, lane, x);
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      top4[k] = fmaxf(fmaxf(x[4 * k], x[4 * k + 1]), fmaxf(x[4 * k + 2], x[4 * k + 3]));
      top = k == 0 ? top4[0] : fmaxf(top, top4[k]);
    }
    m = wave_max(top);
    if (m != -INFINITY && m != INFINITY) {
      const double md = (double)m;
      double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int e = 0; e < N; ++e) part[e & 3] += exp_of((double)x[e] - md);
      s = bm_wave_sum((part[0] + part[1]) + (part[2] + part[3]));
    }
    const uint32_t bound = bm_kth(bm_ordered(top), K);
    const float least = bound == 0 ? -3.4028234663852886e38f : bm_logit(bound);
    auto token = [&](int e) { return t0 + 256 * (e >> 2) + 4 * lane + (e & 3); };
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      if (__ballot(top4[k] >= least) == 0) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 in = __ballot(x[4 * k + j] >= least);
        if (in == 0) continue;
        const int at = n + bm_rank(in);
        if (x[4 * k + j] >= least && at < kBmList) list[wave][at] = bm_key(x[4 * k + j], token(4 * k + j));
        n += __builtin_popcountll(in);
      }
    }
    if (n > kBmList) {
      BmBest best;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (__ballot(x[e] >= least) != 0) best.offer(x[e] >= least ? bm_key(x[e], token(e)) : 0, 0, K);
      }
      if (lane < K) list[wave][lane] = best.key;
      n = K;
    }
  }
  if (lane == 0) {
    count[wave] = n;
    ms[wave] = m;
    ss[wave] = s;
  }
  __syncthreads();
  // the places of the four lists' keys
  const int64_t at = (int64_t)row * a.chunks + chunk;
  const int all = count[0] + count[1] + count[2] + count[3];
  for (int i = lane; i < n; i += 64) {
    const u64 mine = list[wave][i];
    int place = 0;
    for (int w = 0; w < 4; ++w)
      for (int j = 0; j < count[w]; ++j) place += list[w][j] > mine;
    if (place < K) a.keys[at * K + place] = mine;
  }
  if ((int)threadIdx.x < K && (int)threadIdx.x >= all) a.keys[at * K + threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    const float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    double S = 0.0;
    for (int w = 0; w < 4; ++w)
      if (ms[w] != -INFINITY) S += ss[w] * exp_of((double)ms[w] - (double)M);
    a.sums[at].s = S;
    a.sums[at].m = M;
  }
}

// ---------------------------------------------------------------------------
// A request: the K best of each row, then the W best that go on and the stop tokens
// among the W best.
// ---------------------------------------------------------------------------
constexpr int kBmMaxK = kBeamMaxW + kBeamMaxStop;
constexpr int kBmJoinWaves = 16;
__global__ __launch_bounds__(64 * kBmJoinWaves) void k_beam_join(BeamSelectArgs a) {
  __shared__ u64 list[kBmJoinWaves][kBmList];
  __shared__ u64 value[kBeamMaxW * kBmMaxK];  // of (place, rank), ordered; 0: none
  __shared__ int token[kBeamMaxW * kBmMaxK];
  __shared__ int stop[kBeamMaxStop];
  const int b = blockIdx.x, W = a.W, K = a.K;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const BmExp exp_of;
  if (threadIdx.x < kBeamMaxStop) stop[threadIdx.x] = (int)threadIdx.x < a.n_stop ? a.stop[threadIdx.x] : -1;
  for (int w = wave; w < W; w += kBmJoinWaves) {
    const int row = b * W + w;
    const float score = a.score[row];
    bool alive = bm_alive(score);
    if (lane == 0 && (score != score || score == INFINITY)) flag_dev_err(a.err, kDevErrBeam);
    double lse = 0.0;
    if (alive) {
      float m = -INFINITY;
      for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, a.sums[(int64_t)row * a.chunks + c].m);
      m = wave_max(m);
      double s = 0.0;
      for (int c = lane; c < a.chunks; c += 64) {
        const BmSum p = a.sums[(int64_t)row * a.chunks + c];
        if (p.m != -INFINITY) s += p.s * exp_of((double)p.m - (double)m);
      }
      s = bm_wave_sum(s);
      if (lane == 0 && m == INFINITY) flag_dev_err(a.err, kDevErrBeam);
      alive = m > -INFINITY && m < INFINITY;
      lse = (double)m + log(s);
    }
    int n = 0;
    if (alive) {
      const int all = a.chunks * K;
      const u64* keys = a.keys + (int64_t)row * all;
      u64 top = 0;
      for (int i = lane; i < all; i += 64) top = max(top, keys[i]);
      const uint32_t least = bm_kth((uint32_t)(top >> 32), K);
      for (int i0 = 0; i0 < all; i0 += 64) {
        const u64 k = i0 + lane < all ? keys[i0 + lane] : 0;
        const bool is = k != 0 && (uint32_t)(k >> 32) >= least;
        const u64 in = __ballot(is);
        const int at = n + bm_rank(in);
        if (is && at < kBmList) list[wave][at] = k;
        n += __builtin_popcountll(in);
      }
      if (n > kBmList) {
        BmBest best;
        for (int i0 = 0; i0 < all; i0 += 64) best.offer(i0 + lane < all ? keys[i0 + lane] : 0, 0, K);
        if (lane < K) list[wave][lane] = best.key;
        n = K;
      }
      wave_lds_sync();
    }
    if (lane < K && lane >= n) value[w * K + lane] = 0;
    for (int i = lane; i < n; i += 64) {
      const u64 mine = list[wave][i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += list[wave][j] > mine;
      if (place < K) {
        const double v = (double)score + ((double)bm_logit((uint32_t)(mine >> 32)) - lse);
        value[w * K + place] = bm_ordered64(v);
        token[w * K + place] = (int)~(uint32_t)mine;
      }
    }
    wave_lds_sync();  // the list is free
  }
  __syncthreads();
  if (wave > 1) return;
  // wave 0: the W best of all; wave 1: of those that are no stop tokens; equal ones in
  // the order of place and rank
  auto is_stop = [&](int t) {
    bool is = false;
    for (int i = 0; i < a.n_stop; ++i) is |= t == stop[i];
    return is;
  };
  const int all = W * K;
  auto value_of = [&](int i) {
    u64 k = i < all ? value[i] : 0;
    if (wave == 1 && k != 0 && is_stop(token[i])) k = 0;
    return k;
  };
  u64 top = 0;
  for (int i = lane; i < all; i += 64) top = max(top, value_of(i));
  const uint32_t least = bm_kth((uint32_t)(top >> 32), W);
  BmBest best;
  for (int i0 = 0; i0 < all; i0 += 64) {
    const u64 k = value_of(i0 + lane);
    best.offer((uint32_t)(k >> 32) >= least ? k : 0, (uint32_t)i0, W);
  }
  const bool has = lane < W && best.key != 0;
  const int place = has ? (int)best.what / K : -1;
  const int tok = has ? token[best.what] : -1;
  const float v = has ? (float)bm_value64(best.key) : -INFINITY;
  if (wave == 0) {
    if (a.end_token == nullptr) return;
    const bool ends = has && is_stop(tok);
    const u64 over = __ballot(ends);
    const int at = bm_rank(over);
    if (ends) {
      a.end_token[b * W + at] = tok;
      a.end_parent[b * W + at] = b * W + place;
      a.end_score[b * W + at] = v;
    }
    if (lane >= __builtin_popcountll(over) && lane < W) {
      a.end_token[b * W + lane] = -1;
      a.end_parent[b * W + lane] = -1;
      a.end_score[b * W + lane] = -INFINITY;
    }
    return;
  }
  // the first child of a beam keeps its place
  bool keeps = false;
  u64 taken = 0;
  for (int w = 0; w < W; ++w) {
    const u64 children = __ballot(place == w);
    if (children == 0) continue;
    taken |= 1ull << w;
    keeps |= lane == __builtin_ctzll(children);
  }
  const u64 movers = __ballot(lane < W && !keeps);
  int nth = bm_rank(movers);  // the free place that a mover takes
  u64 open = ~taken;
  int to = place;
  if (!keeps) {
    for (; nth > 0; --nth) open &= open - 1;
    to = __builtin_ctzll(open);
  }
  if (lane < W) {
    a.token[b * W + to] = tok;
    a.parent[b * W + to] = has ? b * W + place : -1;
    a.out_score[b * W + to] = v;
  }
}

// Batches of 16 tokens of a lane: four where the chip is full several times over.
static int beam_batches(int64_t rows, int V) {
  const int64_t waves = rows * (((int64_t)V + 1023) / 1024);
  return waves >= 16384 ? 4 : waves >= 4096 ? 2 : 1;
}
static int beam_chunks(int V, int nb) { return (int)(((int64_t)V + 4096 * nb - 1) / (4096 * nb)); }
constexpr int64_t kBmMaxBlocks = 1 << 24;  // of 256 threads: a launch holds fewer than 2^32
bool beam_select_fits(int B, int W, int V) {
  const int64_t rows = (int64_t)B * W;
  return rows * beam_chunks(V, beam_batches(rows, V)) < kBmMaxBlocks;
}
static size_t beam_chunk_bytes(int K) { return (size_t)K * 8 + sizeof(BmSum); }
size_t beam_select_needs(int B, int W, int V, int n_stop) {
  const int64_t rows = (int64_t)B * W;
  return (size_t)rows * beam_chunks(V, beam_batches(rows, V)) * beam_chunk_bytes(W + n_stop);
}
// Fewer rows may be cut into more chunks: the most that any number up to B needs is at
// B or right before a step of beam_batches.
size_t beam_select_workspace(int B, int W, int V, int n_stop) {
  size_t most = beam_select_needs(B, W, V, n_stop);
  int lo = 1, hi = B;
  for (int nb = beam_batches((int64_t)B * W, V); nb > 1; nb >>= 1) {
    for (lo = 1; lo < hi;) {  // the first B with as many batches as this
      const int mid = lo + (hi - lo) / 2;
      if (beam_batches((int64_t)mid * W, V) >= nb) hi = mid;
      else lo = mid + 1;
    }
    hi = lo;
    if (lo > 1) most = std::max(most, beam_select_needs(lo - 1, W, V, n_stop));
  }
  return most;
}
void launch_beam_select(BeamSelectArgs a, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.W;
  const int nb = beam_batches(rows, a.V);
  a.chunks = beam_chunks(a.V, nb);
  a.K = a.W + a.n_stop;
  a.sums = (BmSum*)a.workspace;
  a.keys = (u64*)(a.sums + (size_t)rows * a.chunks);
  const dim3 grid((unsigned)(rows * a.chunks));
  if (nb == 4) hipLaunchKernelGGL(k_beam_part<4>, grid, dim3(256), 0, st, a);
  else if (nb == 2) hipLaunchKernelGGL(k_beam_part<2>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(k_beam_part<1>, grid, dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_beam_join, dim3((unsigned)a.B), dim3(64 * kBmJoinWaves), 0, st, a);
}

// ---------------------------------------------------------------------------
// Moving states: a thread takes one place of the W beams of a request in a state and
// reads all that move there before it writes any, so the move is in place whatever the
// parents are (a permutation too).
// ---------------------------------------------------------------------------
template <class T, int WMAX>
__global__ __launch_bounds__(256) void k_beam_reorder(BeamReorderArgs a) {
  // block: (state, request, slab, part of the slab)
  int64_t id = blockIdx.x;
  const int part = (int)(id % a.parts);
  id /= a.parts;
  const int slab = (int)(id % a.slabs);
  id /= a.slabs;
  const int g = (int)(id % a.groups), x = (int)(id / a.groups);
  const int64_t i = (int64_t)part * 256 + threadIdx.x;  // place in the slab
  T* base = reinterpret_cast<T*>(a.state[x]) + (int64_t)g * a.W * a.seq + slab * a.slab + i;
  T v[WMAX];
  bool moves[WMAX];
#pragma unroll
  for (int w = 0; w < WMAX; ++w) {
    moves[w] = false;
    if (w >= a.W) continue;
    const int row = g * a.W + w, p = a.parent[row] - g * a.W;
    if ((unsigned)p >= (unsigned)a.W) {
      if (p != -1 - g * a.W && threadIdx.x == 0 && part == 0) flag_dev_err(a.err, kDevErrBeam);
      continue;
    }
    if (p == w) continue;
    const int n = a.len != nullptr ? min(max(a.len[g * a.W + p], 0), a.T) : a.T;
    moves[w] = i < (int64_t)n * a.per;
    if (moves[w]) v[w] = base[(int64_t)p * a.seq];
  }
#pragma unroll
  for (int w = 0; w < WMAX; ++w)
    if (moves[w]) base[(int64_t)w * a.seq] = v[w];
}

static int64_t reorder_units(const BeamReorderArgs& a) {  // of a slab
  return (int64_t)a.T * (a.row_bytes % 16 == 0 ? a.row_bytes / 16 : a.row_bytes / 4);
}
bool beam_reorder_fits(const BeamReorderArgs& a) {
  const int64_t parts = (reorder_units(a) + 255) / 256;
  return parts < kBmMaxBlocks && parts * a.slabs < kBmMaxBlocks &&
         parts * a.slabs * a.groups < kBmMaxBlocks;
}
void launch_beam_reorder(BeamReorderArgs a, void* const* states, int n_states, hipStream_t st) {
  const bool wide = a.row_bytes % 16 == 0;
  a.per = wide ? a.row_bytes / 16 : a.row_bytes / 4;
  a.slab = (int64_t)a.T * a.per;
  a.seq = a.slab * a.slabs;
  a.parts = (int)((a.slab + 255) / 256);
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
