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
// The best of a stream, in a wave's lanes: lane i holds the i-th best key and what
// belongs to it.  Keys are 0 where there is none; of equal keys the earlier one
// offered is the better.
// ---------------------------------------------------------------------------
__device__ __forceinline__ u64 bm_lane_key(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)v, lane) |
         (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32;
}
// the value of the lane before (0 for lane 0)
__device__ __forceinline__ uint32_t bm_before(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x138, 0xF, 0xF, false);  // wave_shr 1
}
struct BmBest {
  u64 key = 0;       // the lane's place
  uint32_t what = 0;
  u64 last = 0;      // the K-th best (uniform)
  __device__ __forceinline__ void insert(u64 k, uint32_t w, int K) {
    const int lane = threadIdx.x & 63;
    const int at = __builtin_popcountll(__ballot(key >= k));
    const u64 kb = (u64)bm_before((uint32_t)key) | (u64)bm_before((uint32_t)(key >> 32)) << 32;
    const uint32_t wb = bm_before(what);
    key = lane > at ? kb : lane == at ? k : key;
    what = lane > at ? wb : lane == at ? w : what;
    last = bm_lane_key(key, K - 1);
  }
};
// The largest x that K of the wave's values reach (0 where fewer than K lanes have
// one): a lower bound of the K-th best of whatever the lanes' values are the maxima of.
__device__ __forceinline__ uint32_t bm_kth(uint32_t v, int K) {
  uint32_t x = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t y = x | 1u << bit;
    if (__builtin_popcountll(__ballot(v >= y)) >= K) x = y;
  }
  return x;
}
// Offers N keys of every lane (0: none), in the order of e, then the lane.  top: the
// upper half of the lane's largest.  Where more than K lanes have something to offer,
// a bound from the lanes' maxima leaves few of it.
template <int N, class KEY, class WHAT>
__device__ __forceinline__ void bm_offer(BmBest& best, uint32_t top, int K, KEY key, WHAT what) {
  uint32_t least = (uint32_t)(best.last >> 32);
  const u64 any = __ballot(top != 0 && top >= least);
  if (any == 0) return;
  if (__builtin_popcountll(any) > K) least = max(least, bm_kth(top, K));
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const u64 k = key(e);
    u64 in = __ballot(k > best.last && (uint32_t)(k >> 32) >= least);
    while (in != 0) {
      const int lane = __builtin_ctzll(in);
      best.insert(bm_lane_key(k, lane), (uint32_t)__builtin_amdgcn_readlane((int)what(e), lane), K);
      in &= (~1ull << lane) & __ballot(k > best.last);
    }
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
// the same for a 64-bit value above minus infinity
__device__ __forceinline__ u64 bm_ordered64(double v) {
  const u64 b = __builtin_bit_cast(u64, v + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double bm_value64(u64 k) {
  return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

// exp(x) for x <= 0, to 2^-45: 2^f by a polynomial of degree 9 on [-1/2, 1/2]
// (interpolated at the Chebyshev points, 1.9e-14), the exponent added as an integer.
// 2^-1020 stands for all below it.
__device__ __forceinline__ double bm_exp(double x) {
  constexpr double kMagic = 0x1.8p52;  // its sum's low bits are the nearest integer
  const double t = fmax(x * 1.4426950408889634074, -1020.0);
  const double r = t + kMagic;
  const double f = t - (r - kMagic);
  double p = 0x1.b6571e229927fp-24;
  p = __builtin_fma(p, f, 0x1.63ef9699120e2p-20);
  p = __builtin_fma(p, f, 0x1.ffcb767842e11p-17);
  p = __builtin_fma(p, f, 0x1.43088e2580989p-13);
  p = __builtin_fma(p, f, 0x1.5d87fe908fb19p-10);
  p = __builtin_fma(p, f, 0x1.3b2ab72b175e1p-7);
  p = __builtin_fma(p, f, 0x1.c6b08d7044117p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff8149f2p-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa39f7p-1);
  p = __builtin_fma(p, f, 0x1.000000000003dp+0);
  const u64 b = __builtin_bit_cast(u64, p);
  const uint32_t n = (uint32_t)__builtin_bit_cast(u64, r);
  return __builtin_bit_cast(double, b + ((u64)(n << 20) << 32));
}

template <int OFF = 32>
__device__ __forceinline__ double bm_wave_sum(double v) {
  const u64 b = __builtin_bit_cast(u64, v);
  const uint32_t lo = (uint32_t)xor_lane_i<OFF>((int)(uint32_t)b);
  const uint32_t hi = (uint32_t)xor_lane_i<OFF>((int)(uint32_t)(b >> 32));
  v += __builtin_bit_cast(double, (u64)lo | (u64)hi << 32);
  if constexpr (OFF > 1) return bm_wave_sum<OFF / 2>(v);
  return v;
}
// maximum and sum of exp(l - maximum) of all lanes from those of each
__device__ __forceinline__ void bm_wave_lse(float& m, double& s) {
  const float M = wave_max(m);
  s = m == -INFINITY ? 0.0 : s * bm_exp((double)m - (double)M);
  s = bm_wave_sum(s);
  m = M;
}

// A beam that has a score to go on from.
__device__ __forceinline__ bool bm_alive(float score) { return score > -INFINITY && score < INFINITY; }

// ---------------------------------------------------------------------------
// A chunk of a row: its maximum, the sum of exponentials and its K = W + n_stop best
// tokens (of W + n_stop at least W are no stop tokens, and a stop token that is not
// among them has W better ones in its own row).  A wave takes 1024 tokens at a time,
// 16 of a lane.
// ---------------------------------------------------------------------------
constexpr int kBmBatch = 1024;         // tokens of a wave's step
constexpr int kBmBlock = 4 * kBmBatch;  // of a block's
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
__device__ __forceinline__ void bm_load(const float* row, int V, int t0, int lane, float (&x)[16]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int t = t0 + 256 * k + 4 * lane;
    if (t + 4 <= V) {
      const bm_f4 v = *reinterpret_cast<const bm_f4*>(row + t);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * k + j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * k + j] = t + j < V ? row[t + j] : -INFINITY;
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = x[e] != x[e] ? -INFINITY : x[e];
}

__global__ __launch_bounds__(256) void k_beam_part(BeamSelectArgs a) {
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  if (!bm_alive(a.score[row])) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* l = a.logits + (int64_t)row * a.stride;
  const int K = a.K;
  BmBest best;
  float m = -INFINITY;
  double s = 0.0;
  const int from = chunk * a.steps;
  for (int i = from; i < from + a.steps; ++i) {
    const int t0 = i * kBmBlock + wave * kBmBatch;
    if (t0 >= a.V) break;
    float x[16];
    bm_load(l, a.V, t0, lane, x);
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
    if (top > m) {
      if (m != -INFINITY) s *= bm_exp((double)m - (double)top);
      m = top;
    }
    if (m != -INFINITY && m != INFINITY) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s += bm_exp((double)x[e] - (double)m);
    }
    bm_offer<16>(
        best, bm_ordered(top), K,
        [&](int e) {
          const uint32_t o = bm_ordered(x[e]);
          const uint32_t t = (uint32_t)(t0 + 256 * (e >> 2) + 4 * lane + (e & 3));
          return o == 0 ? 0ull : (u64)o << 32 | (uint32_t)~t;
        },
        [](int) { return 0u; });
  }
  bm_wave_lse(m, s);
  __shared__ u64 keys[4][64];
  __shared__ float ms[4];
  __shared__ double ss[4];
  keys[wave][lane] = lane < K ? best.key : 0;
  if (lane == 0) {
    ms[wave] = m;
    ss[wave] = s;
  }
  __syncthreads();
  // the place of a key among the four waves'
  const int64_t at = (int64_t)row * a.chunks + chunk;
  const u64 mine = keys[wave][lane];
  int place = lane;
  for (int w = 0; w < 4; ++w)
    if (w != wave)
      for (int i = 0; i < K; ++i) place += keys[w][i] > mine || (keys[w][i] == mine && w < wave);
  if (lane < K && place < K) a.keys[at * K + place] = mine;
  if (threadIdx.x == 0) {
    float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    double S = 0.0;
    for (int w = 0; w < 4; ++w)
      if (ms[w] != -INFINITY) S += ss[w] * bm_exp((double)ms[w] - (double)M);
    a.sums[at].s = S;
    a.sums[at].m = M;
  }
}

// ---------------------------------------------------------------------------
// A request: the K best of each row, then the W best that go on and the stop tokens
// among the W best.
// ---------------------------------------------------------------------------
constexpr int kBmMaxK = kBeamMaxW + kBeamMaxStop;
__global__ __launch_bounds__(256) void k_beam_join(BeamSelectArgs a) {
  __shared__ u64 value[kBeamMaxW * kBmMaxK];   // of (place, rank), ordered; 0: none
  __shared__ int token[kBeamMaxW * kBmMaxK];
  __shared__ int stop[kBeamMaxStop];
  const int b = blockIdx.x, W = a.W, K = a.K;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x < kBeamMaxStop) stop[threadIdx.x] = (int)threadIdx.x < a.n_stop ? a.stop[threadIdx.x] : -1;
  for (int w = wave; w < W; w += 4) {
    const int row = b * W + w;
    const float score = a.score[row];
    bool alive = bm_alive(score);
    if (lane == 0 && (score != score || score == INFINITY)) flag_dev_err(a.err, kDevErrBeam);
    BmBest best;
    double lse = 0.0;
    if (alive) {
      float m = -INFINITY;
      double s = 0.0;
      for (int c = lane; c < a.chunks; c += 64) {
        const BmSum p = a.sums[(int64_t)row * a.chunks + c];
        const float M = fmaxf(m, p.m);
        if (M == -INFINITY) continue;
        s = (m == -INFINITY ? 0.0 : s * bm_exp((double)m - (double)M)) +
            (p.m == -INFINITY ? 0.0 : p.s * bm_exp((double)p.m - (double)M));
        m = M;
      }
      bm_wave_lse(m, s);
      if (lane == 0 && m == INFINITY) flag_dev_err(a.err, kDevErrBeam);
      alive = m > -INFINITY && m < INFINITY;
      lse = (double)m + log(s);
    }
    if (alive) {
      const int n = a.chunks * K;
      const u64* keys = a.keys + (int64_t)row * n;
      for (int i0 = 0; i0 < n; i0 += 256) {
        u64 k[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = i0 + 64 * e + lane < n ? keys[i0 + 64 * e + lane] : 0;
        u64 top = k[0] > k[1] ? k[0] : k[1];
        const u64 top2 = k[2] > k[3] ? k[2] : k[3];
        top = top > top2 ? top : top2;
        bm_offer<4>(best, (uint32_t)(top >> 32), K, [&](int e) { return k[e]; }, [](int) { return 0u; });
      }
    }
    if (lane < K) {
      const double v = (double)score + ((double)bm_logit((uint32_t)(best.key >> 32)) - lse);
      value[w * K + lane] = best.key == 0 ? 0 : bm_ordered64(v);
      token[w * K + lane] = (int)~(uint32_t)best.key;
    }
  }
  __syncthreads();
  if (wave > 1) return;
  // wave 0: the W best of all; wave 1: of those that are no stop tokens.  Offered in
  // the order of place and rank, so equal ones come out in that order.
  auto is_stop = [&](int t) {
    bool is = false;
    for (int i = 0; i < a.n_stop; ++i) is |= t == stop[i];
    return is;
  };
  BmBest best;
  for (int i0 = 0; i0 < W * K; i0 += 64) {
    const int i = i0 + lane;
    u64 k = i < W * K ? value[i] : 0;
    if (wave == 1 && k != 0 && is_stop(token[i])) k = 0;
    bm_offer<1>(best, (uint32_t)(k >> 32), W, [&](int) { return k; }, [&](int) { return (uint32_t)i; });
  }
  const bool has = lane < W && best.key != 0;
  const int place = has ? (int)(best.what / (uint32_t)K) : -1;
  const int tok = has ? token[best.what] : -1;
  const float v = has ? (float)bm_value64(best.key) : -INFINITY;
  const u64 below = (1ull << lane) - 1;
  if (wave == 0) {
    if (a.end_token == nullptr) return;
    const bool ends = has && is_stop(tok);
    const u64 all = __ballot(ends);
    const int n = __builtin_popcountll(all);
    const int at = ends ? __builtin_popcountll(all & below) : -1;
    if (ends) {
      a.end_token[b * W + at] = tok;
      a.end_parent[b * W + at] = b * W + place;
      a.end_score[b * W + at] = v;
    }
    if (lane >= n && lane < W) {
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
  int nth = __builtin_popcountll(movers & below);  // the free place that a mover takes
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

static int64_t beam_blocks(int V) { return ((int64_t)V + kBmBlock - 1) / kBmBlock; }
// Steps of a block: about kBmTarget blocks, of whole steps.
constexpr int64_t kBmTarget = 2048;
constexpr int64_t kBmMaxBlocks = 1 << 24;  // of 256 threads: a launch holds fewer than 2^32
static void beam_cut(int rows, int V, int& chunks, int& steps) {
  const int64_t n = beam_blocks(V);
  const int64_t per = (n * rows + kBmTarget - 1) / kBmTarget;
  steps = (int)(per < n ? per : n);
  chunks = (int)((n + steps - 1) / steps);
}
bool beam_select_fits(int B, int W, int V) {
  int chunks, steps;
  if ((int64_t)B * W > 1 << 21) return false;
  beam_cut(B * W, V, chunks, steps);
  return (int64_t)B * W * chunks < kBmMaxBlocks;
}
size_t beam_select_workspace(int B, int W, int V, int n_stop) {
  int chunks, steps;
  beam_cut(B * W, V, chunks, steps);
  return (size_t)B * W * chunks * ((size_t)(W + n_stop) * 8 + sizeof(BmSum));
}
void launch_beam_select(BeamSelectArgs a, hipStream_t st) {
  const int rows = a.B * a.W;
  beam_cut(rows, a.V, a.chunks, a.steps);
  a.K = a.W + a.n_stop;
  a.sums = (BmSum*)a.workspace;
  a.keys = (u64*)(a.sums + (size_t)rows * a.chunks);
  hipLaunchKernelGGL(k_beam_part, dim3((unsigned)(rows * a.chunks)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_beam_join, dim3((unsigned)a.B), dim3(256), 0, st, a);
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
