// neon_paged.hip -- the paged KV cache: appending rotated keys and values,
// reading rows back, and attention over the pages.
//
// A sequence's token t sits in page table[b][t / page], row t % page.  Pages
// are bf16, or MXFP4 in the layout of the checkpoint's expert weights: codes
// [row][D/2] (low nibble = even element) and one E8M0 scale per 32 elements
// along D, so a token is written alone, whatever its neighbours hold.
#include <hip/hip_runtime.h>

#include "neon_common.hpp"
#include "neon_internal.hpp"

namespace neon {

// ---------------------------------------------------------------------------
// Rows of the batch
// ---------------------------------------------------------------------------
// Whether sequence b's rows and length are ones that the buffers hold (device
// data: checked before anything is addressed with it).  A sequence of length 0
// is a free place of the batch: it has no rows to take.
__device__ __forceinline__ bool paged_seq(const PagedRows& r, int page_log2, int b, int& start,
                                          int& n, int& len) {
  start = r.q_start != nullptr ? r.q_start[b] : b;
  const int end = r.q_start != nullptr ? r.q_start[b + 1] : b + 1;
  len = r.kv_len[b];
  n = end - start;
  return start >= 0 && n >= 0 && end <= r.n_rows && len >= n &&
         (int64_t)len <= ((int64_t)r.max_pages << page_log2);
}

// The sequence and position of a row, found by the whole block (every thread
// calls it with the same row); false when the row belongs to no sequence.  The
// block of row 0 reports the sequences that do not fit.
__device__ __forceinline__ bool paged_row(const PagedRows& r, int page_log2, int row, int& b,
                                          int& pos) {
  int start, n, len;
  b = row;
  if (r.q_start != nullptr) {
    __shared__ int found;
    if (threadIdx.x == 0) found = r.B;
    __syncthreads();
    for (int i = threadIdx.x; i < r.B; i += blockDim.x) {
      const int s0 = r.q_start[i], s1 = r.q_start[i + 1];
      if (s0 <= row && row < s1) atomicMin(&found, i);
      if (row == 0 && !paged_seq(r, page_log2, i, start, n, len) && len != 0)
        flag_dev_err(r.err, kDevErrPagedRows);
    }
    __syncthreads();
    b = found;
  }
  if (b >= r.B) return false;
  if (!paged_seq(r, page_log2, b, start, n, len)) {
    if (r.q_start == nullptr && threadIdx.x == 0 && len != 0)
      flag_dev_err(r.err, kDevErrPagedRows);
    return false;
  }
  pos = len - n + (row - start);
  return true;
}

// Index of (page id, head, row of the page), in rows of D.
__device__ __forceinline__ int64_t paged_row_at(const PagedKv& kv, int id, int h, int t) {
  return (((int64_t)id * kv.Hkv + h) << kv.page_log2) + (t & ((1 << kv.page_log2) - 1));
}

// ---------------------------------------------------------------------------
// Append.  A block takes one row; a thread takes 16 elements of a head, d0 ..
// d0 + 7 and their rotation partners d0 + D/2 .. + 7 (value heads the same
// places, not rotated), so a quad of threads holds two whole 32-element
// blocks.  The rotation is rope_pair in fp32.  bf16 rows round it once;
// MXFP4 blocks are taken from the fp32 values, so they round once as well:
// a bf16 step in between would move values across the borders of E2M1.
// Bound: the bytes of the qkv row, q_out and the cache rows.
// ---------------------------------------------------------------------------

// E8M0 byte of a block with largest magnitude amax: 2^(floor(log2 amax) - 2),
// one more where amax would lie past 7, more than half a step above E2M1's
// largest value 6 (OCP MX has no such step: there up to 7.99 become 6).
__device__ __forceinline__ uint32_t mx4_scale_byte(float amax) {
  if (!(amax > 0.0f)) return 127u;
  if (!(amax < INFINITY)) return 255u;
  int e = ilog2f_dev(amax);
  if (__builtin_amdgcn_ldexpf(amax, -e) > 1.75f) e += 1;
  e = e - 2 + 127;
  return (uint32_t)(e < 0 ? 0 : e);  // e <= 127 - 1 + 127
}

// E2M1 code of y, |y| <= 7: nearest, ties to the even code, 6 above 5
__device__ __forceinline__ uint32_t e2m1_code(float y) {
  const float a = fabsf(y);
  const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) +
                     (a >= 3.5f) + (a > 5.0f);
  return c | ((__float_as_uint(y) >> 28) & 8u);
}

// This lane's 8 of a block's 32 values (the block is the quad's): its 8 codes
// and the block's scale byte.  A block with a NaN or an infinity gets the
// scale 0xFF (every value of it reads as NaN) and zero codes.
__device__ __forceinline__ uint32_t mx4_quant8(const float (&v)[8], uint32_t& byte) {
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fabsf(v[j]);
    amax = a < INFINITY ? fmaxf(amax, a) : INFINITY;  // a NaN compares false
  }
  amax = fmaxf(amax, xor_lane<1>(amax));
  amax = fmaxf(amax, xor_lane<2>(amax));
  byte = mx4_scale_byte(amax);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w |= e2m1_code(__builtin_amdgcn_ldexpf(v[j], 127 - (int)byte)) << (4 * j);
  return byte == 255u ? 0u : w;
}

__device__ __forceinline__ void unpack8f(const uint4& w, float (&f)[8]) {
  f[0] = bf_lo(w.x); f[1] = bf_hi(w.x); f[2] = bf_lo(w.y); f[3] = bf_hi(w.y);
  f[4] = bf_lo(w.z); f[5] = bf_hi(w.z); f[6] = bf_lo(w.w); f[7] = bf_hi(w.w);
}
__device__ __forceinline__ uint4 pack8f(const float (&f)[8]) {
  return make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]),
                    pack_bf2(f[6], f[7]));
}

template <bool F4>
__global__ __launch_bounds__(256) void k_paged_append(
    PagedKv kv, PagedRows r, const uint16_t* __restrict__ qkv, int64_t stride,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, int n_pos,
    uint16_t* __restrict__ q_out, int Hq) {
  const int row = blockIdx.x;
  int b, pos;
  if (!paged_row(r, kv.page_log2, row, b, pos)) return;
  if (cos_t != nullptr && pos >= n_pos) {
    if (threadIdx.x == 0) flag_dev_err(r.err, kDevErrPagedRows);
    return;
  }
  const int id = r.table[(int64_t)b * r.max_pages + (pos >> kv.page_log2)];
  const bool page_ok = (unsigned)id < (unsigned)kv.n_pages;
  if (!page_ok && threadIdx.x == 0) flag_dev_err(r.err, kDevErrPageId);
  const int per = kv.D >> 4, half = kv.D >> 1;  // threads of a head
  const int items = (Hq + 2 * kv.Hkv) * per;
  for (int it = threadIdx.x; it < items; it += blockDim.x) {
    const int h = it / per, d0 = (it % per) * 8;
    const uint16_t* src = qkv + (int64_t)row * stride + (int64_t)h * kv.D + d0;
    float x1[8], x2[8];
    unpack8f(*reinterpret_cast<const uint4*>(src), x1);
    unpack8f(*reinterpret_cast<const uint4*>(src + half), x2);
    if (h < Hq + kv.Hkv && cos_t != nullptr) {
      const float* c = cos_t + (int64_t)pos * half + d0;
      const float* s = sin_t + (int64_t)pos * half + d0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float o1, o2;
        rope_pair(x1[j], x2[j], c[j], s[j], o1, o2);
        x1[j] = o1;
        x2[j] = o2;
      }
    }
    if (h < Hq) {
      uint16_t* dst = q_out + ((int64_t)row * Hq + h) * kv.D + d0;
      *reinterpret_cast<uint4*>(dst) = pack8f(x1);
      *reinterpret_cast<uint4*>(dst + half) = pack8f(x2);
      continue;
    }
    if (!page_ok) continue;
    const bool is_k = h < Hq + kv.Hkv;
    const int64_t at = paged_row_at(kv, id, h - Hq - (is_k ? 0 : kv.Hkv), pos);
    uint8_t* pool = is_k ? kv.k : kv.v;
    if constexpr (F4) {
      // a head's threads are whole quads, and quads take or leave every branch
      // above together
      uint32_t b1, b2;
      const uint32_t w1 = mx4_quant8(x1, b1), w2 = mx4_quant8(x2, b2);
      uint8_t* dst = pool + at * half + (d0 >> 1);
      *reinterpret_cast<uint32_t*>(dst) = w1;
      *reinterpret_cast<uint32_t*>(dst + (half >> 1)) = w2;
      if ((it & 3) == 0) {
        uint8_t* sc = (is_k ? kv.ks : kv.vs) + at * (kv.D >> 5) + (d0 >> 5);
        sc[0] = (uint8_t)b1;
        sc[half >> 5] = (uint8_t)b2;
      }
    } else {
      uint16_t* dst = reinterpret_cast<uint16_t*>(pool) + at * kv.D + d0;
      *reinterpret_cast<uint4*>(dst) = pack8f(x1);
      *reinterpret_cast<uint4*>(dst + half) = pack8f(x2);
    }
  }
}

void launch_paged_append(const PagedKv& kv, const PagedRows& r, const uint16_t* qkv, int64_t stride,
                         const float* cos_t, const float* sin_t, int n_pos, uint16_t* q_out, int Hq,
                         hipStream_t st) {
  if (kv.ks != nullptr)
    hipLaunchKernelGGL(k_paged_append<true>, dim3(r.n_rows), dim3(256), 0, st, kv, r, qkv, stride,
                       cos_t, sin_t, n_pos, q_out, Hq);
  else
    hipLaunchKernelGGL(k_paged_append<false>, dim3(r.n_rows), dim3(256), 0, st, kv, r, qkv, stride,
                       cos_t, sin_t, n_pos, q_out, Hq);
}

// 8 MXFP4 values (one dword of codes) as bf16: v_cvt_scalef32_pk_bf16_fp4
// reads the scale's exponent field, so s << 23 serves every scale byte (255:
// NaN), and E2M1 x 2^(s - 127) is a bf16 value
__device__ __forceinline__ uint4 mx4_to_bf16x8(uint32_t w, uint32_t s) {
  const float sc = __uint_as_float(s << 23);
  return make_uint4(
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3)));
}

// Elements d0 .. d0 + 7 of a cached row as bf16.
template <bool F4>
__device__ __forceinline__ uint4 paged_load8(const uint8_t* pool, const uint8_t* scales, int64_t at,
                                             int D, int d0) {
  if constexpr (F4)
    return mx4_to_bf16x8(*reinterpret_cast<const uint32_t*>(pool + at * (D >> 1) + (d0 >> 1)),
                         scales[at * (D >> 5) + (d0 >> 5)]);
  else
    return *reinterpret_cast<const uint4*>(pool + (at * D + d0) * 2);
}

// ---------------------------------------------------------------------------
// Gather: the batch's rows as the cache holds them, a block per row, 8
// elements per thread.  Bound: the bytes read and written.
// ---------------------------------------------------------------------------
template <bool F4>
__global__ __launch_bounds__(256) void k_paged_gather(PagedKv kv, PagedRows r,
                                                      uint16_t* __restrict__ k_out,
                                                      uint16_t* __restrict__ v_out) {
  const int row = blockIdx.x;
  int b, pos;
  if (!paged_row(r, kv.page_log2, row, b, pos)) return;
  const int id = r.table[(int64_t)b * r.max_pages + (pos >> kv.page_log2)];
  if ((unsigned)id >= (unsigned)kv.n_pages) {
    if (threadIdx.x == 0) flag_dev_err(r.err, kDevErrPageId);
    return;
  }
  const int per = kv.D >> 3, items = kv.Hkv * per;
  for (int it = threadIdx.x; it < 2 * items; it += blockDim.x) {
    const bool is_k = it < items;
    const int e = is_k ? it : it - items, h = e / per, d0 = (e % per) * 8;
    const int64_t at = paged_row_at(kv, id, h, pos);
    const uint4 w = paged_load8<F4>(is_k ? kv.k : kv.v, is_k ? kv.ks : kv.vs, at, kv.D, d0);
    uint16_t* dst = (is_k ? k_out : v_out) + ((int64_t)row * kv.Hkv + h) * kv.D + d0;
    *reinterpret_cast<uint4*>(dst) = w;
  }
}

void launch_paged_gather(const PagedKv& kv, const PagedRows& r, uint16_t* k_out, uint16_t* v_out,
                         hipStream_t st) {
  if (kv.ks != nullptr)
    hipLaunchKernelGGL(k_paged_gather<true>, dim3(r.n_rows), dim3(256), 0, st, kv, r, k_out, v_out);
  else
    hipLaunchKernelGGL(k_paged_gather<false>, dim3(r.n_rows), dim3(256), 0, st, kv, r, k_out, v_out);
}

// ---------------------------------------------------------------------------
// Attention: one wave per (row, query head), 64 keys at a time: lane = key for
// the scores, lane = output dims for P V, running maximum and sum in fp32.
// ---------------------------------------------------------------------------
template <int D, bool F4>
__global__ __launch_bounds__(64) void k_paged_attn(PagedAttnArgs a) {
  __shared__ float qs[D];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  int b, pos;
  if (!paged_row(a.r, a.kv.page_log2, row, b, pos)) return;
  const int g = h / (a.Hq / a.kv.Hkv);
  for (int d = lane; d < D; d += 64) qs[d] = bf2f(a.q[(int64_t)row * a.q_stride + (int64_t)h * D + d]);
  __syncthreads();
  const int lo = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  const float scale = D == 64 ? 0.125f : 0.08838834764831845f;
  float m = -INFINITY, l = 0.0f, o[D / 64];
  for (int e = 0; e < D / 64; ++e) o[e] = 0.0f;
  const int32_t* table = a.r.table + (int64_t)b * a.r.max_pages;
  for (int k0 = lo; k0 <= pos; k0 += 64) {
    const int key = k0 + lane;
    int id = key <= pos ? table[key >> a.kv.page_log2] : -1;
    const bool seen = (unsigned)id < (unsigned)a.kv.n_pages;
    if (key <= pos && !seen) flag_dev_err(a.r.err, kDevErrPageId);
    float s = -INFINITY;
    if (seen) {
      const int64_t at = paged_row_at(a.kv, id, g, key);
      float dot = 0.0f;
      for (int d0 = 0; d0 < D; d0 += 8) {
        float kf[8];
        unpack8f(paged_load8<F4>(a.kv.k, a.kv.ks, at, D, d0), kf);
        for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(qs[d0 + e], kf[e], dot);
      }
      s = dot * scale;
    }
    const float mn = fmaxf(m, wave_max(s));
    if (mn == -INFINITY) continue;
    const float al = neon_expf(m - mn), p = neon_expf(s - mn);
    l = l * al + wave_sum(p);
    m = mn;
    for (int e = 0; e < D / 64; ++e) o[e] *= al;
    for (int j = 0; j < 64; ++j) {
      const int idj = __shfl(seen ? id : -1, j);
      const float pj = __shfl(p, j);
      if (idj < 0) continue;
      const int64_t at = paged_row_at(a.kv, idj, g, k0 + j);
      for (int e = 0; e < D / 64; ++e) {
        const int d = lane + 64 * e;
        float v;
        if constexpr (F4) {
          const uint32_t c = a.kv.v[at * (D / 2) + (d >> 1)] >> (4 * (d & 1));
          v = __uint_as_float(
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                               c & 15u, __uint_as_float((uint32_t)a.kv.vs[at * (D / 32) + (d >> 5)] << 23), 0))
              << 16);
        } else {
          v = bf2f(reinterpret_cast<const uint16_t*>(a.kv.v)[at * D + d]);
        }
        o[e] = __builtin_fmaf(pj, v, o[e]);
      }
    }
  }
  if (a.sinks != nullptr) {
    const float sk = bf2f(a.sinks[h]), M = fmaxf(m, sk);
    const float al = m == -INFINITY ? 0.0f : neon_expf(m - M);
    l = l * al + neon_expf(sk - M);
    for (int e = 0; e < D / 64; ++e) o[e] *= al;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int e = 0; e < D / 64; ++e)
    a.out[((int64_t)row * a.Hq + h) * D + lane + 64 * e] = f2bf(o[e] * inv);
}

void launch_paged_attn(const PagedAttnArgs& a, hipStream_t st) {
  const dim3 grid(a.r.n_rows, a.Hq);
#define PA(D, F4) hipLaunchKernelGGL((k_paged_attn<D, F4>), grid, dim3(64), 0, st, a)
  if (a.kv.D == 64) {
    if (a.kv.ks != nullptr) PA(64, true); else PA(64, false);
  } else {
    if (a.kv.ks != nullptr) PA(128, true); else PA(128, false);
  }
#undef PA
}

}  // namespace neon
