// neon_paged.hip -- the paged KV cache: appending rotated keys and values,
// reading rows back, and attention over the pages.
//
// A sequence's token t sits in page table[b][t / page], row t % page.  Pages
// are bf16, or MXFP4 in the layout of the checkpoint's expert weights: codes
// [row][D/2] (low nibble = even element) and one E8M0 scale per 32 elements
// along D, so a token is written alone, whatever its neighbours hold.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "neon_common.hpp"
#include "neon_internal.hpp"

namespace neon {

// ---------------------------------------------------------------------------
// Rows of the batch
// ---------------------------------------------------------------------------
constexpr int kPagedLongest = 1 << 30;
// Whether a sequence's rows and length are ones that the buffers hold (device
// data: checked before anything is addressed with it).  A sequence of length 0
// is a free place of the batch: it has no rows to take.  Lengths up to 2^30
// keep every index below within an int.
__device__ __forceinline__ bool paged_fits(const PagedRows& r, int page_log2, int start, int end,
                                           int len) {
  return (start >= 0) & (end >= start) & (end <= r.n_rows) & (len >= end - start) &
         (len <= kPagedLongest) & ((int64_t)len <= ((int64_t)r.max_pages << page_log2));
}
__device__ __forceinline__ bool paged_seq(const PagedRows& r, int page_log2, int b, int& start,
                                          int& n, int& len) {
  start = r.q_start != nullptr ? r.q_start[b] : b;
  const int end = r.q_start != nullptr ? r.q_start[b + 1] : b + 1;
  len = r.kv_len[b];
  n = end - start;
  return paged_fits(r, page_log2, start, end, len);
}

// The sequence and position of a row, found by the wave (every lane calls it with
// the same row); false when the row belongs to no sequence.  A lane looks at a
// sequence with loads that depend on nothing, so a row costs one round trip
// (reading the found one's numbers again made it three).  A sequence that has rows
// fits up to `most` tokens (the positions that have angles).  The wave that asks for
// row 0 with `report` reports the sequences that do not fit.
__device__ __forceinline__ bool paged_row(const PagedRows& r, int page_log2, int most, int row,
                                          bool report, int& b, int& pos) {
  const int lane = threadIdx.x & 63;
  if (r.q_start == nullptr) {
    b = row;
    const int len = r.kv_len[row];
    pos = len - 1;
    const bool ok = paged_fits(r, page_log2, row, row + 1, len) & (len <= most);
    if (!ok && len != 0 && report && lane == 0) flag_dev_err(r.err, kDevErrPagedRows);
    return ok;
  }
  b = -1;
  for (int i0 = 0; i0 < r.B; i0 += 64) {
    const int i = min(i0 + lane, r.B - 1);  // (past the end: the last one again)
    const int start = r.q_start[i], end = r.q_start[i + 1], len = r.kv_len[i];
    const bool ok = paged_fits(r, page_log2, start, end, len) & ((len <= most) | (start == end));
    if (row == 0 && report && !ok && len != 0) flag_dev_err(r.err, kDevErrPagedRows);
    const uint64_t in = __ballot(ok & (start <= row) & (row < end));
    if (b < 0 && in != 0) {
      const int at = __builtin_ctzll(in);
      b = i0 + at;
      pos = __builtin_amdgcn_readlane(len - end, at) + row;
      if (row != 0) break;
    }
  }
  return b >= 0;
}

// Index of (page id, head, row of the page), in rows of D.
__device__ __forceinline__ int64_t paged_row_at(const PagedKv& kv, int id, int h, int t) {
  return (((int64_t)id * kv.Hkv + h) << kv.page_log2) + (t & ((1 << kv.page_log2) - 1));
}

// ---------------------------------------------------------------------------
// Append.  A block takes one row (all its threads at once, where they are up to
// 512); a thread takes 16 elements of a head, d0 ..
// d0 + 7 and their rotation partners d0 + D/2 .. + 7 (value heads the same
// places, not rotated), so a quad of threads holds two whole 32-element
// blocks.  The rotation is rope_pair in fp32.  bf16 rows round it once;
// MXFP4 blocks are taken from the fp32 values, so they round once as well:
// a bf16 step in between would move values across the borders of E2M1.
// Bound: the bytes of the qkv row, q_out and the cache rows: 9.4k rows of 64 + 8 +
// 8 heads of 64 in 39.0 us, 4.9 TB/s, the rate of a large copy.
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

// This lane's 8 of a block's 32 values (the block is the quad's): its 8 codes and
// the block's scale byte.  The conversion divides by the scale (whose exponent
// field it reads), rounds to the nearest, ties to even, and takes 6 for what is
// past it (the tests compare its codes over every binade and border).  A block
// with a NaN or an infinity gets the scale 0xFF (every value of it reads as NaN)
// and zero codes.
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
  const float sc = __uint_as_float(byte << 23);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
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

// 8 cosines, then 8 sines, from index `at` of the tables (16-byte aligned).
__device__ __forceinline__ void paged_angles(const float* cos_t, const float* sin_t, int64_t at,
                                             float4 (&cs)[4]) {
  cs[0] = *reinterpret_cast<const float4*>(cos_t + at);
  cs[1] = *reinterpret_cast<const float4*>(cos_t + at + 4);
  cs[2] = *reinterpret_cast<const float4*>(sin_t + at);
  cs[3] = *reinterpret_cast<const float4*>(sin_t + at + 4);
}

template <bool F4>
__global__ __launch_bounds__(512) void k_paged_append(
    PagedKv kv, PagedRows r, const uint16_t* __restrict__ qkv, int64_t stride,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, int n_pos,
    uint16_t* __restrict__ q_out, int Hq) {
  const int row = blockIdx.x;
  const int per = kv.D >> 4, half = kv.D >> 1;  // threads of a head
  const int items = (Hq + 2 * kv.Hkv) * per;
  // the thread's first elements are requested before the row is looked up: they
  // need neither its sequence nor its position
  const uint16_t* row_src = qkv + (int64_t)row * stride;
  const int it0 = min((int)threadIdx.x, items - 1);
  const uint16_t* src0 = row_src + (int64_t)(it0 / per) * kv.D + (it0 % per) * 8;
  uint4 w1 = *reinterpret_cast<const uint4*>(src0), w2 = *reinterpret_cast<const uint4*>(src0 + half);
  int b, pos;
  if (!paged_row(r, kv.page_log2, cos_t != nullptr ? n_pos : kPagedLongest, row,
                 threadIdx.x < 64, b, pos))
    return;
  // the first elements' angles with the page id, in one round trip
  const int id = r.table[(int64_t)b * r.max_pages + (pos >> kv.page_log2)];
  float4 cs[4];
  if (cos_t != nullptr) paged_angles(cos_t, sin_t, (int64_t)pos * half + (it0 % per) * 8, cs);
  for (int it = threadIdx.x; it < items; it += blockDim.x) {
    const int h = it / per, d0 = (it % per) * 8;
    if (it != (int)threadIdx.x) {
      const uint16_t* src = row_src + (int64_t)h * kv.D + d0;
      w1 = *reinterpret_cast<const uint4*>(src);
      w2 = *reinterpret_cast<const uint4*>(src + half);
      if (cos_t != nullptr) paged_angles(cos_t, sin_t, (int64_t)pos * half + d0, cs);
    }
    float x1[8], x2[8];
    unpack8f(w1, x1);
    unpack8f(w2, x2);
    if (h < Hq + kv.Hkv && cos_t != nullptr) {
      const float c[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
      const float s[8] = {cs[2].x, cs[2].y, cs[2].z, cs[2].w, cs[3].x, cs[3].y, cs[3].z, cs[3].w};
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
    if ((unsigned)id >= (unsigned)kv.n_pages) {
      if (d0 == 0) flag_dev_err(r.err, kDevErrPageId);
      continue;
    }
    const bool is_k = h < Hq + kv.Hkv;
    const int64_t at = paged_row_at(kv, id, h - Hq - (is_k ? 0 : kv.Hkv), pos);
    uint8_t* pool = is_k ? kv.k : kv.v;
    if constexpr (F4) {
      // a head's threads are whole quads, and quads take or leave every branch
      // above together
      uint32_t b1, b2;
      const uint32_t c1 = mx4_quant8(x1, b1), c2 = mx4_quant8(x2, b2);
      uint8_t* dst = pool + at * half + (d0 >> 1);
      *reinterpret_cast<uint32_t*>(dst) = c1;
      *reinterpret_cast<uint32_t*>(dst + (half >> 1)) = c2;
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

static int append_threads(int Hkv, int Hq, int D) {
  const int items = (Hq + 2 * Hkv) * (D >> 4);
  return items >= 512 ? 512 : (items + 63) & ~63;
}
// a launch holds fewer than 2^32 threads
bool paged_append_fits(int n_rows, int Hkv, int Hq, int D) {
  return (int64_t)n_rows * append_threads(Hkv, Hq, D) < (int64_t)1 << 32;
}

void launch_paged_append(const PagedKv& kv, const PagedRows& r, const uint16_t* qkv, int64_t stride,
                         const float* cos_t, const float* sin_t, int n_pos, uint16_t* q_out, int Hq,
                         hipStream_t st) {
  const dim3 grid(r.n_rows), block(append_threads(kv.Hkv, Hq, kv.D));
#define PAPP(F4)                                                                               \
  hipLaunchKernelGGL(k_paged_append<F4>, grid, block, 0, st, kv, r, qkv, stride, cos_t, sin_t, \
                     n_pos, q_out, Hq)
  if (kv.ks != nullptr) PAPP(true); else PAPP(false);
#undef PAPP
}

// 8 MXFP4 values (one dword of codes) as bf16 with the scale in the low byte of s:
// v_cvt_scalef32_pk_bf16_fp4 reads the exponent field of its scale alone (sign and
// fraction bits change no result for the 256 scales x 256 code bytes, on an
// MI355X), so s << 23 serves every scale byte (255: NaN) whatever lies above it,
// and E2M1 x 2^(s - 127) is a bf16 value
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
// Gather: the batch's rows as the cache holds them, a wave per row, 8 elements a
// lane.  Bound: the bytes read and written (74k rows of 8 heads of 64 from bf16 pages
// 50 us, 6.1 TB/s, from MXFP4 35 us, 5.5); a short call by a wave's chain of lookup,
// page id and loads (36 rows 2.5 us; 6.8k 5.3 and 5.4, MXFP4 at 3.3 TB/s).
// ---------------------------------------------------------------------------
template <bool F4>
__global__ __launch_bounds__(256) void k_paged_gather(PagedKv kv, PagedRows r,
                                                      uint16_t* __restrict__ k_out,
                                                      uint16_t* __restrict__ v_out) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= r.n_rows) return;
  int b, pos;
  if (!paged_row(r, kv.page_log2, kPagedLongest, row, true, b, pos)) return;
  const int id = r.table[(int64_t)b * r.max_pages + (pos >> kv.page_log2)];
  if ((unsigned)id >= (unsigned)kv.n_pages) {
    if (lane == 0) flag_dev_err(r.err, kDevErrPageId);
    return;
  }
  const int per = kv.D >> 3, items = kv.Hkv * per;
  for (int it = lane; it < items; it += 64) {
    const int h = it / per, d0 = (it % per) * 8;
    const int64_t at = paged_row_at(kv, id, h, pos);
    const uint4 k = paged_load8<F4>(kv.k, kv.ks, at, kv.D, d0);
    const uint4 v = paged_load8<F4>(kv.v, kv.vs, at, kv.D, d0);
    const int64_t to = ((int64_t)row * kv.Hkv + h) * kv.D + d0;
    *reinterpret_cast<uint4*>(k_out + to) = k;
    *reinterpret_cast<uint4*>(v_out + to) = v;
  }
}

void launch_paged_gather(const PagedKv& kv, const PagedRows& r, uint16_t* k_out, uint16_t* v_out,
                         hipStream_t st) {
  const dim3 grid((unsigned)((r.n_rows + 3) / 4));
  if (kv.ks != nullptr)
    hipLaunchKernelGGL(k_paged_gather<true>, grid, dim3(256), 0, st, kv, r, k_out, v_out);
  else
    hipLaunchKernelGGL(k_paged_gather<false>, grid, dim3(256), 0, st, kv, r, k_out, v_out);
}

// ---------------------------------------------------------------------------
// Attention
//
// For a KV head g the query rows of a sequence are its (token, head of the
// group) pairs r = i G + (h mod G), so one read of a key or value serves the
// G heads and as many tokens as a tile of rows holds.  A unit of work is
// (sequence, tile of R rows, KV head); its keys are cut into chunks of one
// size for the whole call, and a block takes a chunk of a unit.
//
// The chunk is chosen on the device from the lengths that are there: W = sum of
// (row tiles x keys) over the sequences, chunk = W Hkv / target rounded up, so
// that about `target` blocks of equal work exist whatever the lengths are (a
// batch of one long and many short sequences fills the chip as evenly as equal
// ones).  Every wave finds its block's place by itself, lane = sequence, so
// there is no planning launch and nothing on the host depends on the lengths.
//   blocks  <= W Hkv / chunk + units <= target + units: the host's grid;
//   blocks of units with more than one chunk (ceil(x) <= 2 x for x > 1)
//           <= 2 target: their partial results have slots in the workspace.
// A unit with one chunk is finished by its block.  Of several, each block
// leaves (o, m, l) in its slot and arrives on the unit's counter; the last to
// arrive joins them (stores and loads at agent scope, as in k_attn_split).
// ---------------------------------------------------------------------------
constexpr int kPaTarget = 1024;   // blocks of equal work to aim at: 4 per CU
constexpr int kPmTarget = 512;    // of the many-row kernel: 2 per CU (768 and 1024: 256
                                  // rows of 4000 tokens 55 -> 60 and 69 us, for the joins)
constexpr int kPaFew = 32;        // (token, head) rows per KV head of the few-row kernel
constexpr int kPaArrive = 16;     // ints from one arrival counter to the next
constexpr int kPaMaxBlocks = 1 << 24;  // of 256 threads: a launch holds fewer than 2^32
constexpr float kLog2e = 1.4426950408889634f;
// A row's reference m (in log2 units) may trail its maximum by this much, so that
// most steps neither compare it across the four lanes of a row nor rescale: a
// weight is then up to 2^8, far from any limit, and as exact as one below 1.
constexpr float kPaLag = 8.0f;

typedef float pf4 __attribute__((ext_vector_type(4)));
typedef __bf16 pbf8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ pf4 pa_mfma(const uint4& a, const uint4& b, pf4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pbf8, a),
                                                 __builtin_bit_cast(pbf8, b), c, 0, 0, 0);
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A block's work: keys [k0, k1) of a unit, all wave-uniform.
struct PaWork {
  int b, start, n, len;  // the sequence, its rows and tokens
  int row0;              // the tile's first (token, head) row
  int lo, k0, k1;        // lo: the first key that any row of the tile sees
  int tok0, tok1;        // the tokens of its first and last row
  int chunks, slot;      // of the unit; the slot of its chunk 0
  int c;
  int G;                 // query heads of a KV head, and 1 / G
  float rG;
  __device__ explicit PaWork(const PagedAttnArgs& a) : G(a.G), rG(1.0f / (float)a.G) {}
};

// A sequence's rows (n = 0: none) and length.
struct PaSeq {
  int start, n, len;
};
__device__ __forceinline__ PaSeq pa_seq(const PagedAttnArgs& a, int b) {
  PaSeq q;
  const int at = min(b, a.r.B - 1);
  const bool ok = paged_seq(a.r, a.kv.page_log2, at, q.start, q.n, q.len);
  q.n = ok && b < a.r.B && q.len > 0 ? q.n : 0;
  return q;
}
// The same where it is the kernel's: FEW the ones of up to `few` (token, head) rows
// per KV head, otherwise the longer ones.
template <bool FEW>
__device__ __forceinline__ PaSeq pa_of(const PagedAttnArgs& a, int few, PaSeq q) {
  q.n = (q.n * a.G <= few) == FEW ? q.n : 0;
  return q;
}

// n / d for 0 <= n < 2^31, d > 0, with r = 1 / d to fp32: the fp32 quotient of up
// to 2^22 is off by at most one (an integer division is some 40 instructions, and
// every block makes a dozen before its first load).
__device__ __forceinline__ int pa_div(int n, int d, float r) {
  if (n >= 1 << 22) return n / d;
  int q = (int)((float)n * r);
  const int rest = n - q * d;
  q += rest >= d ? 1 : 0;
  return q - (rest < 0 ? 1 : 0);
}
// inclusive sums over the wave's lanes
template <int CTRL, int ROWS>
__device__ __forceinline__ int pa_add_from(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int pa_scan(int x) {
  x = pa_add_from<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
  x = pa_add_from<0x112, 0xF>(x);
  x = pa_add_from<0x114, 0xF>(x);
  x = pa_add_from<0x118, 0xF>(x);
  x = pa_add_from<0x142, 0xA>(x);  // a row's last lane into the next row
  return pa_add_from<0x143, 0xC>(x);  // lane 31 into the upper half
}

// Keys that any row tile of a sequence may take, its first key rounded down to
// a multiple of ALIGN.
template <int R, int ALIGN>
__device__ __forceinline__ int pa_span(const PagedAttnArgs& a, int G, int len) {
  if (a.window <= 0 || a.window >= len) return len;
  return min(len, a.window + (R - 1) / G + ALIGN);
}

// Row tiles of a sequence, and its blocks in chunks of `chunk` (rc = 1 / chunk).
template <int R>
__device__ __forceinline__ int pa_tiles(const PaWork& w, const PaSeq& q) {
  return (int)((unsigned)(q.n * w.G + R - 1) / R);
}
template <int R, int ALIGN>
__device__ __forceinline__ int pa_chunks(const PagedAttnArgs& a, const PaWork& w, const PaSeq& q,
                                         int chunk, float rc) {
  return pa_div(pa_span<R, ALIGN>(a, w.G, q.len) + chunk - 1, chunk, rc);
}

// The most rows of a sequence that the few-row kernel takes.  All, where the whole
// call is kPaSmall 16-row tiles x keys x KV heads at most: with so little work the
// length of a block's chain counts, and 16 rows have a short one.  128 rows at a time
// against 16, heads of 64, 8 KV heads for 8 unless given: 200 rows of 300 tokens (31000)
// 16.7 -> 7.7 us, 300 of 1000 (152000) 22.6 -> 11.2, 64 heads, 100 of 500 (200000) 21.5
// -> 12.1 and 200 of 300 (240000) 17.2 -> 13.8 (heads of 128 23.5 -> 22.2).  Further up
// the two cross: 64 heads, 400 of 400 (640000) 22.7 and 24.1, heads of 128 32 and 41.
// Both kernels compute it from the same numbers.
constexpr int kPaSmall = 262144;
__device__ __forceinline__ int pa_few_rows(const PagedAttnArgs& a, const PaWork& w,
                                           const PaSeq& first, int turns) {
  if (!a.small) return kPaFew;
  float work = 0.0f;
  auto add = [&](const PaSeq& q) {
    work += (float)pa_tiles<16>(w, q) * (float)pa_span<16, 32>(a, w.G, q.len);
  };
  add(first);
  for (int j = 1; j < turns; ++j) add(pa_seq(a, 64 * j + (threadIdx.x & 63)));
  return uni(wave_sum(work) * (float)a.kv.Hkv <= kPaSmall * 1.001f ? 1 << 30 : kPaFew);
}

// The work of block `idx` of `blocks` (of every KV head alike); false when there is
// none.
// ALIGN: units start at a multiple of it; MINC: the least chunk (chunks are
// multiples of 128); TARGET: blocks to aim at; PLACES: blocks that the chip holds
// at once; FIT: MXFP4.  Lane = sequence, 64 at a time.
template <bool FEW, int R, int ALIGN, int MINC, int TARGET, int PLACES, bool FIT>
__device__ __forceinline__ bool pa_work(const PagedAttnArgs& a, int idx, int blocks, bool report,
                                        PaWork& w) {
  const int lane = threadIdx.x & 63;
  const int turns = (a.r.B + 63) >> 6;
  if (report)  // one block of the launch: the sequences that do not fit
    for (int b = lane; b < a.r.B; b += 64) {
      int start, n, len;
      if (!paged_seq(a.r, a.kv.page_log2, b, start, n, len) && len != 0)
        flag_dev_err(a.r.err, kDevErrPagedRows);
    }
  const PaSeq first = pa_seq(a, lane);  // the only ones of up to 64
  const int few = pa_few_rows(a, w, first, turns);
  PaSeq q = pa_of<FEW>(a, few, first);
  float work = 0.0f, most = 0.0f, units = 0.0f;
  auto add = [&](const PaSeq& p) {
    const float span = (float)pa_span<R, ALIGN>(a, w.G, p.len), tiles = (float)pa_tiles<R>(w, p);
    work += tiles * span;
    units += tiles;
    most = fmaxf(most, tiles > 0.0f ? span : 0.0f);
  };
  add(q);
#pragma unroll 4
  for (int j = 1; j < turns; ++j) add(pa_of<FEW>(a, few, pa_seq(a, 64 * j + lane)));
  // 1.001: the fp32 sum and this product are each off by a few 2^-24.  From
  // 2^30 on no sequence is longer than a chunk.
  const float share = wave_sum(work) * (float)a.kv.Hkv * (1.001f / TARGET);
  // Cutting costs the partial results and the join, by the last block of a unit, one
  // chunk after another:
  // - up to 512 keys are not cut (8 sequences of 40 rows of 300 tokens 24.5 -> 16.7 us);
  // - nor are few rows whose blocks run all at once and none of which is much longer
  //   than a CU's share of the work (of 256; a block alone reads about as fast): 64
  //   sequences of 1000 tokens 31.4 -> 24.0, of 50 to 1500 28.8 -> 25.8; MXFP4 blocks
  //   are slower (64 of 50 to 4000 28.5 -> 32), so two thirds of it there;
  // - chunks of n keys are sqrt(cost n) at least, the cost of joining one against that
  //   of a key (one sequence of 16000 tokens 15.5 -> 12.5, of 30000 25.7 -> 20.5; tiles
  //   of 128 rows: 32 rows of 8000, 64 heads for 8, 68 -> 40, 100 of 60000 of 2 heads
  //   239 -> 88).
  most = wave_max(most);
  const float cost = __builtin_sqrtf((FEW ? 10.0f : 25.0f) * most);
  float least = fmaxf(share, most <= 512.0f ? 511.0f : cost);
  if (FEW && most <= share * (TARGET / (FIT ? 384.0f : 256.0f)) + 512.0f &&
      wave_sum(units) * (float)a.kv.Hkv <= (float)PLACES)
    least = fmaxf(least, most);
  int chunk = uni(max(MINC, (min((int)min(least, 0x1p30f), (1 << 30) - 128) + 128) & ~127));
  // The blocks of the sequences, in order, up to the one that idx lies in.  Row
  // starts that overlap (an error that no single sequence shows) can sum to more
  // blocks than the grid has: the clamp lies above every grid and keeps the sums
  // in an int.
  int at = 0, slot = 0, nc = 0;  // blocks and slots of the sequences before
  float rc = 0.0f;
  uint64_t mine = 0;
  int j = 0;
  for (int fit = 0;; ++fit) {
    rc = 1.0f / (float)chunk;
    nc = pa_chunks<R, ALIGN>(a, w, q, chunk, rc);
    const int nb = min(pa_tiles<R>(w, q) * nc, kPaMaxBlocks);
    const int to = pa_scan(nb), all = __builtin_amdgcn_readlane(to, 63);
    // FIT: a few more blocks than the chip holds cost a round of their own, so
    // larger chunks where that makes them fit (a unit is one block at least).
    // MXFP4, 4 sequences up to 131072 tokens 38.6 -> 37.4 us, 48 of 100 to 6000, heads
    // of 128, 40.9 -> 36.9; where the reads are the bound, small chunks even out the end
    // better (64 bf16 ones: 68 -> 73 us).
    const float over = (float)all * (float)a.kv.Hkv * (1.0f / PLACES);
    if (FIT && fit < 3 && turns == 1 && over > 1.0f && over <= 2.0f) {
      chunk = uni((min((int)((float)chunk * over), (1 << 30) - 128) + 128) & ~127);
      continue;
    }
    const int slots = nc > 1 ? nb : 0, slots_to = pa_scan(slots);
    mine = __ballot(idx < to);
    at = to - nb;
    slot = slots_to - slots;
    if (mine != 0) break;
    const int all_slots = __builtin_amdgcn_readlane(slots_to, 63);
    int before = all, slots_before = all_slots;
    for (j = 1; j < turns; ++j) {
      q = pa_of<FEW>(a, few, pa_seq(a, 64 * j + lane));
      nc = pa_chunks<R, ALIGN>(a, w, q, chunk, rc);
      const int nb2 = min(pa_tiles<R>(w, q) * nc, kPaMaxBlocks), s2 = nc > 1 ? nb2 : 0;
      const int to2 = pa_scan(nb2), st2 = pa_scan(s2);
      mine = __ballot(idx - before < to2);
      at = before + to2 - nb2;
      slot = slots_before + st2 - s2;
      if (mine != 0) break;
      before += __builtin_amdgcn_readlane(to2, 63);
      slots_before += __builtin_amdgcn_readlane(st2, 63);
    }
    break;
  }
  if (mine == 0) return false;
  const int owner = __builtin_ctzll(mine);
  w.b = 64 * j + owner;
  w.start = __builtin_amdgcn_readlane(q.start, owner);
  w.n = __builtin_amdgcn_readlane(q.n, owner);
  w.len = __builtin_amdgcn_readlane(q.len, owner);
  nc = __builtin_amdgcn_readlane(nc, owner);
  const int rel = idx - __builtin_amdgcn_readlane(at, owner);
  const int tiles = (int)((unsigned)(w.n * w.G + R - 1) / R);
  const int before = uni(rel / nc);
  const int tile = tiles - 1 - before;  // the last tiles first: they see the most keys
  w.c = rel - before * nc;
  w.row0 = tile * R;
  w.slot = __builtin_amdgcn_readlane(slot, owner) + tile * nc;
  const int last = min(w.row0 + R, w.n * w.G) - 1;
  w.tok0 = uni(pa_div(w.row0, w.G, w.rG));
  w.tok1 = uni(pa_div(last, w.G, w.rG));
  const int pos0 = w.len - w.n + w.tok0, pos1 = w.len - w.n + w.tok1;
  w.lo = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
  const int from = w.lo / ALIGN * ALIGN;
  w.chunks = uni(pa_div(pos1 + 1 - from + chunk - 1, chunk, rc));
  w.k0 = from + w.c * chunk;
  w.k1 = min(w.k0 + chunk, pos1 + 1);
  // a unit past the grid's end (only row starts that overlap make one) is left out
  // whole: its counter would not come back to 0
  return w.c < w.chunks && idx - w.c + w.chunks <= blocks;
}

// How the kernels take a 16-key step of a wave: S^T = K Q^T with
// v_mfma_f32_16x16x32_bf16 (A: lane c = lane % 16 a key, group g = lane / 16
// eight dims; B: lane c a query row), so lane (g, c) holds the scores of row c
// for the keys 4 g + i, which is also how the second product's B operand wants
// them: O^T = V^T P^T over 32 keys k = 8 g + j, j < 4 the key 4 g + j of the
// first 16 and j >= 4 that of the second.  Its A operand needs eight keys'
// values of one dim in a lane: lane c reads the dims (D/16) c .. of its eight
// keys and two 16-bit halves are paired by a byte permute, so nothing goes
// through LDS or other lanes.  The results of row c for the dims (D/4) g ..
// are in lane (g, c), with the running maximum and sum of row c.

// A wave's two 16-key steps as they come from memory.
template <int D, bool F4>
struct PaTile;
template <int D>
struct PaTile<D, false> {
  uint4 k[2][D / 32];      // dims 32 n + 8 g ..
  uint32_t v[2][4][D / 32];  // keys 4 g + i, dims (D/16) c ..
};
template <int D>
struct PaTile<D, true> {
  uint32_t k[2][D / 32];     // codes of dims (D/4) g ..
  uint32_t v[2][4];          // the word with the codes of keys 4 g + i, dims (D/16) c ..
  uint32_t ks[2];            // the word with the scale of the key's block
  uint32_t vs[2][D / 32];    // scales of the keys 4 g .. 4 g + 3
};
// Words, though D = 64 needs two bytes of v and D / 32 of ks: a narrower load's
// zero extension ends up behind the loop's join, where it waits for the step that
// was only just requested.

template <int D>
__device__ __forceinline__ void pa_load(PaTile<D, false>& t, const PagedKv& kv, int g, int c,
                                        const int64_t (&at)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint8_t* kp = kv.k + at[s] * (2 * D);
    const uint8_t* vp = kv.v + at[s] * (2 * D);
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
      t.k[s][n] = *reinterpret_cast<const uint4*>(kp + (uint32_t)(c * 2 * D + 64 * n + 16 * g));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* p = vp + (uint32_t)((4 * g + i) * 2 * D + (D / 8) * c);
      if constexpr (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        t.v[s][i][0] = x.x; t.v[s][i][1] = x.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        t.v[s][i][0] = x.x; t.v[s][i][1] = x.y; t.v[s][i][2] = x.z; t.v[s][i][3] = x.w;
      }
    }
  }
}
template <int D>
__device__ __forceinline__ void pa_load(PaTile<D, true>& t, const PagedKv& kv, int g, int c,
                                        const int64_t (&at)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint8_t* kp = kv.k + at[s] * (D / 2);
    const uint8_t* vp = kv.v + at[s] * (D / 2);
    const uint8_t* ksp = kv.ks + at[s] * (D / 32);
    const uint8_t* vsp = kv.vs + at[s] * (D / 32);
    t.ks[s] = *reinterpret_cast<const uint32_t*>(ksp + (uint32_t)(c * (D / 32) & ~3));
    if constexpr (D == 64) {
      const uint2 x = *reinterpret_cast<const uint2*>(kp + (uint32_t)(c * 32 + 8 * g));
      t.k[s][0] = x.x; t.k[s][1] = x.y;
      const uint2 y = *reinterpret_cast<const uint2*>(vsp + (uint32_t)(8 * g));
      t.vs[s][0] = y.x; t.vs[s][1] = y.y;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t.v[s][i] = *reinterpret_cast<const uint32_t*>(vp + (uint32_t)((4 * g + i) * 32 + (2 * c & ~3)));
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(kp + (uint32_t)(c * 64 + 16 * g));
      t.k[s][0] = x.x; t.k[s][1] = x.y; t.k[s][2] = x.z; t.k[s][3] = x.w;
      const uint4 y = *reinterpret_cast<const uint4*>(vsp + (uint32_t)(16 * g));
      t.vs[s][0] = y.x; t.vs[s][1] = y.y; t.vs[s][2] = y.z; t.vs[s][3] = y.w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t.v[s][i] = *reinterpret_cast<const uint32_t*>(vp + (uint32_t)((4 * g + i) * 64 + 4 * c));
    }
  }
}

// Steps at the edge: keys that some rows see and others do not, and rows of a page
// that hold no key of the sequence and may hold anything.  A weight of 0 would turn
// an infinity or a NaN among their values into a NaN of a row that does not see
// it, so such values are cleared on the way, and where a key of the sequence had
// one (`odd`), the rows that see it get it after the last step (pa_odd_values).
__device__ __forceinline__ uint32_t pa_odd_halves(uint32_t w) {  // 0xFFFF in each
  return ((w & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) |
         ((w & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u);
}
// clears key i's values: all (none), or the odd ones
template <int D>
__device__ __forceinline__ void pa_clear(PaTile<D, false>& t, int s, int i, int, bool none, bool& odd) {
#pragma unroll
  for (int n = 0; n < D / 32; ++n) {
    const uint32_t m = pa_odd_halves(t.v[s][i][n]);
    odd = odd || (m != 0 && !none);
    t.v[s][i][n] = none ? 0u : t.v[s][i][n] & ~m;
  }
}
template <int D>
__device__ __forceinline__ void pa_clear(PaTile<D, true>& t, int s, int i, int c, bool none, bool& odd) {
  // its scales' word, the bytes of the others there, and the scale of the lane's dims
  uint32_t& word = t.vs[s][i * (D / 32) >> 2];
  const uint32_t keep = D == 128 ? 0u : i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
  const uint32_t byte = D == 64 ? word >> (16 * (i & 1) + (c & 8)) : word >> (2 * (c & 12));
  const bool nan = (byte & 0xFFu) == 0xFFu;
  const bool clear = none || nan;
  // 4 and 6 times 2^126, and from 2 on times 2^127, read as infinities: those codes
  // (the word's other lanes' too, which this lane does not use)
  const uint32_t two = t.v[s][i] & 0x44444444u, four = two & t.v[s][i] << 1;
  uint32_t inf = (byte & 0xFFu) == 254u ? two : (byte & 0xFFu) == 253u ? four : 0u;
  inf |= inf << 1 | inf >> 1 | inf >> 2;
  odd = odd || ((nan || inf != 0) && !none);
  t.v[s][i] = clear ? 0u : t.v[s][i] & ~inf;
  word = clear ? word & keep : word;
}
// fn(key, value(d)) for the keys [kb, kb + n): the infinities and NaNs of a value, 0
// for a finite one, from the pages again.
template <int D, bool F4, class F>
__device__ __forceinline__ void pa_odd_values(const PagedAttnArgs& a, const PaWork& w, int h, int kb,
                                              int n, F fn) {
  const int32_t* table = a.r.table + (int64_t)w.b * a.r.max_pages;
  for (int key = max(kb, w.lo); key < min(kb + n, w.k1); ++key) {
    const int id = table[key >> a.kv.page_log2];
    if ((unsigned)id >= (unsigned)a.kv.n_pages) continue;
    const int64_t at = paged_row_at(a.kv, id, h, key);
    fn(key, [&](int d) {
      const uint4 x = paged_load8<F4>(a.kv.v, a.kv.vs, at, D, d & ~7);
      const uint32_t u = d & 4 ? (d & 2 ? x.w : x.z) : (d & 2 ? x.y : x.x);
      const float v = d & 1 ? bf_hi(u) : bf_lo(u);
      return fabsf(v) < INFINITY ? 0.0f : v;
    });
  }
}

// operand n of a 16-key step's keys: the dims that pa_query gives B
template <int D>
__device__ __forceinline__ uint4 pa_key(const PaTile<D, false>& t, int s, int n, int, int) {
  return t.k[s][n];
}
template <int D>
__device__ __forceinline__ uint4 pa_key(const PaTile<D, true>& t, int s, int n, int g, int c) {
  // byte (c & 1) 2 + g / 2 (D = 64) or g of the scales' word
  return mx4_to_bf16x8(t.k[s][n], t.ks[s] >> (D == 64 ? 16 * (c & 1) + 8 * (g >> 1) : 8 * g));
}
template <int D, bool F4>
__device__ __forceinline__ int pa_query_dim(int n, int g) {
  return F4 ? (D / 4) * g + 8 * n : 32 * n + 8 * g;
}
// values of key 4 g + i, dims (D/16) c ..
template <int D>
__device__ __forceinline__ void pa_value(const PaTile<D, false>& t, int s, int i, int,
                                         uint32_t (&v)[D / 32]) {
#pragma unroll
  for (int n = 0; n < D / 32; ++n) v[n] = t.v[s][i][n];
}
template <int D>
__device__ __forceinline__ void pa_value(const PaTile<D, true>& t, int s, int i, int c,
                                         uint32_t (&v)[D / 32]) {
  // The key's scale byte is byte (i & 1) 2 + c / 8 of word i / 2 (D = 64), byte
  // c / 4 of word i (D = 128); the bytes beside it need no mask.
  const uint32_t b = D == 64 ? t.vs[s][i >> 1] >> (c & 8) : t.vs[s][i] >> (2 * (c & 12));
  const float sc = __uint_as_float(b << (D == 64 && (i & 1) ? 7 : 23));
  const uint32_t w = D == 64 ? t.v[s][i] >> (16 * (c & 1)) : t.v[s][i];
  v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
  v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
  if constexpr (D == 128) {
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
  }
}

// Joins o (unnormalised, with maximum m in log2 units and sum l) with the sink
// and gives the factor that finishes it: 0 where nothing was seen.
__device__ __forceinline__ float pa_finish(const PagedAttnArgs& a, int h, float m, float l) {
  if (a.sinks == nullptr) return l == 0.0f ? 0.0f : 1.0f / l;
  const float sk = bf2f(a.sinks[h]) * kLog2e, M = fmaxf(m, sk);
  if (M == -INFINITY) return 0.0f;
  const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
  const float den = l * f + __builtin_amdgcn_exp2f(sk - M);
  return den == 0.0f ? 0.0f : f / den;
}

__device__ __forceinline__ uint64_t pa_pair(float x, float y) {
  return (uint64_t)__float_as_uint(x) | ((uint64_t)__float_as_uint(y) << 32);
}
__device__ __forceinline__ void pa_store_agent(float* p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), pa_pair(x, y), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pa_load_agent(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Joins what the chunks' blocks left of a tile's 16 rows (in the same launch:
// agent-scope loads), `used` of them: o at part + chunk * step + row D, (m, l)
// behind the rows.  256 threads: 16 for a row's D values; where fewer than 16
// rows are used, the others take a share of the chunks.  fn(row, E values, m, l)
// by 16 threads per row, thread t with the values (t & 15) E ..
// Without the shares and with one chunk's loads at a time the join of a tile of 92
// chunks took 25 us; the whole call for one sequence of 30000 tokens takes 20.
constexpr int kPaJoin = 64;  // chunks whose factors are in LDS at once
template <int D, class F>
__device__ __forceinline__ void pa_join(const float* part, int64_t step, int chunks, int used,
                                        float (*sf)[kPaJoin], float (*sx)[D + 4], F fn) {
  constexpr int R = 16, E = D / 16;
  const int tid = threadIdx.x, lane16 = tid & 15, row16 = tid >> 4;
  const int rows2 = used > 8 ? 16 : used > 4 ? 8 : used > 2 ? 4 : used > 1 ? 2 : 1;
  const int shares = 16 / rows2, share = row16 / rows2, row = row16 & (rows2 - 1);
  float M = -INFINITY, L = 0.0f, x[E];  // M, L of row row16
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.0f;
  const float* pml = part + R * D + 2 * row16;
  for (int c0 = 0; c0 < chunks; c0 += kPaJoin) {
    // the factors of these chunks for row row16, 16 lanes of it
    float2 ml[kPaJoin / 16];
    float mx = M;
#pragma unroll
    for (int i = 0; i < kPaJoin / 16; ++i) {
      const int j = c0 + lane16 + 16 * i;
      ml[i] = pa_load_agent(pml + min(j, chunks - 1) * step);
      if (j >= chunks) ml[i] = make_float2(-INFINITY, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < kPaJoin / 16; ++i) mx = fmaxf(mx, ml[i].x);
    mx = fmaxf(mx, xor_lane<1>(mx));
    mx = fmaxf(mx, xor_lane<2>(mx));
    mx = fmaxf(mx, xor_lane<4>(mx));
    mx = fmaxf(mx, xor_lane<8>(mx));
    const float me = mx == -INFINITY ? 0.0f : mx;
    const float old = __builtin_amdgcn_exp2f(M - me);
    float sum = 0.0f;
    __syncthreads();  // sf is free
#pragma unroll
    for (int i = 0; i < kPaJoin / 16; ++i) {
      const float f = __builtin_amdgcn_exp2f(ml[i].x - me);
      sf[row16][lane16 + 16 * i] = f;
      sum = __builtin_fmaf(ml[i].y, f, sum);
    }
    sum += xor_lane<1>(sum);
    sum += xor_lane<2>(sum);
    sum += xor_lane<4>(sum);
    sum += xor_lane<8>(sum);
    L = __builtin_fmaf(L, old, sum);
    M = mx;
    if (c0 > 0) {  // the values so far, of row `row`
      if (lane16 == 0) sx[row16][0] = old;
      __syncthreads();
      const float f = sx[row][0];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] *= f;
    }
    __syncthreads();
    const int n = min(kPaJoin, chunks - c0);
    const float* po = part + c0 * step + row * D + lane16 * E;
    // U chunks' loads at a time
    auto take = [&](auto u_t, int j0) {
      constexpr int U = decltype(u_t)::value;
      float2 y[U][E / 2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* p = po + min(j0 + u * shares, n - 1) * step;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) y[u][e] = pa_load_agent(p + 2 * e);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j0 + u * shares >= n) break;
        const float f = sf[row][j0 + u * shares];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          x[2 * e] = __builtin_fmaf(y[u][e].x, f, x[2 * e]);
          x[2 * e + 1] = __builtin_fmaf(y[u][e].y, f, x[2 * e + 1]);
        }
      }
    };
    if (n <= 2 * shares) {
      take(std::integral_constant<int, 2>{}, share);
    } else if (n <= 4 * shares) {
      take(std::integral_constant<int, 4>{}, share);
    } else {
      for (int j0 = share; j0 < n; j0 += 8 * shares) take(std::integral_constant<int, 8>{}, j0);
    }
  }
  // the shares of a row; sx row: share * rows2 + row
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) sx[row16][lane16 * E + e] = x[e];
  __syncthreads();
  if (row16 < rows2) {
    for (int k = 1; k < shares; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += sx[k * rows2 + row16][lane16 * E + e];
    if (row16 < used) fn(row16, x, M, L);
  }
}
template <int E>
__device__ __forceinline__ void pa_write(uint16_t* dst, const float (&x)[E], float fin) {
#pragma unroll
  for (int e = 0; e < E; e += 4)
    *reinterpret_cast<uint2*>(dst + e) = make_uint2(pack_bf2(x[e] * fin, x[e + 1] * fin),
                                                    pack_bf2(x[e + 2] * fin, x[e + 3] * fin));
}

// Few rows: 16 per unit, four waves that share nothing but the result, each
// with every fourth 32 keys of the chunk, straight from memory into the
// operands' registers, some steps ahead of the products.
// Bound: the bytes of the visible keys, read once (64 sequences of up to 8192
// tokens, 8 heads of 64 for 64: 285 MB in 65 us, 4.4 TB/s; 256 of 2000: 5.2 TB/s);
// MXFP4 at 2.9 to 3.6 TB/s by the vector units as well, which expand the codes
// (48 sequences of up to 6000 tokens, heads of 128: 73 MB in 25 us, 53% busy); few short
// sequences by the chain of lookups, loads and the join (5 us for one of 64 tokens).
// Waves of a SIMD, and blocks of a CU (four of D = 64: bf16 the same, MXFP4 4 sequences
// of up to 131072 tokens 30.7 -> 31.2 us, 64 of up to 4000 28 -> 26)
constexpr int pa_few_waves(int D, bool f4) { return D == 64 || f4 ? 3 : 2; }
template <int D, bool F4>
__global__ __launch_bounds__(256, pa_few_waves(D, F4)) void k_paged_attn_few(PagedAttnArgs a) {
  constexpr int R = 16, E = D / 16;
  constexpr int NT = 2;  // steps in registers: one in use, the others on their way
  constexpr int kPlaces = 256 * pa_few_waves(D, F4);
  __shared__ __align__(16) float so[4][R][D + 4];
  __shared__ float sm[4][R], sl[4][R];
  __shared__ float sf[16][kPaJoin];
  __shared__ int merge_here;
  const int h = blockIdx.x % a.kv.Hkv;
  PaWork w(a);
  if (!pa_work<true, R, 32, 256, kPaTarget, kPlaces, F4>(
          a, blockIdx.x / a.kv.Hkv, gridDim.x / a.kv.Hkv, blockIdx.x == 0, w))
    return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int G = w.G;
  // the lane's query row
  const int r = w.row0 + c, rows = w.n * G;
  const bool has = r < rows;
  const int tok = has ? pa_div(r, G, w.rG) : 0, hq = h * G + (has ? r - tok * G : 0);
  const int pos = w.len - w.n + tok;
  const int k_hi = has ? pos + 1 : 0;
  const int k_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  // keys that every row of the tile sees
  const int all_hi = w.len - w.n + w.tok0 + 1;
  const int all_lo = a.window > 0 ? max(0, w.len - w.n + w.tok1 - a.window + 1) : 0;
  uint4 q[D / 32];
  {
    const uint16_t* qp = a.q + (int64_t)(w.start + tok) * a.q_stride + (int64_t)hq * D;
#pragma unroll
    for (int n = 0; n < D / 32; ++n) {
      q[n] = *reinterpret_cast<const uint4*>(qp + pa_query_dim<D, F4>(n, g));
      if (!has) q[n] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const float c2 = (D == 64 ? 0.125f : 0.08838834764831845f) * kLog2e;
  pf4 o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY;
  float l = 0.0f;  // of the lane's keys

  const int tiles = (w.k1 - w.k0 + 31) >> 5;
  const int n_it = (tiles - wave + 3) >> 2;  // this wave's
  const int32_t* table = a.r.table + (int64_t)w.b * a.r.max_pages;
  // page ids of the 16-key steps of 32 iterations, one per lane: -1 past the
  // keys and where the table's entry is no page
  auto load_ids = [&](int it) {
    const int key = w.k0 + 32 * (wave + 4 * (it + (lane >> 1))) + 16 * (lane & 1);
    int id = -1;
    if (key < w.k1 && key + 16 > w.lo) {  // pages before the window may be gone
      id = table[key >> a.kv.page_log2];
      if ((unsigned)id >= (unsigned)a.kv.n_pages) {
        id = -1;
        flag_dev_err(a.r.err, kDevErrPageId);
      }
    }
    return id;
  };
  const int page_mask = (1 << a.kv.page_log2) - 1;
  auto load_tile = [&](PaTile<D, F4>& t, int it, int ids, int (&id)[2]) {
    const int kb = w.k0 + 32 * (wave + 4 * it);
    int64_t at[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      id[s] = __builtin_amdgcn_readlane(ids, 2 * (it & 31) + s);
      at[s] = (((int64_t)max(id[s], 0) * a.kv.Hkv + h) << a.kv.page_log2) +
              ((kb + 16 * s) & page_mask);
    }
    pa_load<D>(t, a.kv, g, c, at);
  };
  auto inside = [&](int kb) { return kb >= all_lo && kb + 32 <= all_hi; };
  bool odd = false;
  auto step = [&](PaTile<D, F4>& t, int it, const int (&id)[2]) {
    const int kb = w.k0 + 32 * (wave + 4 * it);
    // every row sees all 32 keys (else the masks: two blocks of selects under a
    // branch of the whole wave)
    const bool full = inside(kb) && (id[0] | id[1]) >= 0;
    float sv[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      pf4 acc = pf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < D / 32; ++n) acc = pa_mfma(pa_key<D>(t, s, n, g, c), q[n], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[s][i] = acc[i];
    }
    if (!full) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kb + 16 * s + 4 * g + i;
          const bool seen = (key >= k_lo) & (key < k_hi) & (id[s] >= 0);
          sv[s][i] = seen ? sv[s][i] : -INFINITY;
          pa_clear<D>(t, s, i, c, (key >= w.k1) | (key < w.lo) | (id[s] < 0), odd);
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[0][2], sv[0][3])),
                     fmaxf(fmaxf(sv[1][0], sv[1][1]), fmaxf(sv[1][2], sv[1][3]))) * c2;
    if (__any(mx > m + kPaLag)) {  // rarely, once a row has seen some keys
      mx = fmaxf(mx, xor_lane<16>(mx));
      mx = fmaxf(mx, xor_lane<32>(mx));
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= f;
      m = mn;
    }
    const float me = m == -INFINITY ? 0.0f : m;
    // P in two bf16 terms (2^-16 of a weight)
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[s][i], c2, -me));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[s][i + 1], c2, -me));
        const uint32_t x = pack_bf2(p0, p1);
        hi[2 * s + i / 2] = x;
        l += p0;
        l += p1;
        lo[2 * s + i / 2] = pack_bf2(p0 - bf_lo(x), p1 - bf_hi(x));
      }
    uint32_t v[2][4][D / 32];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) pa_value<D>(t, s, i, c, v[s][i]);
    const uint4 ph = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    const uint4 pl = make_uint4(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      uint32_t f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        f[k] = __builtin_amdgcn_perm(v[k >> 1][2 * (k & 1) + 1][e >> 1], v[k >> 1][2 * (k & 1)][e >> 1],
                                     e & 1 ? 0x07060302u : 0x05040100u);
      const uint4 vf = make_uint4(f[0], f[1], f[2], f[3]);
      o[e] = pa_mfma(vf, ph, o[e]);
      o[e] = pa_mfma(vf, pl, o[e]);
    }
  };
  if (n_it > 0) {
    PaTile<D, F4> t[NT];
    int id[NT][2];
    int ids = load_ids(0);
    // unconditional loads (past the last step, that one again): a load under a
    // condition is waited for where the paths join
#pragma unroll
    for (int u = 0; u < NT - 1; ++u) load_tile(t[u], min(u, n_it - 1), ids, id[u]);
    for (int it0 = 0; it0 < n_it; it0 += NT) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int it = it0 + u, nx = min(it + NT - 1, n_it - 1);
        if (it >= n_it) break;
        if ((nx & 31) == 0 && nx == it + NT - 1) ids = load_ids(nx);
        load_tile(t[(u + NT - 1) % NT], nx, ids, id[(u + NT - 1) % NT]);
        step(t[u], it, id[u]);
      }
    }
  }
  // An infinity among the values of a step that every row sees meets both terms of P:
  // its product with the second is the other infinity, or NaN.
  l += xor_lane<16>(l);
  l += xor_lane<32>(l);
  float z = 0.0f;  // NaN where an element is not finite
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) z = __builtin_fmaf(o[e][i], 0.0f, z);
  odd = odd || (z != z && l == l);  // (a row with a NaN among its scores is all NaN)
  if (__any(odd)) {  // lane (g, c): row c, dims (D/4) g + E i + e
    pf4 sum[E];      // of the infinities and NaNs alone
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int it = 0; it < n_it; ++it)
      pa_odd_values<D, F4>(a, w, h, w.k0 + 32 * (wave + 4 * it), 32, [&](int key, auto value) {
        const bool seen = (key >= k_lo) & (key < k_hi);
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = value((D / 4) * g + E * i + e);
            if (seen) sum[e][i] += v;
          }
      });
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[e][i] = sum[e][i] != 0.0f ? sum[e][i] : o[e][i];
  }
  // the four waves' states
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < E; e += 4)
      *reinterpret_cast<float4*>(&so[wave][c][(D / 4) * g + E * i + e]) =
          make_float4(o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]);
  if (g == 0) {
    sm[wave][c] = m;
    sl[wave][c] = l;
  }
  __syncthreads();
  // thread: row tr, dims td .. td + E - 1
  const int tr = tid >> 4, td = (tid & 15) * E;
  float M = fmaxf(fmaxf(sm[0][tr], sm[1][tr]), fmaxf(sm[2][tr], sm[3][tr]));
  float L = 0.0f, x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.0f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float f = sm[v][tr] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[v][tr] - M);
    L = __builtin_fmaf(sl[v][tr], f, L);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = __builtin_fmaf(so[v][tr][td + e], f, x[e]);
  }
  const int row = w.row0 + tr;
  if (w.chunks > 1) {
    const int64_t first = ((int64_t)w.slot * a.kv.Hkv + h);
    float* po = a.part + (first + (int64_t)w.c * a.kv.Hkv) * R * (D + 2);
#pragma unroll
    for (int e = 0; e < E; e += 2) pa_store_agent(po + tr * D + td + e, x[e], x[e + 1]);
    if ((tid & 15) == 0) pa_store_agent(po + R * D + 2 * tr, M, L);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores have completed
    __syncthreads();
    int32_t* ctr = a.arrive + first * kPaArrive;
    if (tid == 0)
      merge_here = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                   w.chunks - 1;
    __syncthreads();
    if (!merge_here) return;
    if (tid == 0) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    pa_join<D>(a.part + first * R * (D + 2), (int64_t)a.kv.Hkv * R * (D + 2), w.chunks,
                  min(R, rows - w.row0), sf, so[0], [&](int tr_, const float (&y)[E], float m_, float l_) {
                    const int tok_ = pa_div(w.row0 + tr_, G, w.rG);
                    const int head = h * G + w.row0 + tr_ - tok_ * G;
                    pa_write<E>(a.out + ((int64_t)(w.start + tok_) * a.Hq + head) * D + td, y,
                                pa_finish(a, head, m_, l_));
                  });
    return;
  }
  if (row >= rows) return;
  const int out_tok = pa_div(row, G, w.rG), head = h * G + row - out_tok * G;
  pa_write<E>(a.out + ((int64_t)(w.start + out_tok) * a.Hq + head) * D + td, x,
              pa_finish(a, head, M, L));
}

// Many rows: 128 per unit, 32 of each wave (two tiles of 16), 64 keys at a time
// through LDS, where the four waves share them.  K and V rows lie as they are,
// their words exchanged by the key's low bits so that a read touches every bank
// evenly: K by 16 bytes (16 lanes read one word of 16 keys), V by 32 (16 lanes
// read 32 bytes of 4 keys, and ds_read_b64_tr_b16 gives each lane one dim's four
// values, which are half of its A operand).  MXFP4 pages are expanded when a tile
// is written.  The next tile's loads are on their way while a tile is used, and
// LDS holds two.
// P is kept in two bf16 terms (2^-16 of a weight), as over the contiguous cache: with
// one, 2^-9 of a weight, the prompt chunk below took 253 us.
// Bound: the vector units (76% busy: an exponential and some eight plain instructions
// a score) beside the matrix units (39%): the last 2048 and 819 rows of 6001 and 2925
// tokens, 64 heads, in 341 us, 590 TFLOP/s; one prompt of 8192 tokens 609, heads of
// 128 690.
typedef short ps4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 pa_read_tr(const void* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) ps4*)p));
}
template <int D>
struct PmStage {  // a thread's part of a tile on its way
  uint4 k[D / 32], v[D / 32];
};

// pa_join for a tile of 128 rows: two threads a row for its maximum, sum and the
// chunks' factors sf; then groups of four values, NG of a thread at a time, with U
// chunks' loads on their way: all rows and two (or one) of up to 8 chunks, else
// 4096 / D rows and four (40 rows of 60000 tokens, 8 heads of 128, 146 -> 128 us; 256 of
// 4000 the other way round, 57 -> 55).  By 16 rows at a time, every step for each, two
// chunks of 128 rows of 128 took 13 us.
constexpr int kPmJoin = 32;  // chunks whose factors are in LDS at once
template <int D>
__device__ __forceinline__ void pm_join(const PagedAttnArgs& a, const PaWork& w, int h,
                                        const float* part, int64_t step, float (*sf)[kPmJoin],
                                        float* fin) {
  constexpr int R = 128, Q = D / 4;  // Q groups of a row
  const int tid = threadIdx.x, row = tid >> 1, side = tid & 1;
  const int used = min(R, w.n * w.G - w.row0);
  const float* pml = part + R * D + 2 * row;
  // (m, l) of the chunks from c0 on, every second one of U each
  auto load = [&](auto& ml, int c0) {
    const int n = w.chunks - c0;
#pragma unroll
    for (int u = 0; u < (int)(sizeof(ml) / sizeof(ml[0])); ++u) {
      ml[u] = pa_load_agent(pml + (c0 + min(side + 2 * u, n - 1)) * step);
      if (side + 2 * u >= n) ml[u] = make_float2(-INFINITY, 0.0f);
    }
  };
  float M = -INFINITY, L = 0.0f;
  auto put = [&](const auto& ml) {
    const float me = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int u = 0; u < (int)(sizeof(ml) / sizeof(ml[0])); ++u)
      sf[row][side + 2 * u] = __builtin_amdgcn_exp2f(ml[u].x - me);
  };
  auto totals = [&](auto u_t) {
    constexpr int U = decltype(u_t)::value;
    float2 ml[U];
    for (int c0 = 0; c0 < w.chunks; c0 += 2 * U) {
      load(ml, c0);
      float mx = M;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, ml[u].x);
      mx = fmaxf(mx, xor_lane<1>(mx));
      const float me = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        sum = __builtin_fmaf(ml[u].y, __builtin_amdgcn_exp2f(ml[u].x - me), sum);
      sum += xor_lane<1>(sum);
      L = __builtin_fmaf(L, __builtin_amdgcn_exp2f(M - me), sum);
      M = mx;
    }
    if (w.chunks <= kPmJoin) put(ml);
  };
  if (w.chunks <= 4) totals(std::integral_constant<int, 2>{});
  else if (w.chunks <= 8) totals(std::integral_constant<int, 4>{});
  else totals(std::integral_constant<int, kPmJoin / 2>{});
  auto place = [&](int r, int& tok, int& head) {
    tok = pa_div(w.row0 + r, w.G, w.rG);
    head = h * w.G + w.row0 + r - tok * w.G;
  };
  __syncthreads();
  auto join = [&](auto ng_t, auto u_t) {
    constexpr int NG = decltype(ng_t)::value, U = decltype(u_t)::value, RB = 1024 * NG / D;
    const uint32_t lane4 = 4 * tid;
#pragma unroll 1
    for (int r0 = 0; r0 < used; r0 += RB) {
      float4 x[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
      for (int c0 = 0; c0 < w.chunks; c0 += kPmJoin) {
        if (w.chunks > kPmJoin) {
          float2 ml[kPmJoin / 2];
          load(ml, c0);
          __syncthreads();
          put(ml);
          __syncthreads();
        }
        const int n = min(kPmJoin, w.chunks - c0);
        for (int j0 = 0; j0 < n; j0 += U) {
          float2 y[U][NG][2];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const float* p = part + (c0 + min(j0 + u, n - 1)) * step + r0 * D;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              y[u][i][0] = pa_load_agent(p + 1024 * i + lane4);
              y[u][i][1] = pa_load_agent(p + 1024 * i + 2 + lane4);
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (j0 + u >= n) break;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              const float f = sf[r0 + (tid + 256 * i) / Q][j0 + u];
              x[i].x = __builtin_fmaf(y[u][i][0].x, f, x[i].x);
              x[i].y = __builtin_fmaf(y[u][i][0].y, f, x[i].y);
              x[i].z = __builtin_fmaf(y[u][i][1].x, f, x[i].z);
              x[i].w = __builtin_fmaf(y[u][i][1].y, f, x[i].w);
            }
          }
        }
      }
      if (r0 == 0) {
        if (side == 0 && row < used) {
          int tok, head;
          place(row, tok, head);
          fin[row] = pa_finish(a, head, M, L);
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int r = r0 + (tid + 256 * i) / Q;
        if (r >= used) break;
        int tok, head;
        place(r, tok, head);
        const float f = fin[r];
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(w.start + tok) * a.Hq + head) * D +
                                  4 * (tid % Q)) =
            make_uint2(pack_bf2(x[i].x * f, x[i].y * f), pack_bf2(x[i].z * f, x[i].w * f));
      }
    }
  };
  if (used > 64 && w.chunks <= 8)
    join(std::integral_constant<int, D / 8>{}, std::integral_constant<int, 128 / D>{});
  else
    join(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
}

// Three blocks of a CU at D = 64 (168 registers; 169, and so two of them, made the
// prompt chunk 393 us), two at 128.
template <int D, bool F4>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void k_paged_attn_many(PagedAttnArgs a) {
  constexpr int R = 128, E = D / 16, W = D / 8;  // W: 16-byte words of a row
  __shared__ __align__(16) uint4 kt[2][64 * W], vt[2][64 * W];
  __shared__ int merge_here, odd;
  const int h = blockIdx.x % a.kv.Hkv;
  PaWork w(a);
  if (!pa_work<false, R, 64, 256, kPmTarget, 512, false>(
          a, blockIdx.x / a.kv.Hkv, gridDim.x / a.kv.Hkv, blockIdx.x == 0, w))
    return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int G = w.G, rows = w.n * G, pos0 = w.len - w.n;
  const float c2 = (D == 64 ? 0.125f : 0.08838834764831845f) * kLog2e;
  uint4 q[2][D / 32];
  int k_hi[2], k_lo[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = w.row0 + 32 * wave + 16 * t + c;
    const bool has = r < rows;
    const int tok = has ? r / G : 0, hq = h * G + (has ? r % G : 0);
    k_hi[t] = has ? pos0 + tok + 1 : 0;
    k_lo[t] = a.window > 0 ? max(0, pos0 + tok - a.window + 1) : 0;
    const uint16_t* qp = a.q + (int64_t)(w.start + tok) * a.q_stride + (int64_t)hq * D;
#pragma unroll
    for (int n = 0; n < D / 32; ++n) {
      q[t][n] = *reinterpret_cast<const uint4*>(qp + 32 * n + 8 * g);
      if (!has) q[t][n] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  // of the wave's 32 rows: the keys that all see, and that any sees
  const int r_first = w.row0 + 32 * wave, r_last = min(r_first + 32, rows) - 1;
  const bool idle = r_first >= rows;
  const int all_hi = idle ? 0 : pos0 + r_first / G + 1;
  const int any_hi = idle ? 0 : pos0 + r_last / G + 1;
  const int all_lo = a.window > 0 && !idle ? max(0, pos0 + r_last / G - a.window + 1) : 0;
  const int any_lo = a.window > 0 && !idle ? max(0, pos0 + r_first / G - a.window + 1) : 0;

  // the keys that every row of the block sees
  const int block_hi = pos0 + w.tok0 + 1;
  const int block_lo = a.window > 0 ? max(0, pos0 + w.tok1 - a.window + 1) : 0;
  if (tid == 0) odd = 0;
  __syncthreads();

  const int n_it = (w.k1 - w.k0 + 63) >> 6;
  const int32_t* table = a.r.table + (int64_t)w.b * a.r.max_pages;
  // page ids of the 16-key groups of 16 tiles, one per lane, as in the other kernel
  auto load_ids = [&](int it) {
    const int key = w.k0 + 64 * it + 16 * lane;
    int id = -1;
    if (key < w.k1 && key + 16 > w.lo) {
      id = table[key >> a.kv.page_log2];
      if ((unsigned)id >= (unsigned)a.kv.n_pages) {
        id = -1;
        flag_dev_err(a.r.err, kDevErrPageId);
      }
    }
    return id;
  };
  const int page_mask = (1 << a.kv.page_log2) - 1;
  auto group_at = [&](int it, int ids, int grp) {  // rows of the group's first key
    const int id = max(__builtin_amdgcn_readlane(ids, 4 * (it & 15) + grp), 0);
    return (((int64_t)id * a.kv.Hkv + h) << a.kv.page_log2) +
           ((w.k0 + 64 * it + 16 * grp) & page_mask);
  };
  // bit grp: the tile's group has no page
  auto dead_groups = [&](int it, int ids) {
    uint32_t dead = 0;
#pragma unroll
    for (int grp = 0; grp < 4; ++grp)
      dead |= (uint32_t)(__builtin_amdgcn_readlane(ids, 4 * (it & 15) + grp) < 0) << grp;
    return dead;
  };
  // A tile's loads.  bf16: word tid % W of the keys tid / W + (256 / W) j.  MXFP4:
  // the codes of D/4 dims of key tid / 4 in [0], and the word with their scale in
  // [1].x (see PaTile).
  auto load_tile = [&](PmStage<D>& t, int it, int ids) {
    if constexpr (F4) {
      const int64_t at = group_at(it, ids, wave);
      const int kk = tid >> 2 & 15, part = tid & 3;
      const uint32_t sc = (uint32_t)(kk * (D / 32) & ~3), cd = (uint32_t)(kk * (D / 2) + (D / 8) * part);
      t.k[1].x = *reinterpret_cast<const uint32_t*>(a.kv.ks + at * (D / 32) + sc);
      t.v[1].x = *reinterpret_cast<const uint32_t*>(a.kv.vs + at * (D / 32) + sc);
      if constexpr (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(a.kv.k + at * (D / 2) + cd);
        const uint2 y = *reinterpret_cast<const uint2*>(a.kv.v + at * (D / 2) + cd);
        t.k[0].x = x.x; t.k[0].y = x.y;
        t.v[0].x = y.x; t.v[0].y = y.y;
      } else {
        t.k[0] = *reinterpret_cast<const uint4*>(a.kv.k + at * (D / 2) + cd);
        t.v[0] = *reinterpret_cast<const uint4*>(a.kv.v + at * (D / 2) + cd);
      }
    } else {
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const int key = tid / W + (256 / W) * j;  // its group is the wave's
        const int64_t at = group_at(it, ids, uni(key >> 4)) * (2 * D);
        const uint32_t off = (uint32_t)((key & 15) * 2 * D + 16 * (tid % W));
        t.k[j] = *reinterpret_cast<const uint4*>(a.kv.k + at + off);
        t.v[j] = *reinterpret_cast<const uint4*>(a.kv.v + at + off);
      }
    }
  };
  // whether some row of the block does not see all of the tile's keys
  auto at_edge = [&](int kb) { return kb < block_lo || kb + 64 > block_hi; };
  auto v_word = [&](int key, int word) {
    return key * W + (word ^ (D == 64 ? (key & 6) : (key & 7) << 1));
  };
  auto write_tile = [&](const PmStage<D>& t, int it, int ids) {
    const int buf = it & 1, kb = w.k0 + 64 * it;
    const bool edge = at_edge(kb);
    // (words one by one: a copy of the struct would put the stage in private memory)
    auto put = [&](int key, int word, const uint4& x, const uint4& y) {
      kt[buf][key * W + (word ^ (key & 7))] = make_uint4(x.x, x.y, x.z, x.w);
      uint32_t v[4] = {y.x, y.y, y.z, y.w};
      const bool dead = __builtin_amdgcn_readlane(ids, 4 * (it & 15) + uni(key >> 4)) < 0;
      if (edge || dead) {
        const bool none = (kb + key < w.lo) | (kb + key >= w.k1) | dead;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t m = pa_odd_halves(v[i]);
          any |= m;
          v[i] = none ? 0u : v[i] & ~m;
        }
        if (!none && any != 0) odd = 1;
      }
      vt[buf][v_word(key, word)] = make_uint4(v[0], v[1], v[2], v[3]);
    };
    if constexpr (F4) {
      const int key = tid >> 2, part = tid & 3;
      const int sh = D == 64 ? 16 * (key & 1) + 8 * (part >> 1) : 8 * part;
      const uint32_t kc[4] = {t.k[0].x, t.k[0].y, t.k[0].z, t.k[0].w};
      const uint32_t vc[4] = {t.v[0].x, t.v[0].y, t.v[0].z, t.v[0].w};
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        put(key, part * (D / 32) + j, mx4_to_bf16x8(kc[j], t.k[1].x >> sh),
            mx4_to_bf16x8(vc[j], t.v[1].x >> sh));
    } else {
#pragma unroll
      for (int j = 0; j < D / 32; ++j) put(tid / W + (256 / W) * j, tid % W, t.k[j], t.v[j]);
    }
  };

  pf4 o[2][E];
  float m[2], l[2];  // l: of the lane's keys
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int e = 0; e < E; ++e) o[t][e] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    l[t] = 0.0f;
    m[t] = -INFINITY;
  }
  auto compute = [&](int it, uint32_t dead) {
    const int kb = w.k0 + 64 * it, buf = it & 1;
    if (kb >= any_hi || kb + 64 <= any_lo) return;
    const bool full = kb >= all_lo && kb + 64 <= all_hi && dead == 0;
    pf4 s[2][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 kf[D / 32];
#pragma unroll
      for (int n = 0; n < D / 32; ++n) kf[n] = kt[buf][(16 * k + c) * W + ((4 * n + g) ^ (c & 7))];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t][k] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < D / 32; ++n) s[t][k] = pa_mfma(kf[n], q[t][n], s[t][k]);
      }
    }
    if (!full) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kb + 16 * k + 4 * g + i;
            const bool seen = (key >= k_lo[t]) & (key < k_hi[t]) & !(dead >> k & 1);
            s[t][k][i] = seen ? s[t][k][i] : -INFINITY;
          }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mx = fmaxf(mx, fmaxf(fmaxf(s[t][k][0], s[t][k][1]), fmaxf(s[t][k][2], s[t][k][3])));
      mx *= c2;
      if (__any(mx > m[t] + kPaLag)) {
        mx = fmaxf(mx, xor_lane<16>(mx));
        mx = fmaxf(mx, xor_lane<32>(mx));
        const float mn = fmaxf(m[t], mx);
        const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[t] - mn);
#pragma unroll
        for (int e = 0; e < E; ++e) o[t][e] *= f;
        l[t] *= f;
        m[t] = mn;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint4 ph[2], pl[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float me = m[t] == -INFINITY ? 0.0f : m[t];
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][2 * k + j][i], c2, -me));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][2 * k + j][i + 1], c2, -me));
            const uint32_t x = pack_bf2(p0, p1);
            l[t] += p0 + p1;
            hi[2 * j + i / 2] = x;
            lo[2 * j + i / 2] = pack_bf2(p0 - bf_lo(x), p1 - bf_hi(x));
          }
        ph[t] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        pl[t] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      // lane (g, c) reads dims 4 (c & 3) .. of key 4 g + c / 4 of each 16, for each
      // 16 dims, and gets dim c of the keys 4 g ..
      const int key = 32 * k + 4 * g + (c >> 2);  // (the second 16 exchange alike)
      const char* base = reinterpret_cast<const char*>(&vt[buf][0]) + 8 * (c & 1);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const char* p = base + 16 * v_word(key, 2 * e + (c >> 1 & 1));
        const uint2 x = pa_read_tr(p), y = pa_read_tr(p + 16 * 16 * W);
        const uint4 f = make_uint4(x.x, x.y, y.x, y.y);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          o[t][e] = pa_mfma(f, ph[t], o[t][e]);
          o[t][e] = pa_mfma(f, pl[t], o[t][e]);
        }
      }
    }
  };

  PmStage<D> st;
  int ids = load_ids(0);
  load_tile(st, 0, ids);
  for (int it = 0; it < n_it; ++it) {
    write_tile(st, it, ids);
    const uint32_t dead = dead_groups(it, ids);
    const int nx = min(it + 1, n_it - 1);
    if ((nx & 15) == 0 && nx > it) ids = load_ids(nx);
    load_tile(st, nx, ids);
    lds_barrier();  // the tile is written; the one before it was read before this
    compute(it, dead);
  }

  // lane (g, c): row c of each tile, dims 16 e + 4 g ..
  __syncthreads();
  // as in the other kernel: infinities and NaNs cleared at an edge, and infinities
  // that met both terms of P
  bool more = false;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    l[t] += xor_lane<16>(l[t]);
    l[t] += xor_lane<32>(l[t]);
    float z = 0.0f;  // NaN where an element is not finite
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) z = __builtin_fmaf(o[t][e][i], 0.0f, z);
    more = more || (z != z && l[t] == l[t]);
  }
  if (odd != 0 || __any(more)) {
    pf4 sum[2][E];  // of the infinities and NaNs alone
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < E; ++e) sum[t][e] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    pa_odd_values<D, F4>(a, w, h, w.k0, w.k1 - w.k0, [&](int key, auto value) {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = value(16 * e + 4 * g + i);
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (key >= k_lo[t] && key < k_hi[t]) sum[t][e][i] += v;
        }
    });
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][e][i] = sum[t][e][i] != 0.0f ? sum[t][e][i] : o[t][e][i];
  }
  if (w.chunks == 1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = r_first + 16 * t + c;
      if (r >= rows) continue;
      const int head = h * G + r % G;
      const float fin = pa_finish(a, head, m[t], l[t]);
      uint16_t* dst = a.out + ((int64_t)(w.start + r / G) * a.Hq + head) * D + 4 * g;
#pragma unroll
      for (int e = 0; e < E; ++e)
        *reinterpret_cast<uint2*>(dst + 16 * e) =
            make_uint2(pack_bf2(o[t][e][0] * fin, o[t][e][1] * fin),
                       pack_bf2(o[t][e][2] * fin, o[t][e][3] * fin));
    }
    return;
  }
  const int64_t first = (int64_t)w.slot * a.kv.Hkv + h;
  const int64_t step_c = (int64_t)a.kv.Hkv * R * (D + 2);
  float* p0 = a.part + first * R * (D + 2);
  float* po = p0 + w.c * step_c;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = 32 * wave + 16 * t + c;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      pa_store_agent(po + r * D + 16 * e + 4 * g, o[t][e][0], o[t][e][1]);
      pa_store_agent(po + r * D + 16 * e + 4 * g + 2, o[t][e][2], o[t][e][3]);
    }
    if (g == 0) pa_store_agent(po + R * D + 2 * r, m[t], l[t]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores have completed
  __syncthreads();
  int32_t* ctr = a.arrive + first * kPaArrive;
  if (tid == 0)
    merge_here = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 w.chunks - 1;
  __syncthreads();
  if (!merge_here) return;
  if (tid == 0) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // the tiles' memory is free: every wave is past its last one
  pm_join<D>(a, w, h, p0, step_c, reinterpret_cast<float (*)[kPmJoin]>(&kt[0][0]),
             reinterpret_cast<float*>(&vt[0][0]));
}

// Most keys that a row tile of R rows can see.
static int64_t pa_keys(const PagedAttnArgs& a, int R, int align) {
  const int64_t holds = (int64_t)a.r.max_pages << a.kv.page_log2, longest = 1 << 30;
  const int64_t keys = holds < longest ? holds : longest;
  const int64_t seen = (int64_t)a.window + (R - 1) / a.G + align;
  return a.window > 0 && seen < keys ? seen : keys;
}
// Blocks for `units` units per KV head: target / Hkv of equal work and one more per
// unit, or as many chunks of at least minc keys as the longest sequence that the
// table holds can have.  Blocks without work are not free: a launch of 17000 of
// them before a prompt chunk's took 14 us.
static int64_t pa_blocks(const PagedAttnArgs& a, int64_t units, int64_t keys, int minc, int target) {
  const int64_t even = target / a.kv.Hkv + 1 + units, all = units * ((keys + minc - 1) / minc);
  return (even < all ? even : all) * a.kv.Hkv;
}
struct PaGrid {
  int64_t few, many;  // blocks of the two launches (0: no row can be of that kind)
  bool small;         // the few-row one has room for all rows of a small call
};
// One row per sequence has G rows; with row starts the host does not know, and
// launches both unless all rows together are few, or surely a small call.  Units are
// at most one per R rows and one per sequence; of up to kPaFew rows two a sequence.
static PaGrid pa_grid(const PagedAttnArgs& a) {
  const int64_t rows = (int64_t)a.r.n_rows * a.G;
  const bool none_few = a.r.q_start == nullptr && a.G > kPaFew;
  const bool all_few = a.r.q_start == nullptr ? a.G <= kPaFew : rows <= kPaFew;
  const int64_t units = rows / 16 + a.r.B, two = a.r.B * (int64_t)(kPaFew / 16);
  const int64_t keys = pa_keys(a, 16, 32);
  PaGrid g;
  g.few = none_few ? 0 : pa_blocks(a, units < two ? units : two, keys, 256, kPaTarget);
  if (all_few) return g.many = 0, g.small = false, g;
  const int64_t longer = rows / (kPaFew + 1) + 1;  // sequences of more rows than kPaFew
  g.many = pa_blocks(a, rows / 128 + (longer < a.r.B ? longer : a.r.B), pa_keys(a, 128, 64), 256,
                     kPmTarget);
  // of a small call, sum of tiles x keys / 256 and one more per unit
  const int64_t small = units * a.kv.Hkv + kPaSmall / 256 + 2;
  g.small = small <= (g.few > 2048 ? g.few : 2048);
  if (g.small && g.few < small) g.few = small;
  if (g.small && units * a.kv.Hkv * keys <= kPaSmall) g.many = 0;
  return g;
}

bool paged_attn_fits(int n_rows, int B, int Hq, int Hkv) {
  PagedAttnArgs a{};
  static const int32_t given = 0;
  a.r.q_start = &given;
  a.r.n_rows = n_rows;
  a.r.B = B;
  a.r.max_pages = 1 << 30;
  a.kv.Hkv = Hkv;
  a.G = Hq / Hkv;
  const PaGrid g = pa_grid(a);
  return g.few < kPaMaxBlocks && g.many < kPaMaxBlocks;
}
// The two launches use the same places, one after the other.
size_t paged_attn_workspace(int n_rows, int Hq, int Hkv, int D) {
  const size_t few = (size_t)(2 * kPaTarget) * 16, many = (size_t)(2 * kPmTarget) * 128;
  return ((int64_t)n_rows * (Hq / Hkv) <= kPaFew ? few : many) * (D + 2) * 4;
}
size_t paged_attn_counters() { return (size_t)(2 * kPaTarget) * kPaArrive * 4; }

void launch_paged_attn(PagedAttnArgs a, hipStream_t st) {
  a.G = a.Hq / a.kv.Hkv;
  const PaGrid g = pa_grid(a);
  a.small = g.small;
#define PA(D, F4)                                                                              \
  do {                                                                                         \
    if (g.few)                                                                                   \
      hipLaunchKernelGGL((k_paged_attn_few<D, F4>), dim3((unsigned)g.few), dim3(256), 0, st, a); \
    if (g.many)                                                                                  \
      hipLaunchKernelGGL((k_paged_attn_many<D, F4>), dim3((unsigned)g.many), dim3(256), 0, st, a); \
  } while (0)
  if (a.kv.D == 64) {
    if (a.kv.ks != nullptr) PA(64, true); else PA(64, false);
  } else {
    if (a.kv.ks != nullptr) PA(128, true); else PA(128, false);
  }
#undef PA
}

}  // namespace neon
