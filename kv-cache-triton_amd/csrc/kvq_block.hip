// Attention of a block of query rows over the INT4 cache on the matrix cores
// (gfx950): the kernel behind tree attention and the key weights of decode
// tokens, for 16-bit queries and scales, D 64 and 128, aligned rows.
//
// The query rows of one KV head (positions x the GQA group's heads) are taken
// in chunks of 16 RB. A workgroup owns a chunk and a split of the keys; its
// waves take 64-key tiles in turn, each wave all 16 RB rows, so that a tile's
// codes are decoded once for all of them and nothing is shared between waves
// until the end. Operands never pass through LDS (only the scales, to reach
// the lanes that need them):
//
//   S^T = K Q^T  v_mfma 16x16x32, A = 16 keys x 32 dims of codes. A lane loads
//     its key's 16-byte piece; two rounds of lane swaps (v_permlane32_swap,
//     v_permlane16_swap) give it its four bytes of each 32-dim chunk. A nibble
//     n becomes the 16-bit float 16 + n by a shift and an and-or; the -24 per
//     element that makes it the code n - 8 is in the accumulator's start,
//     -24 sum(q) of the chunk. Codes and queries are exact, so a score has
//     fp32's error only; the chunk's scale multiplies after the product.
//   O^T += V^T P^T  A = 16 dims x 32 keys. Lane i holds the dims (D / 16) i ..
//     of its keys, so its nibble nb gives the matrix of the dims (D / 16) i +
//     nb; codes become fp16 (1024 + n, - 1032, exact) and are multiplied by
//     the key's scale there. Softmax weights are the B operand as they are:
//     the lane that scored a key weighs it.
//
// Layout of the 16x16x32 instruction (lane l: n = l % 16, g = l / 16): A[i][k]
// at lane (i, k / 8), register k % 8; B[k][n] at lane (n, k / 8); C[i][n] at
// lane (n, i / 4), register i % 4. Row i of a 16-key block is key i / 4 +
// 4 (i % 4), so that a value load reads whole rows: lane (n, g) holds, of query
// row n, keys 16 kb + g + 4 j in register j of block kb.
//
// Measured (graph replays): one decode token of 32 heads over 8 KV heads and 16K
// keys with its scores kept 14.3 us and 6.6 for the finish, 0.95 TB/s; eight
// sequences of 32K keys of the 70B shape 102 us, 3.1 TB/s of cache and sums and
// 4.4 with the scores; 64 rows over 16K keys 26 us. Few rows are bound by the
// latency of a workgroup's chain and the merge after it, more by the codes'
// decoding, which 16 or 32 rows share (64 did not fit the registers).
//
// Value scales reach fp16 times a power of two that puts the wave's first
// tile's largest near 1. Keys with a scale that fp16 then does not hold exactly
// (infinite, NaN, over 2^12 or under 2^-14) are left out of the products there,
// and added one at a time to the rows that weigh them, in fp32: so a row that
// does not attend a key never meets its infinity as 0 * inf.

#include <algorithm>

#include "kvq_block_mfma.h"

namespace kvq {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;
constexpr float kNeg = -1.0e30f;
constexpr float kLazyMax = 8.0f;  // slack of the running max, log2 units

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ f32x4_t mfma_f16(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma_bf16(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f32x4_t mfma_q(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (F16) return mfma_f16(a, b, c);
  else return mfma_bf16(a, b, c);
}

__device__ __forceinline__ void swap32(uint32_t& x, uint32_t& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  x = r0;
  y = r1;
}
__device__ __forceinline__ void swap16(uint32_t& x, uint32_t& y) {
  const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  x = r0;
  y = r1;
}
// Over the four lanes of a query row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float row_max(float v) {
  uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
  swap32(x, y);
  v = fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
  x = __builtin_bit_cast(uint32_t, v), y = x;
  swap16(x, y);
  return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float row_sum(float v) {
  uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
  swap32(x, y);
  v = __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
  x = __builtin_bit_cast(uint32_t, v), y = x;
  swap16(x, y);
  return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// The power of two that takes a value scale `top` into [1, 2), between 2^-100
// and 2^20 (a wave whose scales are smaller still takes its keys one at a
// time; a larger factor could overflow a larger scale that follows).
__device__ __forceinline__ float value_unit(float top) {
  if (!(top > 0.0f)) return 1.0f;
  const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
  const int u = -e < -100 ? -100 : (-e > 20 ? 20 : -e);
  return __builtin_bit_cast(float, (uint32_t)(u + 127) << 23);
}
// Whether fp16 does not hold a value scale, and its products with a code, exactly.
__device__ __forceinline__ bool value_scale_odd(float s) {
  return !(fabsf(s) <= 0x1p12f) || (s != 0.0f && fabsf(s) < 0x1p-14f);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const f16x2_t h = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, h);
}
// (x & m) | o in one instruction: with constants in plain sight the compiler
// writes two, each with its literal.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t d;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(d) : "v"(x), "s"(m), "v"(o));
  return d;
}

// The eight nibbles of w as 16-bit floats 16 + n: pair p is (nibble p, nibble
// p + 4). The queries are put in the same order.
template <bool F16>
__device__ __forceinline__ uint4 unpack_keys(uint32_t w) {
  if constexpr (F16) {
    constexpr uint32_t m = 0x03c003c0u, o = 0x4c004c00u;
    return make_uint4(and_or(w << 6, m, o), and_or(w << 2, m, o), and_or(w >> 2, m, o), and_or(w >> 6, m, o));
  } else {
    constexpr uint32_t m = 0x00780078u, o = 0x41804180u;
    return make_uint4(and_or(w << 3, m, o), and_or(w >> 1, m, o), and_or(w >> 5, m, o), and_or(w >> 9, m, o));
  }
}
__device__ __forceinline__ uint4 pair_queries(uint4 x) {  // dims (0, 4), (1, 5), (2, 6), (3, 7)
  return make_uint4(__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                    __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u));
}

// A pair of codes (4-bit fields `shift` of y's halves) as fp16 n - 8, times a
// pair of scales.
__device__ __forceinline__ uint32_t value_pair(uint32_t y, int shift, uint32_t scales) {
  const uint32_t x = and_or(y >> shift, 0x000f000fu, 0x64006400u);
  const f16x2_t off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
  const f16x2_t v = (__builtin_bit_cast(f16x2_t, x) + off) * __builtin_bit_cast(f16x2_t, scales);
  return __builtin_bit_cast(uint32_t, v);
}

template <int D, bool QF16, int RB, int NW, bool PAGED, bool SCORES>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
void block_attn_kernel(const BlockMfmaArgs a) {
  constexpr int NC = D / 32;    // 32-dim chunks
  constexpr int VN = D / 16;    // 16-dim blocks of O^T; dims a lane holds of a value row
  constexpr int ROWS = 16 * RB;
  constexpr int NT = 64 * NW;
  constexpr int OP = D + 4;     // row pitch of the epilogue's buffer
  constexpr int SC_BYTES = NC * kKeys * 6;  // a wave's key scales (fp32) and value scales (fp16)
  constexpr int O_BYTES = NW * 16 * OP * 4;
  constexpr int LDS = NW * SC_BYTES > O_BYTES ? NW * SC_BYTES : O_BYTES;
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ float2 ml_lds[NW][ROWS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  // workgroup -> (unit fastest: the chunks and splits of a KV head land on one
  // XCD where the units are a multiple of 8, and share its L2)
  int wg = blockIdx.x;
  const int unit = wg % a.n_units;
  wg /= a.n_units;
  const int chunk = wg % a.row_chunks, sp = wg / a.row_chunks;
  const int kvh = unit % a.b.Hkv, b = unit / a.b.Hkv;
  const int len = (int)block_len(a.b, b), base = len - a.b.T;
  const int rows = a.b.ratio * a.b.T;
  const int tiles = (len + kKeys - 1) / kKeys;
  const int tile_lo = (int)((int64_t)tiles * sp / a.n_split), tile_hi = (int)((int64_t)tiles * (sp + 1) / a.n_split);

  const uint8_t* kp = a.b.kp + b * a.b.kps_b + kvh * a.b.kps_h;
  const uint8_t* vp = a.b.vp + b * a.b.vps_b + kvh * a.b.vps_h;
  const uint16_t* ks = (const uint16_t*)a.b.ks + b * a.b.kss_b + kvh * a.b.kss_h;
  const uint16_t* vs = (const uint16_t*)a.b.vs + b * a.b.vss_b + kvh * a.b.vss_h;
  constexpr uint32_t KV_ROW = D / 2;  // bytes of a row's codes (rows are dense: constant load offsets)
  const uint32_t srow = 2u * (uint32_t)a.ng;  // bytes of a row's scales
  const int32_t* bt = PAGED ? a.b.pm.table + (int64_t)b * a.b.pm.tab_stride : nullptr;

  // first cache row of tile t, or -1 (past the split, or on a page without a block)
  auto block_of = [&](int t) -> int32_t {
    if (t >= tile_hi) return -1;
    const int64_t pg = (int64_t)t * kKeys >> a.b.pm.page_shift;
    return pg < a.b.pm.n_pages ? bt[pg] : -1;
  };
  auto row_of = [&](int t, int32_t blk) -> int64_t {
    if constexpr (!PAGED) return t < tile_hi ? (int64_t)t * kKeys : -1;
    if (t >= tile_hi || blk < 0 || blk >= a.b.pm.n_blocks) return -1;
    return ((int64_t)blk << a.b.pm.page_shift) | ((int64_t)t * kKeys & ((int64_t(1) << a.b.pm.page_shift) - 1));
  };

  uint4 kraw[4];            // lane (n, g): piece g (D / 8 bytes) of key row 16 kb + n / 4 + 4 (n % 4)
  uint32_t vraw[2][8];      // lane (n, g): its dims of key rows 32 h + 16 (e / 4) + g + 4 (e % 4)
  uint2 ksr, vsr;           // lane l: the scale rows of key l
  auto load_scales = [&](int64_t r0, uint32_t lim) {
    const __amdgpu_buffer_rsrc_t rk = rsrc_of((const uint8_t*)ks + r0 * srow, lim * srow);
    const __amdgpu_buffer_rsrc_t rv = rsrc_of((const uint8_t*)vs + r0 * srow, lim * srow);
    ksr = make_uint2(0u, 0u);
    vsr = make_uint2(0u, 0u);
    if (a.ng == 4) {
      ksr = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rk, 8 * lane, 0, 0));
      vsr = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rv, 8 * lane, 0, 0));
    } else if (a.ng == 2) {
      ksr.x = __builtin_amdgcn_raw_buffer_load_b32(rk, 4 * lane, 0, 0);
      vsr.x = __builtin_amdgcn_raw_buffer_load_b32(rv, 4 * lane, 0, 0);
    } else {
      ksr.x = __builtin_amdgcn_raw_buffer_load_b16(rk, 2 * lane, 0, 0);
      vsr.x = __builtin_amdgcn_raw_buffer_load_b16(rv, 2 * lane, 0, 0);
    }
  };
  const uint32_t k_at = ((n >> 2) + 4 * (n & 3)) * KV_ROW + (D / 8) * g;
  auto load_keys = [&](int64_t r0, uint32_t lim) {
    const __amdgpu_buffer_rsrc_t rk = rsrc_of(kp + r0 * KV_ROW, lim * KV_ROW);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      if constexpr (D == 128) {
        kraw[kb] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_at + 16 * kb * KV_ROW, 0, 0));
      } else {
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rk, k_at + 16 * kb * KV_ROW, 0, 0));
        kraw[kb] = make_uint4(x.x, x.y, 0u, 0u);
      }
    }
  };
  const uint32_t v_at = g * KV_ROW + (D == 128 ? 4u * n : 4u * (n >> 1));
  auto load_values = [&](int64_t r0, uint32_t lim, int h) {
    const __amdgpu_buffer_rsrc_t rv = rsrc_of(vp + r0 * KV_ROW, lim * KV_ROW);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vraw[h][e] = __builtin_amdgcn_raw_buffer_load_b32(rv, v_at + (32 * h + 16 * (e >> 2) + 4 * (e & 3)) * KV_ROW, 0, 0);
  };

  // the first tile's loads, then the queries (which the loop waits for first)
  int t = tile_lo + wave;
  int32_t blk = 0, blk_next = 0;
  if constexpr (PAGED) {
    blk = __builtin_amdgcn_readfirstlane(block_of(t));
    blk_next = block_of(t + NW);
  }
  int64_t r0 = row_of(t, blk);
  uint32_t lim = r0 < 0 ? 0u : (uint32_t)min(kKeys, len - t * kKeys);

  // queries as the B operand: lane (n, g) holds dims 32 c + 8 g .. + 7 of row n
  // in unpack_keys' order; the sign of sm_scale goes into them, and scores
  // reach the softmax times c = |sm_scale| log2(e) > 0
  const float c = fmaxf(fabsf(a.b.scale_log2), 1.0e-30f);
  const uint32_t qneg = a.b.scale_log2 < 0.0f ? 0x80008000u : 0u;
  uint4 q[RB][NC];
  int row_i[RB];  // block row of this lane's query row (-1: none)
  bool careful = false;  // a query or a key scale of the tile is not finite
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int R = chunk * ROWS + 16 * r + n;
    const int i = R / a.b.ratio, h = kvh * a.b.ratio + R % a.b.ratio;
    row_i[r] = R < rows ? i : -1;
    const uint16_t* qr = (const uint16_t*)a.b.q + b * a.b.qs_b + (int64_t)h * a.b.qs_h + (int64_t)(R < rows ? i : 0) * a.b.qs_s;
    if (R >= rows) qr = (const uint16_t*)a.b.q + b * a.b.qs_b + (int64_t)(kvh * a.b.ratio) * a.b.qs_h;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      const uint16_t* p = qr + 32 * cc + 8 * g;
      if (a.q_vec) {
        x = *(const uint4*)p;
      } else {
        x = make_uint4((uint32_t)p[0] | ((uint32_t)p[1] << 16), (uint32_t)p[2] | ((uint32_t)p[3] << 16),
                       (uint32_t)p[4] | ((uint32_t)p[5] << 16), (uint32_t)p[6] | ((uint32_t)p[7] << 16));
      }
      const uint32_t keep = R < rows ? 0xffffffffu : 0u;
      x = make_uint4((x.x & keep) ^ qneg, (x.y & keep) ^ qneg, (x.z & keep) ^ qneg, (x.w & keep) ^ qneg);
      const uint32_t top = QF16 ? 0x7c00u : 0x7f80u;
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) careful = careful || (w[k] & top) == top || ((w[k] >> 16) & top) == top;
      q[r][cc] = pair_queries(x);
    }
  }
  const bool q_careful = __builtin_amdgcn_ballot_w64(careful) != 0;
  load_scales(r0 < 0 ? 0 : r0, lim);
  load_keys(r0 < 0 ? 0 : r0, lim);
  load_values(r0 < 0 ? 0 : r0, lim, 0);
  load_values(r0 < 0 ? 0 : r0, lim, 1);

  // -24 sum(q) of each chunk, where the products start: A = a matrix of -24
  float bias[RB][NC];
  {
    const uint32_t m24 = QF16 ? 0xce00ce00u : 0xc1c0c1c0u;
    const uint4 am = make_uint4(m24, m24, m24, m24);
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) bias[r][cc] = mfma_q<QF16>(am, q[r][cc], f32x4_t{0.0f, 0.0f, 0.0f, 0.0f})[0];
  }

  f32x4_t o[RB][VN];
  float m_run[RB], l_run[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int nb = 0; nb < VN; ++nb) o[r][nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    m_run[r] = kNeg;
    l_run[r] = 0.0f;
  }

  float* ksc = (float*)(lds + wave * SC_BYTES);               // [NC][64], a key at 16 kb + 4 (i % 4) + i / 4
  _Float16* vsc = (_Float16*)(lds + wave * SC_BYTES + NC * kKeys * 4);
  const int my_pos = (lane & 48) | ((lane & 3) << 2) | ((lane >> 2) & 3);
  float v_unit = 0.0f;  // the power of two on the value scales (0: not known yet)
  auto scale_of = [&](uint64_t row, int cc) {
    const uint32_t x = (uint32_t)(row >> (16 * ((cc * a.ng) / NC))) & 0xffffu;
    return a.s_f16 ? f16_bits_to_f32(x) : bf16_bits_to_f32(x);
  };
  const int v_chunk = (VN * n) / 32;  // the 32-dim chunk of this lane's value dims

  for (; t < tile_hi; t += NW) {
    const int t0 = t * kKeys;
    const bool has = lim > 0;  // (a tile whose page has no block is passed over)
    // ---- scales to the lanes that use them ----
    const uint64_t kb64 = ((uint64_t)ksr.y << 32) | ksr.x, vb64 = ((uint64_t)vsr.y << 32) | vsr.x;
    float vf[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) vf[cc] = scale_of(vb64, cc);
    if (v_unit == 0.0f) {  // the wave's first tile
      float top = 0.0f;
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) top = fmaxf(top, fabsf(vf[cc]) < __builtin_inff() ? fabsf(vf[cc]) : 0.0f);
      v_unit = value_unit(wave_max(top));
    }
    bool k_bad = false, v_bad = false;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      const float kf = scale_of(kb64, cc);
      k_bad = k_bad || !(fabsf(kf) < __builtin_inff());
      const float vu = vf[cc] * v_unit;
      const bool odd = value_scale_odd(vu);
      v_bad = v_bad || odd;
      ksc[cc * kKeys + my_pos] = kf;
      vsc[cc * kKeys + my_pos] = (_Float16)(odd ? 0.0f : vu);
    }
    const bool fix = __builtin_amdgcn_ballot_w64(k_bad) != 0 || q_careful;
    const uint64_t bad_keys = __builtin_amdgcn_ballot_w64(v_bad);
    // ---- the next tile of this wave (none: no rows, no traffic) ----
    const int64_t r0_now = r0;
    if constexpr (PAGED) {
      blk = __builtin_amdgcn_readfirstlane(blk_next);
      blk_next = block_of(t + 2 * NW);
    }
    r0 = row_of(t + NW, blk);
    lim = r0 < 0 ? 0u : (uint32_t)min(kKeys, len - (t + NW) * kKeys);
    if (r0 < 0) r0 = 0;
    load_scales(r0, lim);

    // ---- scores: register j of block kb is key 16 kb + g + 4 j ----
    f32x4_t s[RB][4];
    uint32_t w[4][4];  // [kb][chunk]: this lane's four bytes of the chunk
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      w[kb][0] = kraw[kb].x; w[kb][1] = kraw[kb].y; w[kb][2] = kraw[kb].z; w[kb][3] = kraw[kb].w;
      if constexpr (D == 128) {
        swap32(w[kb][0], w[kb][2]);
        swap32(w[kb][1], w[kb][3]);
        swap16(w[kb][0], w[kb][1]);
        swap16(w[kb][2], w[kb][3]);
      } else {
        swap16(w[kb][0], w[kb][1]);
        swap32(w[kb][0], w[kb][1]);
      }
    }
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      f32x4_t start[RB];
#pragma unroll
      for (int r = 0; r < RB; ++r) start[r] = f32x4_t{bias[r][cc], bias[r][cc], bias[r][cc], bias[r][cc]};
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const uint4 ka = unpack_keys<QF16>(w[kb][cc]);
        const float4 sc = *(const float4*)(ksc + cc * kKeys + 16 * kb + 4 * g);
        const float scj[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const f32x4_t x = mfma_q<QF16>(ka, q[r][cc], start[r]);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[r][kb][j] = cc == 0 ? x[j] * scj[j] : __builtin_fmaf(x[j], scj[j], s[r][kb][j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (one chunk's operands at a time: registers)
    }
    load_keys(r0, lim);
    __builtin_amdgcn_sched_barrier(0);

    // ---- masks: only tiles with keys that some row does not attend ----
    if (fix) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[r][kb][j] = block_score(s[r][kb][j]);
    }
    if (!has || t0 + kKeys > (a.b.kind == kMaskNone ? len : base)) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        uint32_t seen = 0u;
#pragma unroll 1
        for (int x = 0; x < 16; ++x) {
          const int key = t0 + 16 * (x >> 2) + g + 4 * (x & 3);
          const int at = key - base;
          bool on = has && row_i[r] >= 0 && key < len;
          if (on && a.b.kind != kMaskNone && at >= 0) on = block_sees(a.b, b, row_i[r], at);
          seen |= on ? 1u << x : 0u;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (!((seen >> x) & 1u)) s[r][x >> 2][x & 3] = -__builtin_inff();
      }
    }
    if constexpr (SCORES) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float* dst = a.scores + (((int64_t)unit * a.tiles_max + t) * rows + chunk * ROWS + 16 * r + n) * kKeys;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[r][kb][j] *= c;
          if (row_i[r] >= 0)
            *(float4*)(dst + 16 * kb + 4 * g) = make_float4(s[r][kb][0], s[r][kb][1], s[r][kb][2], s[r][kb][3]);
        }
      }
    }

    // ---- online softmax, base 2, with a lazy running max ----
    float mt[RB];
    bool grow = false;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float mx = s[r][0][0];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[r][kb][j]);
      mt[r] = SCORES ? row_max(mx) : row_max(mx) * c;
      grow = grow || mt[r] > m_run[r] + kLazyMax;
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float m_new = fmaxf(m_run[r], mt[r]);
        const float alpha = __builtin_amdgcn_exp2f(m_run[r] - m_new);
        m_run[r] = m_new;
        l_run[r] *= alpha;
#pragma unroll
        for (int nb = 0; nb < VN; ++nb) o[r][nb] *= alpha;
      }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = SCORES ? s[r][kb][j] - m_run[r] : __builtin_fmaf(s[r][kb][j], c, -m_run[r]);
          s[r][kb][j] = __builtin_amdgcn_exp2f(x);
          l_run[r] += s[r][kb][j];
        }

    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t scp[4];  // scales of the pairs of keys
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint2 v = *(const uint2*)(vsc + v_chunk * kKeys + 16 * (2 * h + x) + 4 * g);
        scp[2 * x] = v.x;
        scp[2 * x + 1] = v.y;
      }
      uint4 pb[RB];
#pragma unroll
      for (int r = 0; r < RB; ++r)
        pb[r] = make_uint4(pack_f16(s[r][2 * h][0], s[r][2 * h][1]), pack_f16(s[r][2 * h][2], s[r][2 * h][3]),
                           pack_f16(s[r][2 * h + 1][0], s[r][2 * h + 1][1]),
                           pack_f16(s[r][2 * h + 1][2], s[r][2 * h + 1][3]));
#pragma unroll
      for (int half = 0; half < D / 64; ++half) {
        __builtin_amdgcn_sched_barrier(0);
        uint32_t y[4];  // the pairs' 16 bits of codes
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t sel = D == 128 ? (half ? 0x07060302u : 0x05040100u) : ((n & 1) ? 0x07060302u : 0x05040100u);
          y[p] = __builtin_amdgcn_perm(vraw[h][2 * p + 1], vraw[h][2 * p], sel);
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint4 va = make_uint4(value_pair(y[0], 4 * d, scp[0]), value_pair(y[1], 4 * d, scp[1]),
                                      value_pair(y[2], 4 * d, scp[2]), value_pair(y[3], 4 * d, scp[3]));
#pragma unroll
          for (int r = 0; r < RB; ++r) o[r][4 * half + d] = mfma_f16(va, pb[r], o[r][4 * half + d]);
        }
      }
      load_values(r0, lim, h);
    }
    // keys with an odd value scale: one at a time, to the rows that weigh them.
    // Lane (n, g) holds dims VN (4 g + j) + nb of row n, all in one chunk; the
    // key's weight is on lane n + 16 (key % 4), register (key % 16) / 4 of
    // block key / 16.
    if (bad_keys != 0) {
      uint64_t left = bad_keys;
#pragma unroll 1
      while (left != 0) {
        const int key = __builtin_ctzll(left);
        left &= left - 1;
        const uint32_t* vrow = (const uint32_t*)(vp + (r0_now + key) * KV_ROW + 2 * VN * g);
        const uint32_t sw = vs[(r0_now + key) * a.ng + (VN * g / 8 * a.ng) / NC];
        const float sf = (a.s_f16 ? f16_bits_to_f32(sw) : bf16_bits_to_f32(sw)) * v_unit;
        const bool nf = value_scale_odd(sf);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          float p = 0.0f;
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (x == 4 * (key >> 4) + ((key & 15) >> 2)) p = s[r][x >> 2][x & 3];
          p = __shfl(p, n + 16 * (key & 3));
          if (p > 0.0f && nf) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int nb = 0; nb < VN; ++nb) {
                const int e = VN * j + nb;  // of the lane's 4 VN dims
                o[r][nb][j] = fmaf(p, (float)((int)((vrow[e / 8] >> (4 * (e % 8))) & 15u) - 8) * sf, o[r][nb][j]);
              }
          }
        }
      }
    }
  }

  // ---- the waves' partials to one: max and sum, then rows scaled and added ----
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    l_run[r] = row_sum(l_run[r]);
    if (g == 0) ml_lds[wave][16 * r + n] = make_float2(m_run[r], l_run[r]);
  }
  __syncthreads();  // (also: every wave is done with its scales)
  float* obuf = (float*)lds;  // [wave][16][OP]
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    float M = kNeg;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml_lds[w][16 * r + n].x);
    // (v_unit is 0 for a wave without tiles, whose values are 0)
    const float f = v_unit == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m_run[r] - M) / v_unit;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int x = 0; x < VN / 4; ++x)
        *(float4*)(obuf + (wave * 16 + n) * OP + VN * (4 * g + j) + 4 * x) =
            make_float4(o[r][4 * x][j] * f, o[r][4 * x + 1][j] * f, o[r][4 * x + 2][j] * f, o[r][4 * x + 3][j] * f);
    __syncthreads();
    for (int x = tid; x < 16 * (D / 4); x += NT) {
      const int row = x / (D / 4), d = 4 * (x % (D / 4));
      float Mr = kNeg, L = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) Mr = fmaxf(Mr, ml_lds[w][16 * r + row].x);
#pragma unroll
      for (int w = 0; w < NW; ++w)
        L = fmaf(ml_lds[w][16 * r + row].y, __builtin_amdgcn_exp2f(ml_lds[w][16 * r + row].x - Mr), L);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float4 v = *(const float4*)(obuf + (w * 16 + row) * OP + d);
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      }
      const int R = chunk * ROWS + 16 * r + row;
      if (R >= rows) continue;
      const int64_t slot = ((int64_t)unit * rows + R) * a.n_split + sp;
      if ((SCORES || a.n_split > 1) && d == 0) a.ws_ml[slot] = make_float2(Mr, L);
      if (a.n_split > 1) *(float4*)(a.ws_o + slot * D + d) = acc;
      else block_store_row<QF16>(a, b, kvh, R, d, Mr, L, acc);
    }
    if (r + 1 < RB) __syncthreads();
  }
}

// Combines the splits' partials of row `row` (log-sum-exp in base 2) in dims
// d .. d + 3 and stores them. Memory-bound: it reads every partial once.
template <int D, bool QF16>
__device__ __forceinline__ void merge_row(const BlockMfmaArgs& a, int64_t row, int rows, int d) {
  const int unit = (int)(row / rows), R = (int)(row % rows);
  const int64_t slot = row * a.n_split;
  float M = kNeg, L = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = 0; s0 < a.n_split; s0 += 8) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t x = slot + min(s0 + j, a.n_split - 1);
      ml[j] = a.ws_ml[x];
      v[j] = *(const float4*)(a.ws_o + x * D + d);
    }
    float mb = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) mb = fmaxf(mb, ml[j].x);
    const float al = __builtin_amdgcn_exp2f(M - mb);
    M = mb;
    L *= al;
    acc.x *= al; acc.y *= al; acc.z *= al; acc.w *= al;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = s0 + j < a.n_split ? __builtin_amdgcn_exp2f(ml[j].x - mb) : 0.0f;
      L = fmaf(ml[j].y, w, L);
      acc.x = fmaf(v[j].x, w, acc.x);
      acc.y = fmaf(v[j].y, w, acc.y);
      acc.z = fmaf(v[j].z, w, acc.z);
      acc.w = fmaf(v[j].w, w, acc.w);
    }
  }
  block_store_row<QF16>(a, unit / a.b.Hkv, unit % a.b.Hkv, R, d, M, L, acc);
}

template <int D, bool QF16>
__global__ __launch_bounds__(256) void block_merge_kernel(const BlockMfmaArgs a) {
  const int rows = a.b.ratio * a.b.T;
  const int64_t row = (int64_t)blockIdx.x * (1024 / D) + threadIdx.x / (D / 4);
  if (row < (int64_t)a.n_units * rows) merge_row<D, QF16>(a, row, rows, 4 * (threadIdx.x % (D / 4)));
}

// After a launch that kept its scores: each key's weights from them and the
// rows' statistics, and (in workgroups of their own) the splits' merge. A
// thread owns one key; scores are read in their storage order. Memory-bound:
// rows * 4 bytes a key, and the running sum once.
constexpr int kFinishKeys = 256;

template <int D, bool QF16>
__global__ __launch_bounds__(256) void block_finish_kernel(const BlockMfmaArgs a, int key_wgs) {
  __shared__ float2 st[kMaxScoreRows];
  const int rows = a.b.ratio * a.b.T;
  if ((int)blockIdx.x >= key_wgs) {
    const int64_t row = (int64_t)(blockIdx.x - key_wgs) * (1024 / D) + threadIdx.x / (D / 4);
    if (row < (int64_t)a.n_units * rows) merge_row<D, QF16>(a, row, rows, 4 * (threadIdx.x % (D / 4)));
    return;
  }
  const int unit = blockIdx.x % a.n_units, tile0 = (blockIdx.x / a.n_units) * (kFinishKeys / kKeys);
  const int kvh = unit % a.b.Hkv, b = unit / a.b.Hkv;
  const int len = (int)block_len(a.b, b);
  if (tile0 * kKeys >= len) return;
  if ((int)threadIdx.x < rows) {
    const float2* ml = a.ws_ml + ((int64_t)unit * rows + threadIdx.x) * a.n_split;
    float M = kNeg, L = 0.0f;
    for (int s = 0; s < a.n_split; ++s) M = fmaxf(M, ml[s].x);
    for (int s = 0; s < a.n_split; ++s) L = fmaf(ml[s].y, __builtin_amdgcn_exp2f(ml[s].x - M), L);
    st[threadIdx.x] = make_float2(M, L > 0.0f ? 1.0f / L : 0.0f);
  }
  __syncthreads();
  const int tile = tile0 + threadIdx.x / kKeys, pos = threadIdx.x % kKeys;
  const int key = tile * kKeys + (pos & 48) + ((pos >> 2) & 3) + 4 * (pos & 3);
  if (tile * kKeys >= len) return;
  const float* sc = a.scores + ((int64_t)unit * a.tiles_max + tile) * rows * kKeys + pos;
  float* w = a.weights + b * a.w_b + kvh * a.w_h + key * a.w_k;
  const bool on = key < len;
  const float before = on ? *w : 0.0f;
  float sum = 0.0f;
  for (int r0 = 0; r0 < rows; r0 += 8) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = sc[min(r0 + k, rows - 1) * kKeys];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (r0 + k < rows) sum = fmaf(__builtin_amdgcn_exp2f(x[k] - st[r0 + k].x), st[r0 + k].y, sum);
  }
  if (on) *w = before + sum;
}

template <int D, bool QF16>
void launch_merge(const BlockMfmaArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.n_units * a.b.ratio * a.b.T;
  hipLaunchKernelGGL((block_merge_kernel<D, QF16>), dim3((unsigned)((rows + 1024 / D - 1) / (1024 / D))), dim3(256), 0, st, a);
}

template <int D, bool QF16, int RB, int NW, bool SCORES>
void launch_block(const BlockMfmaArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.n_units * a.row_chunks * a.n_split)), block(64 * NW);
  if (a.b.pm.paged) {
    if constexpr (!SCORES) hipLaunchKernelGGL((block_attn_kernel<D, QF16, RB, NW, true, false>), grid, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((block_attn_kernel<D, QF16, RB, NW, false, SCORES>), grid, block, 0, st, a);
  }
  if (a.n_split > 1 && !SCORES) launch_merge<D, QF16>(a, st);
}

template <int D, bool QF16>
void launch_rb(const BlockMfmaArgs& a, int rb, hipStream_t st) {
  if (a.scores) {
    if (rb == 1) launch_block<D, QF16, 1, 8, true>(a, st);
    else launch_block<D, QF16, 2, 8, true>(a, st);
    const int key_wgs = a.n_units * ((a.tiles_max * kKeys + kFinishKeys - 1) / kFinishKeys);
    const int64_t rows = (int64_t)a.n_units * a.b.ratio * a.b.T;
    const int merge_wgs = a.n_split > 1 ? (int)((rows + 1024 / D - 1) / (1024 / D)) : 0;
    if (key_wgs + merge_wgs > 0)
      hipLaunchKernelGGL((block_finish_kernel<D, QF16>), dim3((unsigned)(key_wgs + merge_wgs)), dim3(256), 0, st, a,
                         key_wgs);
    return;
  }
  if (rb == 1) launch_block<D, QF16, 1, 8, false>(a, st);
  else launch_block<D, QF16, 2, 8, false>(a, st);
}

}  // namespace

BlockPlan block_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk) {
  const int64_t rows = T * (Hq / Hkv), units = B * Hkv;
  BlockPlan p;
  p.rb = rows <= 16 ? 1 : 2;
  p.nw = 8;
  p.row_chunks = (rows + 16 * p.rb - 1) / (16 * p.rb);
  // the split with the least estimate: rounds of one workgroup per CU, each its
  // waves' tiles and about two tiles' time of prologue and epilogue; a merge
  // costs about a tile's time and its partials' traffic
  const int64_t tiles = (Sk + kKeys - 1) / kKeys, wgs = units * p.row_chunks;
  p.n_split = 1;
  double best = 0.0;
  for (int64_t ns = 1; ns <= std::min<int64_t>(64, std::max<int64_t>(1, (tiles + p.nw - 1) / p.nw)); ++ns) {
    const double rounds = (double)((wgs * ns + 255) / 256);
    const double cost = rounds * ((double)((tiles + ns * p.nw - 1) / (ns * p.nw)) + 2.0) +
                        (ns > 1 ? 1.0 + (double)(units * rows * ns) * (double)D * 8.0 / 8.0e6 : 0.0);
    if (ns == 1 || cost < best) {
      best = cost;
      p.n_split = ns;
    }
  }
  p.ml_bytes = 0;
  p.o_bytes = 0;
  if (p.n_split > 1) {
    p.ml_bytes = (units * rows * p.n_split * 8 + 255) / 256 * 256;
    p.o_bytes = units * rows * p.n_split * D * 4;
  }
  return p;
}

namespace {
bool dense_rows(const void* p, int64_t b, int64_t h, int64_t s, int64_t row, int64_t n, int64_t size) {
  return s == row && (uintptr_t)p % (n * size) == 0 && b % n == 0 && h % n == 0;
}
}  // namespace

bool block_mfma_takes_keys(const BlockArgs& a) {
  if (!(a.D == 64 || a.D == 128) || !(a.G == 32 || a.G == 64 || a.G == 128) || a.D % a.G != 0) return false;
  const int ng = a.D / a.G;
  return a.q_dt != KVQ_F32 && a.s_dt != KVQ_F32 && a.qs_d == 1 && (!a.pm.paged || (a.pm.page_shift >= 6 && a.pm.n_pages > 0)) &&
         a.Sk < (int64_t(1) << 30) && dense_rows(a.kp, a.kps_b, a.kps_h, a.kps_s, a.D / 2, a.D / 8, 1) &&
         dense_rows(a.ks, a.kss_b, a.kss_h, a.kss_s, ng, ng, 2);
}

bool block_mfma_takes(const BlockArgs& a) {
  return block_mfma_takes_keys(a) && a.os_d == 1 && dense_rows(a.vp, a.vps_b, a.vps_h, a.vps_s, a.D / 2, 4, 1) &&
         dense_rows(a.vs, a.vss_b, a.vss_h, a.vss_s, a.D / a.G, a.D / a.G, 2);
}

void launch_block_merge(const BlockMfmaArgs& a, hipStream_t st) {
  const bool f16 = a.b.q_dt == KVQ_F16;
  if (a.b.D == 128) f16 ? launch_merge<128, true>(a, st) : launch_merge<128, false>(a, st);
  else f16 ? launch_merge<64, true>(a, st) : launch_merge<64, false>(a, st);
}

void fill_block_mfma(BlockMfmaArgs* a, const BlockArgs& b) {
  *a = BlockMfmaArgs{};
  a->b = b;
  a->n_units = b.B * b.Hkv;
  a->ng = b.D / b.G;
  a->s_f16 = b.s_dt == KVQ_F16;
  a->tiles_max = (int)((b.Sk + kKeys - 1) / kKeys);
  auto mult = [](const void* p, int64_t bytes, int64_t s0, int64_t s1, int64_t s2, int64_t n) {
    return (uintptr_t)p % bytes == 0 && s0 % n == 0 && s1 % n == 0 && s2 % n == 0;
  };
  a->q_vec = mult(b.q, 16, b.qs_b, b.qs_h, b.qs_s, 8);
  a->o_vec = b.out && mult(b.out, 8, b.os_b, b.os_h, b.os_s, 4);
}

namespace {

int launch_any(const BlockMfmaArgs& a, const BlockPlan& p, hipStream_t st) {
  if ((int64_t)a.n_units * a.row_chunks * a.n_split >= (int64_t(1) << 31)) return KVQ_EUNSUP;
  const bool f16 = a.b.q_dt == KVQ_F16;
  if (a.b.D == 128) {
    if (f16) launch_rb<128, true>(a, p.rb, st);
    else launch_rb<128, false>(a, p.rb, st);
  } else {
    if (f16) launch_rb<64, true>(a, p.rb, st);
    else launch_rb<64, false>(a, p.rb, st);
  }
  return KVQ_OK;
}

}  // namespace

int64_t block_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool s_f16) {
  if (T * (Hq / Hkv) > rows_min(s_f16)) {
    const RowsPlan p = rows_plan(B, Hq, Hkv, T, D, Sk, s_f16, false);
    return p.ml_bytes + p.o_bytes;
  }
  const BlockPlan p = block_plan(B, Hq, Hkv, T, D, Sk);
  return p.ml_bytes + p.o_bytes;
}

int launch_block_mfma(const BlockArgs& b, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  const bool fits = workspace != nullptr && (uintptr_t)workspace % 16 == 0 &&
                    workspace_bytes >= block_workspace_bytes(b.B, b.Hq, b.Hkv, b.T, b.D, b.Sk, b.s_dt == KVQ_F16);
  if ((int64_t)b.T * b.ratio > rows_min(b.s_dt == KVQ_F16)) {
    RowsPlan p = rows_plan(b.B, b.Hq, b.Hkv, b.T, b.D, b.Sk, b.s_dt == KVQ_F16, false);
    if (!fits) p.n_split = 1;
    RowsArgs a = {};
    fill_block_mfma(&a.m, b);
    a.m.ws_ml = (float2*)workspace;
    a.m.ws_o = (float*)((char*)workspace + p.ml_bytes);
    return launch_rows(a, p, st);
  }
  BlockPlan p = block_plan(b.B, b.Hq, b.Hkv, b.T, b.D, b.Sk);
  if (!fits) p.n_split = 1;
  BlockMfmaArgs a;
  fill_block_mfma(&a, b);
  a.row_chunks = (int)p.row_chunks;
  a.n_split = (int)p.n_split;
  a.ws_ml = (float2*)workspace;
  a.ws_o = (float*)((char*)workspace + p.ml_bytes);
  return launch_any(a, p, st);
}

int64_t block_scores_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk) {
  const int64_t rows = T * (Hq / Hkv);
  if (rows > kMaxScoreRows) return 0;
  const BlockPlan p = block_plan(B, Hq, Hkv, T, D, Sk);
  const int64_t ml = (B * Hkv * rows * p.n_split * 8 + 255) / 256 * 256;
  return ml + p.o_bytes + B * Hkv * ((Sk + kKeys - 1) / kKeys) * rows * kKeys * 4;
}

int launch_block_weights(const BlockArgs& b, float* weights, const int64_t* ws, void* workspace, hipStream_t st) {
  const int64_t rows = (int64_t)b.ratio * b.T;
  const BlockPlan p = block_plan(b.B, b.Hq, b.Hkv, b.T, b.D, b.Sk);
  BlockMfmaArgs a;
  fill_block_mfma(&a, b);
  a.row_chunks = (int)p.row_chunks;
  a.n_split = (int)p.n_split;
  const int64_t ml = ((int64_t)a.n_units * rows * p.n_split * 8 + 255) / 256 * 256;
  a.ws_ml = (float2*)workspace;
  a.ws_o = (float*)((char*)workspace + ml);
  a.scores = (float*)((char*)workspace + ml + p.o_bytes);
  a.weights = weights;
  a.w_b = ws[0]; a.w_h = ws[1]; a.w_k = ws[2];
  if ((int64_t)a.n_units * (a.tiles_max / 4 + 1) + a.n_units * rows >= (int64_t(1) << 31)) return KVQ_EUNSUP;
  return launch_any(a, p, st);
}

}  // namespace kvq
