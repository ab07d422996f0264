// The 32x32x16 matrix instruction's operands from the INT4 cache, shared by the
// kernels of many query rows (kvq_rows.hip) and of key weights (kvq_sums.hip).
//
// Scores are exact to fp32's rounding: a key's scales and a row's queries are
// brought near 1 by powers of two of their own (taken back in fp32 after the
// product), and then
//   - a bf16 query fits fp16;
//   - a code times a bf16 scale has 3 + 8 significant bits and fits fp16 too (a
//     group whose scale is under 2^-14 of the key's largest is off by 2^-25 of
//     that, fp32's own rounding of the sum);
//   - a code times an fp16 scale has 14 bits: TWO keeps it as fp16 hi + lo, for
//     two products; without it such a key is rounded to fp16.
// The eight dims of an operand piece are in the order (0, 4), (1, 5), (2, 6),
// (3, 7) of pairs, which the nibbles of a code word give for free.
#pragma once

#include "kvq_block_mfma.h"

namespace kvq {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16_t mfma(uint4 a, uint4 b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t d;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(d) : "v"(x), "s"(m), "v"(o));
  return d;
}
__device__ __forceinline__ uint32_t u32_of(f16x2_t v) { return __builtin_bit_cast(uint32_t, v); }

// The power of two that takes x > 0 into [1, 2), between 2^-100 and 2^100 (1 for 0).
__device__ __forceinline__ float unit_of(float x) {
  if (!(x > 0.0f)) return 1.0f;
  const int e = 127 - (int)(__builtin_bit_cast(uint32_t, x) >> 23);
  const int u = e < -100 ? -100 : (e > 100 ? 100 : e);
  return __builtin_bit_cast(float, (uint32_t)(u + 127) << 23);
}

// Codes times scales, as fp16. EXACT24 (bf16 scales): nibbles enter as fp16
// 16 + n (nibble at mantissa bits 6 .. 9), and one fma with -24 s, which has
// 8 + 2 bits, gives (n - 8) s exactly. fp16 scales: 1024 + n (bits 0 .. 3), minus
// 1032, times s.
struct CodeScale {
  uint32_t s, c;  // the pair of scales, and of -24 times them
};
template <bool EXACT24>
__device__ __forceinline__ CodeScale code_scale(uint32_t scales) {
  const f16x2_t k = {(_Float16)-24.0f, (_Float16)-24.0f};
  CodeScale r = {scales, 0u};
  if constexpr (EXACT24) r.c = u32_of(__builtin_bit_cast(f16x2_t, scales) * k);
  return r;
}
// The nibbles at bit `at` of x's halves.
template <bool EXACT24>
__device__ __forceinline__ uint32_t code_pair(uint32_t x, int at, CodeScale cs) {
  const f16x2_t s = __builtin_bit_cast(f16x2_t, cs.s);
  if constexpr (EXACT24) {
    const uint32_t y = at < 6 ? x << (6 - at) : x >> (at - 6);
    return u32_of(__builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, and_or(y, 0x03c003c0u, 0x4c004c00u)), s,
                                            __builtin_bit_cast(f16x2_t, cs.c)));
  } else {
    const f16x2_t off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    return u32_of((__builtin_bit_cast(f16x2_t, and_or(x >> at, 0x000f000fu, 0x64006400u)) + off) * s);
  }
}

// The eight codes of w times the scale s, as fp16 (TWO: the rest of the product
// as fp16 in lo).
template <bool TWO, bool EXACT24 = false>
__device__ __forceinline__ uint4 decode(uint32_t w, _Float16 s, uint4* lo) {
  const f16x2_t ss = {s, s};
  uint32_t hi[4], rest[4];
  if constexpr (TWO) {
    const f16x2_t off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const f16x2_t n = __builtin_bit_cast(f16x2_t, and_or(w >> (4 * p), 0x000f000fu, 0x64006400u)) + off;
      const f16x2_t v = n * ss;
      hi[p] = u32_of(v);
      rest[p] = u32_of(__builtin_elementwise_fma(n, ss, -v));
    }
    *lo = make_uint4(rest[0], rest[1], rest[2], rest[3]);
  } else {
    const CodeScale cs = code_scale<EXACT24>(u32_of(ss));
#pragma unroll
    for (int p = 0; p < 4; ++p) hi[p] = code_pair<EXACT24>(w, 4 * p, cs);
  }
  return make_uint4(hi[0], hi[1], hi[2], hi[3]);
}

// A key's scale row (up to four 16-bit scales in x): scale c as fp32.
__device__ __forceinline__ float scale_at(uint64_t x, int c, int s_f16) {
  const uint32_t v = (uint32_t)(x >> (16 * c)) & 0xffffu;
  return s_f16 ? f16_bits_to_f32(v) : bf16_bits_to_f32(v);
}
__device__ __forceinline__ uint64_t load_scale_row(const uint16_t* p, int ng) {
  if (ng == 4) {
    const uint2 v = *(const uint2*)p;
    return ((uint64_t)v.y << 32) | v.x;
  }
  return ng == 2 ? *(const uint32_t*)p : *p;
}
__device__ __forceinline__ uint2 load_scales(__amdgpu_buffer_rsrc_t r, uint32_t row, int ng) {
  uint2 v = make_uint2(0u, 0u);
  if (ng == 4) v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, 8 * row, 0, 0));
  else if (ng == 2) v.x = __builtin_amdgcn_raw_buffer_load_b32(r, 4 * row, 0, 0);
  else v.x = __builtin_amdgcn_raw_buffer_load_b16(r, 2 * row, 0, 0) & 0xffffu;
  return v;
}
// The power of two of a key's scales, and whether one is not finite.
__device__ __forceinline__ float key_unit(uint64_t x, int ng, int s_f16, bool* odd) {
  float top = 0.0f;
  for (int c = 0; c < ng; ++c) {
    const float v = fabsf(scale_at(x, c, s_f16));
    if (v < __builtin_inff()) top = fmaxf(top, v);
    else *odd = true;
  }
  return unit_of(top);
}

// Eight query elements, as fp32 and as an operand piece times `unit`.
template <bool QF16>
__device__ __forceinline__ void query_floats(uint4 x, float (&f)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = QF16 ? f16_bits_to_f32(w[k] & 0xffffu) : bf16_bits_to_f32(w[k] & 0xffffu);
    f[2 * k + 1] = QF16 ? f16_bits_to_f32(w[k] >> 16) : bf16_bits_to_f32(w[k] >> 16);
  }
}
template <bool QF16>
__device__ __forceinline__ uint4 query_piece(uint4 x, float unit) {
  float f[8];
  query_floats<QF16>(x, f);
  uint32_t p[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const f16x2_t v = {(_Float16)(f[k] * unit), (_Float16)(f[k + 4] * unit)};
    p[k] = u32_of(v);
  }
  return make_uint4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ uint4 load_query(const uint16_t* p, bool vec) {
  if (vec) return *(const uint4*)p;
  return make_uint4((uint32_t)p[0] | ((uint32_t)p[1] << 16), (uint32_t)p[2] | ((uint32_t)p[3] << 16),
                    (uint32_t)p[4] | ((uint32_t)p[5] << 16), (uint32_t)p[6] | ((uint32_t)p[7] << 16));
}


// A query row (this lane's half of each step's 16 dims, from p) as the B
// operand, times the power of two that is returned; `odd`: an element is not
// finite (all of the row's scores then are not). qneg flips the signs. The
// conversion is a loop over one piece that turns the registers round: this runs
// once per wave, and straight code would wait for its instructions.
template <bool QF16, int KS>
__device__ __forceinline__ float query_operand(const uint16_t* p, bool vec, uint32_t qneg, uint4 (&q)[KS], bool* odd) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  if (vec) {
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) q[kk] = *(const uint4*)(p + 16 * kk);
  } else {
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) q[kk] = load_query(p + 16 * kk, false);
  }
  u16x2_t top = {0, 0};
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) {
    const uint32_t w[4] = {q[kk].x, q[kk].y, q[kk].z, q[kk].w};
#pragma unroll
    for (int x = 0; x < 4; ++x) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[x] & 0x7fff7fffu));
  }
  const uint32_t lo = top[0], hi = top[1];
  uint32_t t = lo > hi ? lo : hi;
  const auto r = __builtin_amdgcn_permlane32_swap(t, t, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  t = r0 > r1 ? r0 : r1;
  *odd = t >= (QF16 ? 0x7c00u : 0x7f80u);
  const float u = *odd ? 1.0f : unit_of(QF16 ? f16_bits_to_f32(t) : bf16_bits_to_f32(t));
  const float un = qneg ? -u : u;
#pragma unroll 1
  for (int kk = 0; kk < KS; ++kk) {
    const uint4 x = query_piece<QF16>(q[0], un);
#pragma unroll
    for (int j = 0; j + 1 < KS; ++j) q[j] = q[j + 1];
    q[KS - 1] = x;
  }
  return u;
}

// The power of two that takes a value scale `top` into [1, 2), between 2^-100
// and 2^20 (scales that stay smaller are taken one key at a time; a larger
// factor could overflow a larger scale that follows).
__device__ __forceinline__ float value_unit(float top) {
  if (!(top > 0.0f)) return 1.0f;
  const int e = 127 - (int)(__builtin_bit_cast(uint32_t, top) >> 23);
  const int u = e < -100 ? -100 : (e > 20 ? 20 : e);
  return __builtin_bit_cast(float, (uint32_t)(u + 127) << 23);
}
// Whether fp16 does not hold a scale and its products with a code: a bf16
// scale's 8 + 3 bits exactly, an fp16 scale's rounded to 11.
__device__ __forceinline__ bool scale_odd(float s) {
  return !(fabsf(s) <= 0x1p12f) | ((s != 0.0f) & (fabsf(s) < 0x1p-14f));
}

}  // namespace kvq
