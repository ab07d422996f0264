// Key weights of long query blocks (prompts, prompt chunks) on the matrix
// cores (gfx950), for 16-bit queries and scales, D 64 and 128, aligned rows.
//
// Two passes over the scores S^T = K Q^T (v_mfma 32x32x16, both operands fp16),
// since a key's sum needs every row's softmax statistics first:
//   row_stats_kernel   (m, l) of each row over a share of the keys: the queries
//                      stay in registers (64 rows a wave), key tiles are decoded
//                      once per workgroup into an LDS image of the A operand
//   row_merge_kernel   the shares' statistics to (m, 1 / l)
//   key_sums_kernel    sum over a share of the rows of 2^(s - m) / l: the keys
//                      stay in registers, query tiles go through LDS
//   key_add_kernel     the shares' sums to the running sums, in a fixed order
//
// Scores are exact to fp32's rounding (kvq_operands.h).
// Both passes form them by the same instructions in the same order, so that a
// row's weights add up to 1.
//
// Layout of the 32x32x16 instruction (lane l: n = l % 32, g = l / 32): A[i][k] and
// B[k][n] at lane (i or n, k / 8), register k % 8; C[r][n] at lane n + 32 ((r / 4)
// % 2), register 4 (r / 8) + r % 4. A lane holds, of query row n, keys 8 (r / 4) +
// 4 g + r % 4.

#include <algorithm>

#include "kvq_operands.h"

namespace kvq {
namespace {

constexpr int kTile = 64;  // keys of a tile of the first pass, rows of one of the second
constexpr float kNeg = -1.0e30f;
constexpr float kLazyMax = 8.0f;
constexpr int kStatRows = 256;   // rows of a workgroup of the first pass (64 a wave)
constexpr int kStatTiles = 16;   // key tiles of its share
constexpr int kSumRowTiles = 16; // row tiles of a share of the second pass

struct SumArgs {
  BlockArgs b;
  int n_units, ng, s_f16, q_vec;
  int row_blocks, splits;  // first pass: row blocks, shares of the keys
  int key_blocks, chunks;  // second pass: key blocks, shares of the rows
  float2* part;            // [unit][row][split] (m, l)
  float* row_unit;         // [unit][row] power of two of the row's queries
  float2* stats;           // [unit][row] (m, 1 / l)
  float* sums;             // [unit][chunk][Sk]
  float* weights;
  int64_t w_b, w_h, w_k;
};

// Keys that row R may attend: [0, limit).
__device__ __forceinline__ int row_limit(const SumArgs& a, int R, int len) {
  if (R >= a.b.ratio * a.b.T) return 0;
  if (a.b.kind == kMaskNone) return len;
  const int x = len - a.b.T + R / a.b.ratio + 1;
  return x < 0 ? 0 : x;
}

// ---------------------------------------------------------------------------

template <int D, bool QF16, bool TWO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void row_stats_kernel(const SumArgs a) {
  constexpr int KS = D / 16;       // 16-dim steps
  constexpr int KP = D / 8 / 4;    // code words a thread decodes: a quarter of a key's
  constexpr int IMG = 2 * KS * 64; // pieces of a tile's image (per term)
  __shared__ __align__(16) uint4 img[2][(TWO ? 2 : 1) * IMG];
  __shared__ __align__(16) float back[2][kTile];  // what undoes the key's unit, times nothing else
  __shared__ int odd_lds[2][4];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, g = lane >> 5;
  int wg = blockIdx.x;
  const int unit = wg % a.n_units;
  wg /= a.n_units;
  const int blk = a.row_blocks - 1 - wg % a.row_blocks, sp = wg / a.row_blocks;  // blocks with the most keys first
  const int kvh = unit % a.b.Hkv, b = unit / a.b.Hkv;
  const int rows = a.b.ratio * a.b.T, len = (int)block_len(a.b, b);
  const int r_last = min((blk + 1) * kStatRows, rows) - 1;
  const int kend = row_limit(a, r_last, len);
  const int lo = sp * kStatTiles, hi = min((kend + kTile - 1) / kTile, lo + kStatTiles);

  // queries as the B operand, rows 32 r + n of the wave
  const float c = fmaxf(fabsf(a.b.scale_log2), 1.0e-30f);
  const uint32_t qneg = a.b.scale_log2 < 0.0f ? 0x80008000u : 0u;
  uint4 q[2][KS];
  float cr[2];
  int lim[2];
  bool odd_q = false;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int R = blk * kStatRows + wave * 64 + 32 * r + n, Rc = R < rows ? R : rows - 1;
    lim[r] = row_limit(a, R, len);
    const int i = Rc / a.b.ratio, h = kvh * a.b.ratio + Rc % a.b.ratio;
    const uint16_t* p = (const uint16_t*)a.b.q + b * a.b.qs_b + (int64_t)h * a.b.qs_h + (int64_t)i * a.b.qs_s + 8 * g;
    float top = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      uint4 x = load_query(p + 16 * kk, a.q_vec);
      x = make_uint4(x.x ^ qneg, x.y ^ qneg, x.z ^ qneg, x.w ^ qneg);
      q[r][kk] = x;
      float f[8];
      query_floats<QF16>(x, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float v = fabsf(f[k]);
        if (v < __builtin_inff()) top = fmaxf(top, v);
        else odd_q = true;
      }
    }
    const float u = unit_of(pair_max(top));
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) q[r][kk] = query_piece<QF16>(q[r][kk], u);
    cr[r] = c / u;
    if (sp == 0 && g == 0 && R < rows) a.row_unit[(int64_t)unit * rows + R] = u;
  }
  odd_q = __builtin_amdgcn_ballot_w64(odd_q) != 0;
  // keys every row of the wave attends (its first row's)
  const int R0 = blk * kStatRows + wave * 64;
  const int lim_wave = R0 < rows ? row_limit(a, R0, len) : 0x7fffffff;

  // tile loads: thread (key tid % 64, quarter tid / 64) takes KP code words
  const uint8_t* kp = a.b.kp + b * a.b.kps_b + kvh * a.b.kps_h;
  const uint16_t* ks = (const uint16_t*)a.b.ks + b * a.b.kss_b + kvh * a.b.kss_h;
  const int key = tid & 63, part = tid >> 6;
  uint32_t raw[KP];
  uint64_t sraw;
  auto load = [&](int t) {
    const int64_t j = min((int64_t)t * kTile + key, (int64_t)len - 1);  // (past the end: the last key, never attended)
    const uint8_t* p = kp + j * (D / 2) + part * (4 * KP);
    if constexpr (KP == 4) {
      const uint4 v = *(const uint4*)p;
      raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
    } else {
      const uint2 v = *(const uint2*)p;
      raw[0] = v.x; raw[1] = v.y;
    }
    sraw = load_scale_row(ks + j * a.ng, a.ng);
  };
  auto store = [&](int buf) {
    bool odd = false;
    const float u = key_unit(sraw, a.ng, a.s_f16, &odd);
    const _Float16 s = (_Float16)(scale_at(sraw, part * (8 * KP) / a.b.G, a.s_f16) * u);
#pragma unroll
    for (int j = 0; j < KP; ++j) {  // dims 8 (KP part + j) .. + 7: step (KP part + j) / 2, half j % 2
      const int piece = KP * part + j;
      uint4 rest;
      uint4* dst = img[buf] + ((key >> 5) * KS + (piece >> 1)) * 64 + 32 * (piece & 1) + (key & 31);
      *dst = decode<TWO>(raw[j], s, &rest);
      if constexpr (TWO) dst[IMG] = rest;
    }
    if (part == 0) back[buf][key] = 1.0f / u;
    const bool any = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) odd_lds[buf][wave] = any;
  };

  float m[2] = {kNeg, kNeg}, l[2] = {0.0f, 0.0f};
  if (lo < hi) {
    load(lo);
    store(0);
    if (lo + 1 < hi) load(lo + 1);
  }
  __syncthreads();
  for (int t = lo; t < hi; ++t) {
    const int cur = (t - lo) & 1, t0 = t * kTile;
    const uint4* kt = img[cur];
    if (t + 1 < hi) {
      store(cur ^ 1);
      if (t + 2 < hi) load(t + 2);
    }
    const bool odd = odd_q || (odd_lds[cur][0] | odd_lds[cur][1] | odd_lds[cur][2] | odd_lds[cur][3]) != 0;
    f32x16_t s[2][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        const uint4 x = kt[(kb * KS + kk) * 64 + lane];
        f32x16_t zero;
#pragma unroll
        for (int j = 0; j < 16; ++j) zero[j] = 0.0f;
#pragma unroll
        for (int r = 0; r < 2; ++r) s[r][kb] = mfma(x, q[r][kk], kk == 0 ? zero : s[r][kb]);
        if constexpr (TWO) {
          const uint4 y = kt[IMG + (kb * KS + kk) * 64 + lane];
#pragma unroll
          for (int r = 0; r < 2; ++r) s[r][kb] = mfma(y, q[r][kk], s[r][kb]);
        }
      }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float4 u = *(const float4*)(back[cur] + 32 * kb + 8 * x + 4 * g);
        const float uj[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[r][kb][4 * x + j] *= uj[j];
      }
    if (odd) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[r][kb][j] = block_score(s[r][kb][j]);
    }
    if (t0 + kTile > lim_wave) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (t0 + 32 * kb + 8 * (j >> 2) + 4 * g + (j & 3) >= lim[r]) s[r][kb][j] = -__builtin_inff();
    }
    float mt[2];
    bool grow = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = s[r][0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[r][kb][j]);
      mt[r] = pair_max(mx) * cr[r];
      grow = grow || mt[r] > m[r] + kLazyMax;
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m_new = fmaxf(m[r], mt[r]);
        l[r] *= __builtin_amdgcn_exp2f(m[r] - m_new);
        m[r] = m_new;
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x[2] = {0.0f, 0.0f};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j & 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][kb][j], cr[r], -m[r]));
      l[r] += x[0] + x[1];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int R = blk * kStatRows + wave * 64 + 32 * r + n;
    const float L = pair_sum(l[r]);
    if (g == 0 && R < rows) a.part[((int64_t)unit * rows + R) * a.splits + sp] = make_float2(m[r], L);
  }
}

// A thread a row: memory-bound, 8 bytes a share.
__global__ __launch_bounds__(256) void row_merge_kernel(const SumArgs a, int64_t n) {
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= n) return;
  const float2* p = a.part + row * a.splits;
  float M = kNeg, L = 0.0f;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, p[s].x);
  for (int s = 0; s < a.splits; ++s) L = fmaf(p[s].y, __builtin_amdgcn_exp2f(p[s].x - M), L);
  a.stats[row] = L > 0.0f ? make_float2(M, 1.0f / L) : make_float2(0.0f, 0.0f);
}

// KB = 32-key blocks a wave keeps in registers (TWO: one, whose two terms take
// the registers of two).
template <int D, bool QF16, bool TWO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void key_sums_kernel(const SumArgs a) {
  constexpr int KS = D / 16, KB = TWO ? 1 : 2;
  constexpr int KEYS = 4 * 32 * KB;  // keys of a workgroup
  constexpr int PC = 2 * KS / 4;     // pieces of a row tile that a thread brings in
  __shared__ __align__(16) uint4 img[2][2 * KS * 64];
  __shared__ __align__(16) float4 row_lds[2][kTile];  // (m, 1 / l, c / unit, limit as bits)
  __shared__ int odd_lds[2][4];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, g = lane >> 5;
  int wg = blockIdx.x;
  const int unit = wg % a.n_units;
  wg /= a.n_units;
  const int kblk = wg % a.key_blocks, ch = wg / a.key_blocks;
  const int kvh = unit % a.b.Hkv, b = unit / a.b.Hkv;
  const int rows = a.b.ratio * a.b.T, len = (int)block_len(a.b, b);
  const int k0 = kblk * KEYS;
  float* dst = a.sums + ((int64_t)unit * a.chunks + ch) * a.b.Sk;
  if (k0 >= len) return;  // (nothing reads these sums)
  // row tiles of this share in which some row attends key k0
  int first = 0;
  if (a.b.kind != kMaskNone) {
    const int64_t i = (int64_t)k0 - (len - a.b.T);
    first = i <= 0 ? 0 : (int)(i * a.b.ratio / kTile);
  }
  const int lo = max(ch * kSumRowTiles, first), hi = min((ch + 1) * kSumRowTiles, (rows + kTile - 1) / kTile);

  // this wave's keys as the A operand
  const uint8_t* kp = a.b.kp + b * a.b.kps_b + kvh * a.b.kps_h;
  const uint16_t* ks = (const uint16_t*)a.b.ks + b * a.b.kss_b + kvh * a.b.kss_h;
  uint4 k[KB][(TWO ? 2 : 1) * KS];
  float back[KB][16];  // register j of a block: key 8 (j / 4) + 4 g + j % 4
  bool odd_k = false;
  const int kw = k0 + wave * 32 * KB;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int64_t j = min((int64_t)kw + 32 * kb + n, (int64_t)len - 1);
    const uint64_t sraw = load_scale_row(ks + j * a.ng, a.ng);
    const float u = key_unit(sraw, a.ng, a.s_f16, &odd_k);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const uint32_t w = *(const uint32_t*)(kp + j * (D / 2) + 4 * (2 * kk + g));
      const _Float16 s = (_Float16)(scale_at(sraw, 16 * kk / a.b.G, a.s_f16) * u);
      uint4 rest;
      k[kb][kk] = decode<TWO>(w, s, &rest);
      if constexpr (TWO) k[kb][KS + kk] = rest;
    }
    const float ub = 1.0f / u;
#pragma unroll
    for (int x = 0; x < 16; ++x) back[kb][x] = __shfl(ub, 8 * (x >> 2) + 4 * g + (x & 3));
  }
  odd_k = __builtin_amdgcn_ballot_w64(odd_k) != 0;

  // row tiles: wave w brings the pieces of steps w, w + 4 of both 32-row blocks
  const float c = fmaxf(fabsf(a.b.scale_log2), 1.0e-30f);
  const uint32_t qneg = a.b.scale_log2 < 0.0f ? 0x80008000u : 0u;
  uint4 raw[PC];
  float unit_raw[2];
  float4 st_raw;
  auto load = [&](int t) {
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int R = min(t * kTile + 32 * rb + n, rows - 1);
      const int i = R / a.b.ratio, h = kvh * a.b.ratio + R % a.b.ratio;
      const uint16_t* p = (const uint16_t*)a.b.q + b * a.b.qs_b + (int64_t)h * a.b.qs_h + (int64_t)i * a.b.qs_s + 8 * g;
      // (a row that weighs nothing enters as zeros, whatever it holds)
      unit_raw[rb] = a.stats[(int64_t)unit * rows + R].y > 0.0f ? a.row_unit[(int64_t)unit * rows + R] : 0.0f;
#pragma unroll
      for (int x = 0; x < PC / 2; ++x) raw[rb * (PC / 2) + x] = load_query(p + 16 * (wave + 4 * x), a.q_vec);
    }
    if (tid < kTile) {
      const int R = t * kTile + tid, Rc = min(R, rows - 1);
      const float2 st = a.stats[(int64_t)unit * rows + Rc];
      const int lim = row_limit(a, R, len);  // (0 past the last row)
      st_raw = make_float4(st.x, R < rows ? st.y : 0.0f, c / a.row_unit[(int64_t)unit * rows + Rc],
                           __builtin_bit_cast(float, lim));
    }
  };
  auto store = [&](int buf) {
    bool odd = false;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int x = 0; x < PC / 2; ++x) {
        uint4 v = raw[rb * (PC / 2) + x];
        const uint32_t top = QF16 ? 0x7c00u : 0x7f80u;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) odd = odd || (w[y] & top) == top || ((w[y] >> 16) & top) == top;
        const uint32_t keep = unit_raw[rb] > 0.0f ? 0xffffffffu : 0u;
        v = make_uint4((v.x & keep) ^ qneg, (v.y & keep) ^ qneg, (v.z & keep) ^ qneg, (v.w & keep) ^ qneg);
        img[buf][(rb * KS + wave + 4 * x) * 64 + lane] = query_piece<QF16>(v, unit_raw[rb]);
      }
    if (tid < kTile) row_lds[buf][tid] = st_raw;
    const bool any = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) odd_lds[buf][wave] = any;
  };

  float sum[KB][16];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[kb][x] = 0.0f;
  if (lo < hi) {
    load(lo);
    store(0);
    if (lo + 1 < hi) load(lo + 1);
  }
  __syncthreads();
  for (int t = lo; t < hi; ++t) {
    const int cur = (t - lo) & 1;
    if (t + 1 < hi) {
      store(cur ^ 1);
      if (t + 2 < hi) load(t + 2);
    }
    const bool odd = odd_k || (odd_lds[cur][0] | odd_lds[cur][1] | odd_lds[cur][2] | odd_lds[cur][3]) != 0;
    // the fewest keys a row of the tile attends: its first row's
    const int lim_tile = row_limit(a, t * kTile, len);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const float4 rs = row_lds[cur][32 * rb + n];
      const float m = rs.x, inv = rs.y, cr = rs.z;
      const int lim = __builtin_bit_cast(int, rs.w);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        f32x16_t s;
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          const uint4 q = img[cur][(rb * KS + kk) * 64 + lane];
          s = mfma(k[kb][kk], q, s);
          if constexpr (TWO) s = mfma(k[kb][KS + kk], q, s);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] *= back[kb][x];
        if (odd) {
#pragma unroll
          for (int x = 0; x < 16; ++x) s[x] = block_score(s[x]);
        }
        if (kw + 32 * (kb + 1) > lim_tile || (t + 1) * kTile > rows) {
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (kw + 32 * kb + 8 * (x >> 2) + 4 * g + (x & 3) >= lim) s[x] = -__builtin_inff();
        }
#pragma unroll
        for (int x = 0; x < 16; ++x)
          sum[kb][x] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[x], cr, -m)), inv, sum[kb][x]);
        __builtin_amdgcn_sched_barrier(0);  // (one score block at a time: registers)
      }
    }
    __syncthreads();
  }
  // over the 32 lanes of a key's rows
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      float v = sum[kb][x];
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor(v, d);
      const int key = kw + 32 * kb + 8 * (x >> 2) + 4 * g + (x & 3);
      if (n == 0 && key < len) dst[key] = v;
    }
}

// A thread a key: memory-bound.
__global__ __launch_bounds__(256) void key_add_kernel(const SumArgs a) {
  const int unit = blockIdx.y, kvh = unit % a.b.Hkv, b = unit / a.b.Hkv;
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j >= block_len(a.b, b)) return;
  const float* p = a.sums + (int64_t)unit * a.chunks * a.b.Sk + j;
  float v = 0.0f;
  for (int x = 0; x < a.chunks; ++x) v += p[x * a.b.Sk];
  a.weights[b * a.w_b + kvh * a.w_h + j * a.w_k] += v;
}

template <int D, bool QF16, bool TWO>
void launch(const SumArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.n_units * a.b.ratio * a.b.T;
  hipLaunchKernelGGL((row_stats_kernel<D, QF16, TWO>), dim3((unsigned)((int64_t)a.n_units * a.row_blocks * a.splits)),
                     dim3(256), 0, st, a);
  hipLaunchKernelGGL(row_merge_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, st, a, rows);
  hipLaunchKernelGGL((key_sums_kernel<D, QF16, TWO>), dim3((unsigned)((int64_t)a.n_units * a.key_blocks * a.chunks)),
                     dim3(256), 0, st, a);
  hipLaunchKernelGGL(key_add_kernel, dim3((unsigned)((a.b.Sk + 255) / 256), (unsigned)a.n_units), dim3(256), 0, st, a);
}

struct SumPlan {
  int64_t row_blocks, splits, key_blocks, chunks;
  int64_t part, unit, stats, sums;  // bytes
};

SumPlan sum_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t Sk, bool two) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t rows = T * (Hq / Hkv), units = B * Hkv, keys = two ? 128 : 256;
  SumPlan p;
  p.row_blocks = (rows + kStatRows - 1) / kStatRows;
  p.splits = std::max<int64_t>(1, ((Sk + kTile - 1) / kTile + kStatTiles - 1) / kStatTiles);
  p.key_blocks = (Sk + keys - 1) / keys;
  p.chunks = ((rows + kTile - 1) / kTile + kSumRowTiles - 1) / kSumRowTiles;
  p.part = up(units * rows * p.splits * 8);
  p.unit = up(units * rows * 4);
  p.stats = up(units * rows * 8);
  p.sums = up(units * p.chunks * Sk * 4);
  return p;
}

}  // namespace

int64_t sums_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t Sk, bool s_f16) {
  const SumPlan p = sum_plan(B, Hq, Hkv, T, Sk, s_f16);
  return p.part + p.unit + p.stats + p.sums;
}

int launch_key_sums(const BlockArgs& b, float* weights, const int64_t* ws, void* workspace, hipStream_t st) {
  const bool two = b.s_dt == KVQ_F16;
  const SumPlan p = sum_plan(b.B, b.Hq, b.Hkv, b.T, b.Sk, two);
  const int64_t units = (int64_t)b.B * b.Hkv;
  if (b.Sk == 0) return KVQ_OK;
  if (units * p.row_blocks * p.splits >= (int64_t(1) << 31) || units * p.key_blocks * p.chunks >= (int64_t(1) << 31) ||
      units >= 65536 || (int64_t)b.T * b.ratio >= (int64_t(1) << 30))
    return KVQ_EUNSUP;
  SumArgs a = {};
  a.b = b;
  a.n_units = (int)units;
  a.ng = b.D / b.G;
  a.s_f16 = two;
  a.q_vec = (uintptr_t)b.q % 16 == 0 && b.qs_b % 8 == 0 && b.qs_h % 8 == 0 && b.qs_s % 8 == 0;
  a.row_blocks = (int)p.row_blocks; a.splits = (int)p.splits;
  a.key_blocks = (int)p.key_blocks; a.chunks = (int)p.chunks;
  char* w = (char*)workspace;
  a.part = (float2*)w;
  a.row_unit = (float*)(w + p.part);
  a.stats = (float2*)(w + p.part + p.unit);
  a.sums = (float*)(w + p.part + p.unit + p.stats);
  a.weights = weights;
  a.w_b = ws[0]; a.w_h = ws[1]; a.w_k = ws[2];
  const bool f16 = b.q_dt == KVQ_F16;
  if (b.D == 128) {
    if (f16) two ? launch<128, true, true>(a, st) : launch<128, true, false>(a, st);
    else two ? launch<128, false, true>(a, st) : launch<128, false, false>(a, st);
  } else {
    if (f16) two ? launch<64, true, true>(a, st) : launch<64, true, false>(a, st);
    else two ? launch<64, false, true>(a, st) : launch<64, false, false>(a, st);
  }
  return KVQ_OK;
}

}  // namespace kvq
