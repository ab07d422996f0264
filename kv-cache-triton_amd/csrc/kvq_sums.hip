// Key weights of long query blocks (prompts, prompt chunks) on the matrix
// cores (gfx950), for 16-bit queries and scales, D 64 and 128, aligned rows.
//
// Two passes over the scores S^T = K Q^T (v_mfma 32x32x16, both operands fp16),
// since a key's sum needs every row's softmax statistics first:
//   the attention (kvq_rows.hip), or without values
//   row_stats_kernel   (m, l) of each row over a share of the keys: the queries
//                      stay in registers (64 rows a wave), key tiles are decoded
//                      once per workgroup into an LDS image of the A operand
//   row_merge_kernel   the shares' statistics to (m, 1 / l)
// either of which also leaves the queries as fp16 operands, and
//   key_sums_kernel    sum over a share of the rows of 2^(s - m) / l: the keys
//                      stay in registers, query tiles go through LDS
//   key_add_kernel     the shares' sums to the running sums, in a fixed order
//
// Measured on a causal 4K prompt, 32 query heads over 8: key_sums_kernel 139 us
// (494 TFLOP/s of scores; 246 when queries were converted in every workgroup and
// products and exponentials took turns, 203 with the shares of the rows fixed),
// row_stats_kernel 140, the additions 5. Bound by matrix cycles and exponentials,
// which add up (256 and 450 cycles a 32 x 32 block).
//
// Scores are exact to fp32's rounding (kvq_operands.h). Both passes form them by
// the same instructions in the same order, so that a row's weights add up to 1.
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

struct SumArgs {
  BlockArgs b;
  QueryImages qi;
  int n_units, ng, s_f16, q_vec;
  int row_blocks, splits;  // first pass: row blocks, shares of the keys
  int key_blocks, chunks, chunk_tiles;  // second pass: key blocks, shares of the rows, row tiles of a share
  float2* part;            // [unit][row][split] (m, l)
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
  uint4 q[2][KS];
  float cr[2];
  int lim[2];
  bool odd_q = false;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int R0 = blk * kStatRows + wave * 64 + 32 * r, R = R0 + n, Rc = R < rows ? R : rows - 1;
    lim[r] = row_limit(a, R, len);
    const int i = Rc / a.b.ratio, h = kvh * a.b.ratio + Rc % a.b.ratio;
    const uint16_t* p = (const uint16_t*)a.b.q + b * a.b.qs_b + (int64_t)h * a.b.qs_h + (int64_t)i * a.b.qs_s + 8 * g;
    bool odd = false;
    const float u = query_operand<QF16, KS>(p, a.q_vec, a.b.scale_log2 < 0.0f, q[r], &odd);
    odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    odd_q = odd_q || odd;
    cr[r] = c / u;
    if (sp == 0 && R0 < rows) {
      const int64_t block = (int64_t)unit * a.qi.blocks + R0 / 32;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) a.qi.img[(block * KS + kk) * 64 + lane] = q[r][kk];
      if (lane == 0) a.qi.odd[block] = odd;
      if (g == 0 && R < rows) a.qi.unit[(int64_t)unit * rows + R] = u;
    }
  }
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
    const _Float16 s = (_Float16)(scale_at(sraw, part * (8 * KP) * a.ng / D, a.s_f16) * u);
#pragma unroll
    for (int j = 0; j < KP; ++j) {  // dims 8 (KP part + j) .. + 7: step (KP part + j) / 2, half j % 2
      const int piece = KP * part + j;
      uint4 rest;
      uint4* dst = img[buf] + ((key >> 5) * KS + (piece >> 1)) * 64 + 32 * (piece & 1) + (key & 31);
      *dst = decode<TWO, !TWO>(raw[j], s, &rest);
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
// the registers of two). The products of one 32 x 32 block of scores are issued
// between the exponentials of the block before: matrix instructions hide the
// vector work of their own wave only.
template <int D, bool TWO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void key_sums_kernel(const SumArgs a) {
  constexpr int KS = D / 16, KB = TWO ? 1 : 2;
  constexpr int KEYS = 4 * 32 * KB;      // keys of a workgroup
  constexpr int IMG = 2 * KS * 64;       // 16-byte pieces of a row tile
  constexpr int PC = IMG / 256;          // of them a thread's
  constexpr int NM = KS * (TWO ? 2 : 1); // products of a block
  __shared__ __align__(16) uint4 img[2][IMG];
  __shared__ __align__(16) float4 row_lds[2][kTile];  // (m, 1 / l, c / unit, limit as bits)

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
  const int lo = max(ch * a.chunk_tiles, first), hi = min((ch + 1) * a.chunk_tiles, (rows + kTile - 1) / kTile);
  if (lo >= hi) {
    for (int j = k0 + tid; j < min(k0 + KEYS, len); j += 256) dst[j] = 0.0f;
    return;
  }

  // row tiles: thread tid brings pieces tid, tid + 256, ...
  const float c = fmaxf(fabsf(a.b.scale_log2), 1.0e-30f);
  const uint4* qi = a.qi.img + (int64_t)unit * a.qi.blocks * KS * 64 + tid;
  const int* q_odd = a.qi.odd + (int64_t)unit * a.qi.blocks;
  uint4 raw[PC];
  float4 st_raw;
  int odd_next = 0;  // of the tile in `raw`
  auto load = [&](int t) {
#pragma unroll
    for (int x = 0; x < PC; ++x) {
      const int rb = x / (PC / 2);  // (past the last block: the last, weighed 0)
      raw[x] = qi[(int64_t)min(2 * t + rb, a.qi.blocks - 1) * KS * 64 + 256 * (x % (PC / 2))];
    }
    odd_next = q_odd[min(2 * t, a.qi.blocks - 1)] | q_odd[min(2 * t + 1, a.qi.blocks - 1)];
    // (a row that weighs nothing, or is past the last: 2^(s - 3e38) times 0)
    const int R = t * kTile + lane, Rc = min(R, rows - 1);
    const float2 st = a.stats[(int64_t)unit * rows + Rc];
    const bool on = R < rows && st.y > 0.0f;
    st_raw = make_float4(on ? st.x : 3.0e38f, on ? st.y : 0.0f, c / a.qi.unit[(int64_t)unit * rows + Rc],
                         __builtin_bit_cast(float, row_limit(a, R, len)));
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int x = 0; x < PC; ++x) img[buf][tid + 256 * x] = raw[x];
    if (wave == 0) row_lds[buf][lane] = st_raw;
  };
  load(lo);

  // this wave's keys as the A operand, times the power of two of the key with
  // the largest scale; keys that fp16 would not hold so take their own, and the
  // rare path their difference
  const uint8_t* kp = a.b.kp + b * a.b.kps_b + kvh * a.b.kps_h;
  const uint16_t* ks = (const uint16_t*)a.b.ks + b * a.b.kss_b + kvh * a.b.kss_h;
  uint4 k[KB][(TWO ? 2 : 1) * KS];
  float back[KB][16];  // of register j of a block: key 8 (j / 4) + 4 g + j % 4
  bool odd_k = false;
  const int kw = k0 + wave * 32 * KB;
  // (no branches and few instructions: this runs once per workgroup, and straight
  // code waits for its instructions)
  constexpr int NC = D / 32;
  float sc[KB][NC], u[KB], u_wave = 0x1p100f;
  uint32_t w[KB][KS];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int64_t j = min((int64_t)kw + 32 * kb + n, (int64_t)len - 1);
    uint32_t bits[NC], top = 0u;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) bits[cc] = ks[j * a.ng + cc * a.ng / NC];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) w[kb][kk] = *(const uint32_t*)(kp + j * (D / 2) + 4 * (2 * kk + g));
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      top = max(top, bits[cc] & 0x7fffu);
      sc[kb][cc] = TWO ? f16_bits_to_f32(bits[cc]) : bf16_bits_to_f32(bits[cc]);
    }
    const bool odd = top >= (TWO ? 0x7c00u : 0x7f80u);  // (a key that is not finite: the unit 1)
    odd_k |= odd;
    u[kb] = odd ? 1.0f : unit_of(TWO ? f16_bits_to_f32(top) : bf16_bits_to_f32(top));
    u_wave = fminf(u_wave, u[kb]);
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) u_wave = fminf(u_wave, __shfl_xor(u_wave, d));
  bool any_far = false;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const bool far = u_wave < u[kb] * 0x1p-13f;
    any_far |= far;
    u[kb] = far ? u[kb] : u_wave;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      uint4 rest;
      k[kb][kk] = decode<TWO, !TWO>(w[kb][kk], (_Float16)(sc[kb][kk / 2] * u[kb]), &rest);
      if constexpr (TWO) k[kb][KS + kk] = rest;
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) back[kb][x] = 1.0f;
  }
  if (__builtin_amdgcn_ballot_w64(any_far) != 0) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const float ub = u_wave / u[kb];
#pragma unroll
      for (int x = 0; x < 16; ++x) back[kb][x] = __shfl(ub, 8 * (x >> 2) + 4 * g + (x & 3));
    }
  }
  odd_k = __builtin_amdgcn_ballot_w64(odd_k | any_far) != 0;
  const float back_wave = 1.0f / u_wave;

  float sum[KB][16];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int x = 0; x < 16; ++x) sum[kb][x] = 0.0f;
  store(0);
  int odd = odd_k | odd_next;
  if (lo + 1 < hi) load(lo + 1);
  __syncthreads();

  // the block before: its scores, rows and whether it needs the rare path
  f32x16_t s_old;
#pragma unroll
  for (int x = 0; x < 16; ++x) s_old[x] = -__builtin_inff();
  float4 r_old = make_float4(0.0f, 0.0f, 1.0f, 0.0f);
  bool rare_old = false;
  // scores that are not finite or of keys with units of their own, and keys that
  // a row does not attend, of keys k_first ..
  auto rare = [&](f32x16_t& s, const float (&bk)[16], float lim, int k_first) {
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      s[x] = block_score(s[x] * bk[x]);
      if (k_first + 8 * (x >> 2) + 4 * g + (x & 3) >= __builtin_bit_cast(int, lim)) s[x] = -__builtin_inff();
    }
  };
  auto weigh = [&](const f32x16_t& s, const float4& r, float (&to)[16], int x) {
    to[x] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[x], r.z, -r.x)), r.y, to[x]);
  };
#pragma unroll 1
  for (int t = lo; t < hi; ++t) {
    const int cur = (t - lo) & 1;
    const int odd_cur = odd;
    if (t + 1 < hi) {
      store(cur ^ 1);
      odd = odd_k | odd_next;
      if (t + 2 < hi) load(t + 2);
    }
    // the fewest keys a row of the tile attends: its first row's
    const int lim_tile = row_limit(a, t * kTile, len);
    const uint4* qt = img[cur] + lane;
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j) {
      const int rb = j / KB, kb = j % KB, kb_old = (j + KB - 1) % KB;
      if (rare_old) rare(s_old, back[kb_old], r_old.w, kw + 32 * kb_old);
      f32x16_t s;
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] = 0.0f;
      uint4 f[2];
      f[0] = qt[rb * KS * 64];
#pragma unroll
      for (int x = 0; x < NM; ++x) {
        const int kk = TWO ? x / 2 : x;
        if ((!TWO || x % 2 == 0) && kk + 1 < KS) f[(kk + 1) & 1] = qt[(rb * KS + kk + 1) * 64];
        s = mfma(k[kb][TWO && x % 2 == 1 ? KS + kk : kk], f[kk & 1], s);
#pragma unroll
        for (int y = 0; y < 16 / NM; ++y) {
          weigh(s_old, r_old, sum[kb_old], x * (16 / NM) + y);
          asm volatile("" : "+v"(sum[kb_old][x * (16 / NM) + y]));  // (here, not where the sums are next read)
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      s_old = s;
      r_old = row_lds[cur][32 * rb + n];
      r_old.z *= back_wave;
      rare_old = odd_cur || kw + 32 * (kb + 1) > lim_tile;
    }
    __syncthreads();
  }
  if (rare_old) rare(s_old, back[KB - 1], r_old.w, kw + 32 * (KB - 1));
#pragma unroll
  for (int x = 0; x < 16; ++x) weigh(s_old, r_old, sum[KB - 1], x);
  // over the 32 lanes of a key's rows: at each step a lane passes on half of its
  // keys and takes the other half's sums, so that lane n ends with key n's
  float v[16 * KB];
#pragma unroll
  for (int x = 0; x < 16 * KB; ++x) v[x] = sum[x / 16][x % 16];
  int d = 16;
#pragma unroll
  for (int half = 8 * KB; half >= 1; half /= 2) {
    const bool up = (n & d) != 0;
#pragma unroll
    for (int x = 0; x < half; ++x) {
      const float mine = up ? v[x + half] : v[x], other = up ? v[x] : v[x + half];
      v[x] = mine + __shfl_xor(other, d);
    }
    d /= 2;
  }
  if constexpr (KB == 1) v[0] += __shfl_xor(v[0], 1);
  const int e = KB == 1 ? n >> 1 : n;  // block e / 16, register e % 16
  const int key = kw + 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * g + (e & 3);
  if (key < len && (KB == 2 || n % 2 == 0)) dst[key] = v[0];
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

struct SumPlan {
  int64_t row_blocks, splits, key_blocks, chunks, chunk_tiles, q_blocks;
  int64_t unit, img, odd, stats, scratch;  // bytes
  RowsPlan rows;
};

SumPlan sum_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool causal, bool two, bool attend) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t rows = T * (Hq / Hkv), units = B * Hkv, keys = two ? 128 : 256;
  SumPlan p;
  p.row_blocks = (rows + kStatRows - 1) / kStatRows;
  p.splits = std::max<int64_t>(1, ((Sk + kTile - 1) / kTile + kStatTiles - 1) / kStatTiles);
  p.key_blocks = (Sk + keys - 1) / keys;
  // shares of the rows: the number of them with the least estimate, in tiles'
  // times: rounds of the 512 workgroups that are resident together, each its
  // tiles and about three tiles' time of prologue (4K prompt with its attention:
  // 12 shares 315 us, 16 323, 20, the estimate's, 303, 32 324, 48 332)
  const int64_t tiles = (rows + kTile - 1) / kTile, ratio = Hq / Hkv;
  double best = 0.0;
  p.chunks = p.chunk_tiles = 0;
  for (const int64_t n : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 48, 64}) {
    if (n > tiles) break;
    const int64_t each = (tiles + n - 1) / n, shares = (tiles + each - 1) / each;
    int64_t wgs = 0;  // that some row attends
    for (int64_t x = 0; x < shares; ++x) {
      const int64_t last = std::min((x + 1) * each * kTile, rows) - 1, seen = Sk - T + last / ratio + 1;
      wgs += causal ? std::min(p.key_blocks, std::max<int64_t>(0, seen + keys - 1) / keys) : p.key_blocks;
    }
    const double cost = (double)((units * wgs + 511) / 512) * (double)(each + 3);
    if (n == 1 || cost < best) {
      best = cost;
      p.chunks = shares;
      p.chunk_tiles = each;
    }
  }
  p.q_blocks = (rows + 31) / 32;
  p.unit = up(units * rows * 4);
  p.img = units * p.q_blocks * 32 * D * 2;
  p.odd = up(units * p.q_blocks * 4);
  p.stats = up(units * rows * 8);
  // one after the other: the first pass's partials, the second's sums
  p.scratch = units * p.chunks * Sk * 4;
  if (attend) {
    p.rows = rows_plan(B, Hq, Hkv, T, D, Sk, two, true);
    p.scratch = std::max(p.scratch, p.rows.ml_bytes + p.rows.o_bytes);
  } else {
    p.scratch = std::max(p.scratch, units * rows * p.splits * 8);
  }
  return p;
}

template <int D, bool QF16, bool TWO>
void launch_stats(const SumArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.n_units * a.b.ratio * a.b.T;
  hipLaunchKernelGGL((row_stats_kernel<D, QF16, TWO>), dim3((unsigned)((int64_t)a.n_units * a.row_blocks * a.splits)),
                     dim3(256), 0, st, a);
  hipLaunchKernelGGL(row_merge_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, st, a, rows);
}

template <int D, bool TWO>
void launch_sums(const SumArgs& a, bool stats, hipStream_t st) {
  if (stats) {
    if (a.b.q_dt == KVQ_F16) launch_stats<D, true, TWO>(a, st);
    else launch_stats<D, false, TWO>(a, st);
  }
  hipLaunchKernelGGL((key_sums_kernel<D, TWO>), dim3((unsigned)((int64_t)a.n_units * a.key_blocks * a.chunks)),
                     dim3(256), 0, st, a);
  hipLaunchKernelGGL(key_add_kernel, dim3((unsigned)((a.b.Sk + 255) / 256), (unsigned)a.n_units), dim3(256), 0, st, a);
}

}  // namespace

int64_t sums_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool s_f16, bool attend) {
  // (the mask is the call's: as much as either needs)
  const SumPlan c = sum_plan(B, Hq, Hkv, T, D, Sk, true, s_f16, attend), f = sum_plan(B, Hq, Hkv, T, D, Sk, false, s_f16, attend);
  return c.unit + c.img + c.odd + c.stats + std::max(c.scratch, f.scratch);
}

int launch_key_sums(const BlockArgs& b, bool attend, float* weights, const int64_t* ws, void* workspace, hipStream_t st) {
  const bool two = b.s_dt == KVQ_F16;
  const SumPlan p = sum_plan(b.B, b.Hq, b.Hkv, b.T, b.D, b.Sk, b.kind == kMaskCausal, two, attend);
  const int64_t units = (int64_t)b.B * b.Hkv;
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
  a.key_blocks = (int)p.key_blocks; a.chunks = (int)p.chunks; a.chunk_tiles = (int)p.chunk_tiles;
  char* w = (char*)workspace;
  a.qi.img = (uint4*)w;
  w += p.img;
  a.qi.unit = (float*)w;
  w += p.unit;
  a.qi.odd = (int*)w;
  a.qi.blocks = (int)p.q_blocks;
  w += p.odd;
  a.stats = (float2*)w;
  w += p.stats;
  a.part = (float2*)w;
  a.sums = (float*)w;
  a.weights = weights;
  a.w_b = ws[0]; a.w_h = ws[1]; a.w_k = ws[2];
  if (attend) {
    RowsArgs r = {};
    fill_block_mfma(&r.m, b);
    r.m.b.stats = a.stats;
    r.m.ws_ml = (float2*)w;
    r.m.ws_o = (float*)(w + p.rows.ml_bytes);
    r.qi = a.qi;
    const int rc = launch_rows(r, p.rows, st);
    if (rc != KVQ_OK) return rc;
  }
  if (b.Sk == 0) return KVQ_OK;
  if (b.D == 128) two ? launch_sums<128, true>(a, !attend, st) : launch_sums<128, false>(a, !attend, st);
  else two ? launch_sums<64, true>(a, !attend, st) : launch_sums<64, false>(a, !attend, st);
  return KVQ_OK;
}

}  // namespace kvq
