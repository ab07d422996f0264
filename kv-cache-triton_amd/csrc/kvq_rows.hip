// Attention of many query rows over the INT4 cache on the matrix cores
// (gfx950): trees of more than rows_min rows per KV head, and the blocks whose key
// weights are counted but for those of few rows, for 16-bit queries and scales, D 64
// and 128, aligned rows.
//
// A wave takes 32 query rows, a workgroup of NW waves 32 NW rows of one KV head
// and a split of the keys. Each 64-key tile is decoded once per workgroup, into
// LDS images in the order the matrix operands are read, and every wave reads
// them from there (conflict-free 16-byte reads). v_mfma 32x32x16, fp16 operands:
//   S^T = K Q^T, O^T += V^T P^T.
// Scores are exact to fp32's rounding: fp16 scales take two products
// (kvq_operands.h). Scales enter times one power of two for the keys and one for
// the values; the rare key whose scale fp16 does not hold even so has its score,
// or its share of the output, formed in fp32. Values times fp16 scales, and the
// weights, are rounded to fp16 (2^-12, near the output's own rounding or under it).
//
// In iteration i a wave's matrix instructions and vector work come in two pairs
// that do not wait for each other: S(i) with the decoding of tile i + 1's keys
// and tile i's values, and the softmax of S(i) with the products of tile i - 1's
// weights. Neither pair has a branch in it, so that they are one stream of
// instructions: matrix instructions hide the vector work of their own wave only.
//
// Bound by the sum of matrix cycles (44 %) and vector cycles (56 %: decoding,
// 32 exponentials and about 200 other instructions a wave and tile), which hardly
// overlap between the waves of a SIMD. Measured: 404 rows of 16 heads over 30K
// fp16 keys 172 us (577 TFLOP/s; 141 with one term a score), 8 heads of a causal
// 4K prompt 160 us (859 TFLOP/s); before the interleaving and with branches in
// the loop the former took 238. A launch of one tile takes 15 us: four dependent
// round trips and the fetch of its instructions, so the prologue is rolled up.
// 256 rows a workgroup halve the decoding of 128, for one workgroup per CU.
//
// Layout (lane l: n = l % 32, g = l / 32): a lane holds, of query row n, keys
// 8 (r / 4) + 4 g + r % 4 of a 32-key block in register r; registers 8 h .. 8 h + 7
// of block kb are the B operand of 16-key step t = 2 kb + h, and the value image
// has its keys in that order: 16 t + 4 g + e % 4 + 8 (e / 4).

#include <algorithm>

#include "kvq_operands.h"

namespace kvq {
namespace {

constexpr int kTile = 64;
constexpr float kNeg = -1.0e30f;
constexpr float kLazyMax = 8.0f;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// SUMS: for key weights, the query operands are kept, and the softmax sums the
// weights as they are. Else, with bf16 scales (whose values are exact in fp16), it
// sums the rounded weights that the products take, two in an instruction.
template <int D, bool QF16, bool SF16, bool SUMS, int NW, bool PAGED>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2)))
void rows_attn_kernel(const RowsArgs a) {
  constexpr bool TWO = SF16;
  constexpr int NT = 64 * NW, ROWS = 32 * NW;
  constexpr int KS = D / 16;           // 16-dim steps of S^T
  constexpr int NDB = D / 32;          // 32-dim blocks of O^T
  constexpr int NC = D / 32;           // 32-dim chunks
  constexpr int IMG = 8 * D;           // 16-byte pieces of a key (per term) or value image
  constexpr int KPW = D / 8 / NW;      // code words of a key that a thread decodes
  constexpr int DPT = 8 * D / NT;      // value dims of eight keys that a thread decodes
  constexpr uint32_t ROW = D / 2;      // bytes of a row's codes
  __shared__ __align__(16) uint4 k_img[2][(TWO ? 2 : 1) * IMG];
  __shared__ __align__(16) uint4 v_img[2][IMG];
  __shared__ __align__(16) _Float16 v_sc[2][NW][kTile];  // value scales of chunk w % NC, keys in the images' order
  __shared__ __align__(16) uint64_t odd_keys[2][2 * NW]; // per wave: keys left out of the key image, of the value image
  __shared__ float tops[2 * NW];

  const BlockArgs& ab = a.m.b;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, g = lane >> 5;
  // (unit fastest: a head's row blocks and splits share an XCD and its L2; row
  // blocks with the most keys first)
  const int unit = blockIdx.x, blk = a.m.row_chunks - 1 - (int)blockIdx.y, sp = blockIdx.z;
  const int kvh = unit % ab.Hkv, b = unit / ab.Hkv;
  const int rows = ab.ratio * ab.T, len = (int)block_len(ab, b), base = len - ab.T;
  // Keys that row i of the block attends (a tree's: may attend): [0, limit).
  auto limit = [&](int i) { return ab.kind != kMaskCausal ? len : max(base + i + 1, 0); };
  const int tiles = (limit((min((blk + 1) * ROWS, rows) - 1) / ab.ratio) + kTile - 1) / kTile;
  const int lo = (int)((uint32_t)tiles * (uint32_t)sp / (uint32_t)a.m.n_split);
  const int hi = (int)((uint32_t)tiles * (uint32_t)(sp + 1) / (uint32_t)a.m.n_split);

  const int R0 = blk * ROWS + wave * 32, R = R0 + n;
  const int row_i = min(R, rows - 1) / ab.ratio, head = kvh * ab.ratio + (min(R, rows - 1) - row_i * ab.ratio);
  // keys that every row of the wave attends
  int lim_wave = R0 < rows ? limit(R0 / ab.ratio) : 0x7fffffff;
  if (ab.kind == kMaskTree) lim_wave = min(lim_wave, max(base, 0));

  // ---- tiles: first cache row and rows of tile t ----
  const uint8_t* kp = ab.kp + b * ab.kps_b + kvh * ab.kps_h;
  const uint8_t* vp = ab.vp + b * ab.vps_b + kvh * ab.vps_h;
  const uint16_t* ks = (const uint16_t*)ab.ks + b * ab.kss_b + kvh * ab.kss_h;
  const uint16_t* vs = (const uint16_t*)ab.vs + b * ab.vss_b + kvh * ab.vss_h;
  const int ng = a.m.ng;
  const uint32_t srow = 2u * (uint32_t)ng;
  const int32_t* bt = PAGED ? ab.pm.table + (int64_t)b * ab.pm.tab_stride : nullptr;
  auto row_of = [&](int t, uint32_t* n_rows) -> int64_t {
    int64_t r0 = (int64_t)t * kTile;
    bool there = t < hi;
    if constexpr (PAGED) {
      const int64_t pg = min(r0 >> ab.pm.page_shift, (int64_t)ab.pm.n_pages - 1);
      const int32_t blkid = __builtin_amdgcn_readfirstlane(bt[pg]);
      there = there && blkid >= 0 && blkid < ab.pm.n_blocks;
      r0 = ((int64_t)blkid << ab.pm.page_shift) | (r0 & ((int64_t(1) << ab.pm.page_shift) - 1));
    }
    *n_rows = there ? (uint32_t)min(kTile, len - t * kTile) : 0u;
    return there ? r0 : 0;
  };

  // keys: thread (key tid % 64, part tid / 64) decodes KPW words, all of one scale
  const int part = wave;
  const uint32_t k_at = lane * ROW + 4 * KPW * part;
  const uint32_t ks_at = lane * srow + 2u * (uint32_t)((8 * KPW * part / 32) * ng / NC);
  uint32_t kraw[KPW], ks_raw;
  auto load_keys = [&](int64_t r0, uint32_t nr) {
    const __amdgpu_buffer_rsrc_t rk = rsrc_of(kp + r0 * ROW, nr * ROW);
    if constexpr (KPW == 4) {
      const uint4 v = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_at, 0, 0));
      kraw[0] = v.x; kraw[1] = v.y; kraw[2] = v.z; kraw[3] = v.w;
    } else if constexpr (KPW == 2) {
      const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rk, k_at, 0, 0));
      kraw[0] = v.x; kraw[1] = v.y;
    } else {
      kraw[0] = __builtin_amdgcn_raw_buffer_load_b32(rk, k_at, 0, 0);
    }
    ks_raw = __builtin_amdgcn_raw_buffer_load_b16(rsrc_of((const uint8_t*)ks + r0 * srow, nr * srow), ks_at, 0, 0) & 0xffffu;
  };
  float k_unit = 1.0f, v_unit = 1.0f;
  auto scale_f32 = [&](uint32_t x) { return SF16 ? f16_bits_to_f32(x) : bf16_bits_to_f32(x); };
  _Float16 k_scale;
  auto key_scale = [&](int buf) {
    const float sf = scale_f32(ks_raw) * k_unit;
    const bool odd = scale_odd(sf);
    k_scale = (_Float16)(odd ? 0.0f : sf);
    odd_keys[buf][wave] = __builtin_amdgcn_ballot_w64(odd);
  };
  uint4* const k_dst = k_img[0] + (lane >> 5) * KS * 64 + (lane & 31);
  auto key_word = [&](int buf, int j) {  // dims 8 piece .. + 7: step piece / 2, half piece % 2
    const int piece = KPW * part + j;
    uint4 rest;
    uint4* dst = k_dst + buf * (TWO ? 2 : 1) * IMG + (piece >> 1) * 64 + 32 * (piece & 1);
    *dst = decode<TWO, !SF16>(kraw[j], k_scale, &rest);
    if constexpr (TWO) dst[IMG] = rest;
  };
  // values: thread (eight keys 16 t + 4 gg + e % 4 + 8 (e / 4), dims d0 .. d0 + DPT - 1)
  constexpr int DG = D / DPT;  // threads of the same eight keys
  const int v_c8 = tid / DG, v_d0 = (tid % DG) * DPT;
  const uint32_t v_at = (16 * (v_c8 >> 1) + 4 * (v_c8 & 1)) * ROW + v_d0 / 2;
  uint32_t vraw[8], vs_raw;
  auto load_values = [&](int64_t r0, uint32_t nr) {
    const __amdgpu_buffer_rsrc_t rv = rsrc_of(vp + r0 * ROW, nr * ROW);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t at = v_at + ((e & 3) + 8 * (e >> 2)) * ROW;
      if constexpr (DPT == 4) vraw[e] = __builtin_amdgcn_raw_buffer_load_b16(rv, at, 0, 0);
      else vraw[e] = __builtin_amdgcn_raw_buffer_load_b8(rv, at, 0, 0);
    }
  };
  // Dim d of the 32 of a block lies at piece value_at(d): the pieces that eight
  // lanes of a wave store at once then lie in all banks.
  auto value_at = [](int d) { return DPT == 4 ? d ^ ((d >> 4) & 1) ^ ((d >> 2) & 2) : DPT == 2 ? d ^ ((d >> 4) & 1) : d; };
  uint4* const v_dst = v_img[0] + ((v_d0 >> 5) * 4 + (v_c8 >> 1)) * 64 + 32 * (v_c8 & 1);
  uint32_t vy[4];
  CodeScale v_cs[4];
  auto value_codes = [&](int buf) {
    const uint4 sc = *(const uint4*)(v_sc[buf][v_d0 / 32] + 8 * v_c8);
    const uint32_t scp[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      vy[p] = __builtin_amdgcn_perm(vraw[2 * p + 1], vraw[2 * p], 0x05040100u);
      if constexpr (DPT == 1) vy[p] = (vy[p] >> (4 * (v_d0 & 1)));
      v_cs[p] = code_scale<!SF16>(scp[p]);
    }
  };
  auto value_dim = [&](int buf, int d) {
    uint32_t w[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) w[p] = code_pair<!SF16>(vy[p], 4 * d, v_cs[p]);
    v_dst[buf * IMG + value_at((v_d0 & 31) + d)] = make_uint4(w[0], w[1], w[2], w[3]);
  };
  // value scales: wave w takes chunk w % NC of all keys
  const uint32_t vs_at = lane * srow + 2u * (uint32_t)((wave % NC) * ng / NC);
  const int v_pos = 8 * (2 * (lane >> 4) + ((lane >> 2) & 1)) + 4 * ((lane >> 3) & 1) + (lane & 3);
  auto load_v_scales = [&](int64_t r0, uint32_t nr) {
    vs_raw = __builtin_amdgcn_raw_buffer_load_b16(rsrc_of((const uint8_t*)vs + r0 * srow, nr * srow), vs_at, 0, 0) & 0xffffu;
  };
  auto store_v_scales = [&](int buf) {
    const float s = scale_f32(vs_raw) * v_unit;
    const bool odd = scale_odd(s);
    v_sc[buf][wave][v_pos] = (_Float16)(odd ? 0.0f : s);
    odd_keys[buf][NW + wave] = __builtin_amdgcn_ballot_w64(odd);
  };

  f32x16_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[db][j] = 0.0f;
  float m_run = kNeg, l_run = 0.0f;
  uint4 p[4];  // weights of the tile before

  int64_t r0_cur = 0, r0_next = 0, r0_after = 0;  // first rows of tiles i, i + 1, i + 2
  uint32_t nr_cur = 0, nr_next = 0, nr_after = 0;

  if (lo < hi) {
    r0_cur = row_of(lo, &nr_cur);
    r0_next = row_of(lo + 1, &nr_next);
    r0_after = row_of(lo + 2, &nr_after);
    load_keys(r0_cur, nr_cur);
    load_v_scales(r0_cur, nr_cur);
    load_values(r0_cur, nr_cur);
  }

  // ---- queries (on their way with the first tile): lane (n, g) holds dims
  // 16 kk + 8 g .. + 7 of its row ----
  uint4 q[KS];
  float cr, q_unit;
  bool q_odd = false;
  {
    const uint16_t* p = (const uint16_t*)ab.q + b * ab.qs_b + (int64_t)head * ab.qs_h + (int64_t)row_i * ab.qs_s + 8 * g;
    q_unit = query_operand<QF16, KS>(p, a.m.q_vec, ab.scale_log2 < 0.0f, q, &q_odd);
    q_odd = __builtin_amdgcn_ballot_w64(q_odd) != 0;
    if (SUMS && sp == 0 && R0 < rows) {
      const int64_t block = (int64_t)unit * a.qi.blocks + R0 / 32;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) a.qi.img[(block * KS + kk) * 64 + lane] = q[kk];
      if (lane == 0) a.qi.odd[block] = q_odd;
      if (g == 0 && R < rows) a.qi.unit[(int64_t)unit * rows + R] = q_unit;
    }
  }

  if (lo < hi) {
    {  // the powers of two of the scales, from the first tile's
      float tk = fabsf(scale_f32(ks_raw)), tv = fabsf(scale_f32(vs_raw));
      tk = tk < __builtin_inff() ? tk : 0.0f;
      tv = tv < __builtin_inff() ? tv : 0.0f;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) {
        tk = fmaxf(tk, __shfl_xor(tk, d));
        tv = fmaxf(tv, __shfl_xor(tv, d));
      }
      tops[wave] = tk;
      tops[NW + wave] = tv;
    }
    const uint4 zero4 = make_uint4(0u, 0u, 0u, 0u);
    for (int j = tid; j < IMG; j += NT) v_img[1][j] = zero4;  // "tile lo - 1": weights 0 times finite values
#pragma unroll
    for (int t = 0; t < 4; ++t) p[t] = zero4;
    __syncthreads();
    float tk = 0.0f, tv = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      tk = fmaxf(tk, tops[w]);
      tv = fmaxf(tv, tops[NW + w]);
    }
    k_unit = value_unit(tk);
    v_unit = value_unit(tv);
    key_scale(0);
#pragma unroll
    for (int j = 0; j < KPW; ++j) key_word(0, j);
    store_v_scales(0);
    load_keys(r0_next, nr_next);
    load_v_scales(r0_next, nr_next);
    __syncthreads();
  }
  cr = fmaxf(fabsf(ab.scale_log2), 1.0e-30f) / (q_unit * k_unit);

  const int v_lane = 32 * g + value_at(n);
  // what a step does between its first matrix instructions, one item at a time
  constexpr int ITEMS = KPW + DPT + 4;
  auto item = [&](int x, int par) {
    if (x == 0) key_scale(par ^ 1);
    else if (x <= KPW) key_word(par ^ 1, x - 1);
    else if (x == KPW + 1) value_codes(par);
    else if (x <= KPW + 1 + DPT) value_dim(par, x - KPW - 2);
    else if (x == KPW + DPT + 2) store_v_scales(par ^ 1);
    else {
      load_keys(r0_after, nr_after);
      load_values(r0_next, nr_next);
      load_v_scales(r0_after, nr_after);
    }
  };

#pragma unroll 1
  for (int i = lo; i < hi; ++i) {
    const int par = (i - lo) & 1;
    // ---- S(i), while tile i's values and tile i + 1's keys are decoded ----
    const uint4* kt = k_img[par] + lane;
    const uint64_t odd_lane = odd_keys[par][lane & (2 * NW - 1)];
    f32x16_t s[2];
    {
      constexpr int T2 = TWO ? 2 : 1;
      uint4 f[2][2 * T2];  // a step's operands, read a step ahead
      auto read = [&](int kk, uint4 (&x)[2 * T2]) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int t = 0; t < T2; ++t) x[kb * T2 + t] = kt[t * IMG + (kb * KS + kk) * 64];
      };
      read(0, f[0]);
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        if (kk + 1 < KS) read(kk + 1, f[(kk + 1) & 1]);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int t = 0; t < T2; ++t) {
            f32x16_t zero;
#pragma unroll
            for (int j = 0; j < 16; ++j) zero[j] = 0.0f;
            s[kb] = mfma(f[kk & 1][kb * T2 + t], q[kk], kk == 0 && t == 0 ? zero : s[kb]);
          }
#pragma unroll
        for (int x = 0; x < ITEMS; ++x)
          if (x * KS / ITEMS == kk) item(x, par);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const uint64_t odd_waves = __builtin_amdgcn_ballot_w64(odd_lane != 0);  // bit w: keys, NW + w: values
    const int t0 = i * kTile;
    if (t0 + kTile > lim_wave || nr_cur == 0 || q_odd || (odd_waves & ((1u << NW) - 1)) != 0) {
      // (nothing of the rare path is computed or loaded ahead, in registers of the loop)
      int gc = g;
      auto again = (const __attribute__((address_space(4))) RowsArgs*)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+v"(gc), "+s"(again));
      const auto& cb = again->m.b;
      // ---- keys whose scale the image does not hold: one at a time ----
      uint64_t left = 0;
      for (int w = 0; w < NW; ++w) left |= odd_keys[par][w];
      left = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(left >> 32)) << 32) |
             (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)left);
#pragma unroll 1
      while (left != 0) {
        const int k = __builtin_ctzll(left);
        left &= left - 1;
        float dot = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          const uint32_t w = *(const uint32_t*)(kp + (r0_cur + k) * ROW + 8 * kk + 4 * gc);
          uint32_t qw[4] = {q[kk].x, q[kk].y, q[kk].z, q[kk].w};
          asm volatile("" : "+v"(qw[0]), "+v"(qw[1]), "+v"(qw[2]), "+v"(qw[3]));
          float part_dot = 0.0f;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            part_dot = fmaf((float)((int)((w >> (4 * x)) & 15u) - 8), f16_bits_to_f32(qw[x] & 0xffffu), part_dot);
            part_dot = fmaf((float)((int)((w >> (4 * x + 16)) & 15u) - 8), f16_bits_to_f32(qw[x] >> 16), part_dot);
          }
          dot = fmaf(part_dot, scale_f32(ks[(r0_cur + k) * ng + (kk / 2) * ng / NC]) * k_unit, dot);
        }
        const float v = pair_sum(dot);
#pragma unroll
        for (int x = 0; x < 32; ++x)
          if (x == 16 * (k >> 5) + 4 * ((k & 31) >> 3) + (k & 3) && gc == ((k >> 2) & 1)) s[x >> 4][x & 15] = v;
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[kb][j] = block_score(s[kb][j]);
      // ---- masks ----
      uint32_t seen = 0u;
      if (nr_cur > 0) {
        if (cb.kind == kMaskTree) {
          // (clamped loads without conditions: sixteen in flight)
          const uint8_t* mrow = cb.mask + b * cb.ms_b + (int64_t)row_i * cb.ms_i;
          const int64_t ms_t = cb.ms_t;
          const int T = cb.T;
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            uint32_t on = 0u;
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              const int k = t0 + 32 * x + 8 * (y >> 2) + 4 * gc + (y & 3), t = k - base;
              const uint8_t set = mrow[(int64_t)min(max(t, 0), T - 1) * ms_t];
              on |= k < len && (t < 0 || set != 0) ? 1u << y : 0u;
            }
            seen |= on << (16 * x);
          }
        } else {
          const int lim = limit(row_i);
#pragma unroll
          for (int x = 0; x < 32; ++x)
            seen |= t0 + 32 * (x >> 4) + 8 * ((x >> 2) & 3) + 4 * gc + (x & 3) < lim ? 1u << x : 0u;
        }
      }
#pragma unroll
      for (int x = 0; x < 32; ++x)
        if (!((seen >> x) & 1u)) s[x >> 4][x & 15] = -__builtin_inff();
    }
    // ---- softmax of S(i), with the products of tile i - 1's weights ----
    constexpr int NM = 4 * NDB, MAXES = NM / 4;
    const uint4* vt = v_img[par ^ 1] + v_lane;
    float mx = -__builtin_inff(), alpha = 1.0f, ls = l_run;
    bool grow = false;
    uint4 pc[4];
    uint4 vf[2][2];  // operands, read two products ahead
    vf[0][0] = vt[0];
    vf[0][1] = vt[256];
#pragma unroll
    for (int x = 0; x < NM; ++x) {  // product x: 16-key step x / NDB, 32-dim block x % NDB
      if (x % 2 == 0 && x + 2 < NM) {
        vf[(x / 2 + 1) & 1][0] = vt[(((x + 2) % NDB) * 4 + (x + 2) / NDB) * 64];
        vf[(x / 2 + 1) & 1][1] = vt[(((x + 3) % NDB) * 4 + (x + 3) / NDB) * 64];
      }
      o[x % NDB] = mfma(vf[(x / 2) & 1][x & 1], p[x / NDB], o[x % NDB]);
      if (x < MAXES) {
#pragma unroll
        for (int j = 0; j < 32 / MAXES; j += 2) {
          const int e = x * (32 / MAXES) + j;
          mx = fmaxf(fmaxf(mx, s[e >> 4][e & 15]), s[e >> 4][(e & 15) + 1]);
        }
      } else if (x == MAXES) {
        const float mt = pair_max(mx) * cr;
        grow = __builtin_amdgcn_ballot_w64(mt > m_run + kLazyMax) != 0;
        const float m_new = grow ? fmaxf(m_run, mt) : m_run;
        alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        ls *= alpha;
      } else {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
          if (MAXES + 1 + w * (NM - MAXES - 1) / 16 != x) continue;
          const int kb = w >> 3, r = 2 * (w & 7);
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], cr, -m_run));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r + 1], cr, -m_run));
          const f16x2_t h = {(_Float16)e0, (_Float16)e1}, one = {(_Float16)1.0f, (_Float16)1.0f};
          if constexpr (SUMS || SF16) ls += e0 + e1;
          else ls = __builtin_amdgcn_fdot2(h, one, ls, false);
          ((uint32_t*)&pc[w >> 2])[w & 3] = u32_of(h);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l_run = ls;
#pragma unroll
    for (int t = 0; t < 4; ++t) p[t] = pc[t];
    if (grow || (odd_waves >> NW) != 0) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= alpha;
      // ---- keys whose value scale the image does not hold: one at a time ----
      int gc = g;
      asm volatile("" : "+v"(gc));
      uint64_t left = 0;
      for (int w = 0; w < NW; ++w) left |= odd_keys[par][NW + w];
      left = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(left >> 32)) << 32) |
             (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)left);
#pragma unroll 1
      while (left != 0) {
        const int k = __builtin_ctzll(left);
        left &= left - 1;
        // its weight: lane n + 32 ((k / 4) % 2), half k % 2 of word (k % 16) / 8 * 2 + (k % 4) / 2 of step k / 16
        uint32_t pw = 0u;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t w[4] = {p[t].x, p[t].y, p[t].z, p[t].w};
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (4 * t + x == 4 * (k >> 4) + 2 * ((k >> 3) & 1) + ((k >> 1) & 1)) pw = w[x];
        }
        pw = __shfl(pw, (lane & 31) + 32 * ((k >> 2) & 1));
        const float pk = f16_bits_to_f32((k & 1) ? pw >> 16 : pw & 0xffffu);
        const uint8_t* vrow = vp + (r0_cur + k) * ROW;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          float sf = scale_f32(vs[(r0_cur + k) * ng + db * ng / NC]) * v_unit;
          sf = (pk > 0.0f) & scale_odd(sf) ? sf : 0.0f;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t w = *(const uint16_t*)(vrow + 16 * db + 4 * x + 2 * gc);
#pragma unroll
            for (int y = 0; y < 4; ++y)
              o[db][4 * x + y] = fmaf(pk, (float)((int)((w >> (4 * y)) & 15u) - 8) * sf, o[db][4 * x + y]);
          }
        }
      }
    }
    r0_cur = r0_next; nr_cur = nr_next;
    r0_next = r0_after; nr_next = nr_after;
    r0_after = row_of(i + 3, &nr_after);
    __syncthreads();
  }
  if (lo < hi) {
    const uint4* vt = v_img[(hi - 1 - lo) & 1] + v_lane;
#pragma unroll
    for (int x = 0; x < 4 * NDB; ++x) o[x % NDB] = mfma(vt[((x % NDB) * 4 + x / NDB) * 64], p[x / NDB], o[x % NDB]);
  }

  // lane (n, g) holds dims 32 db + 8 x + 4 g .. + 3 of its row in registers 4 x .. + 3 of block db
  const float l = pair_sum(l_run);
  if (R >= rows) return;
  if (a.m.n_split > 1) {
    const float f = 1.0f / v_unit;
    const int64_t slot = ((int64_t)unit * rows + R) * a.m.n_split + sp;
    if (g == 0) a.m.ws_ml[slot] = make_float2(m_run, l);
    float* dst = a.m.ws_o + slot * D + 4 * g;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *(float4*)(dst + 32 * db + 8 * x) =
            make_float4(o[db][4 * x] * f, o[db][4 * x + 1] * f, o[db][4 * x + 2] * f, o[db][4 * x + 3] * f);
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f, f = inv / v_unit;
  if (ab.stats && g == 0) ab.stats[(int64_t)unit * rows + R] = make_float2(m_run, inv);
  uint16_t* dst = (uint16_t*)ab.out + b * ab.os_b + (int64_t)head * ab.os_h + (int64_t)row_i * ab.os_s + 4 * g;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t w[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float v0 = o[db][4 * x + 2 * y] * f, v1 = o[db][4 * x + 2 * y + 1] * f;
        if constexpr (QF16) {
          const f16x2_t v = {(_Float16)v0, (_Float16)v1};
          w[y] = __builtin_bit_cast(uint32_t, v);
        } else {
          const bf16x2_t v = {(__bf16)v0, (__bf16)v1};
          w[y] = __builtin_bit_cast(uint32_t, v);
        }
      }
      uint16_t* at = dst + 32 * db + 8 * x;
      if (a.m.o_vec) {
        *(uint2*)at = make_uint2(w[0], w[1]);
      } else {
        at[0] = (uint16_t)w[0]; at[1] = (uint16_t)(w[0] >> 16);
        at[2] = (uint16_t)w[1]; at[3] = (uint16_t)(w[1] >> 16);
      }
    }
}

template <int D, bool QF16, bool SF16, bool SUMS, int NW>
void launch(const RowsArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.m.n_units, (unsigned)a.m.row_chunks, (unsigned)a.m.n_split), block(64 * NW);
  if constexpr (!SUMS)
    if (a.m.b.pm.paged) {
      hipLaunchKernelGGL((rows_attn_kernel<D, QF16, SF16, SUMS, NW, true>), grid, block, 0, st, a);
      return;
    }
  hipLaunchKernelGGL((rows_attn_kernel<D, QF16, SF16, SUMS, NW, false>), grid, block, 0, st, a);
}

template <int D, bool QF16, bool SF16>
void launch_waves(const RowsArgs& a, int nw, hipStream_t st) {
  if (a.qi.img) launch<D, QF16, SF16, true, 8>(a, st);
  else if (SF16 || nw == 8) launch<D, QF16, SF16, false, 8>(a, st);
  else if constexpr (!SF16) launch<D, QF16, SF16, false, 4>(a, st);
}

template <int D>
void launch_types(const RowsArgs& a, int nw, hipStream_t st) {
  const bool q16 = a.m.b.q_dt == KVQ_F16;
  if (a.m.s_f16) q16 ? launch_waves<D, true, true>(a, nw, st) : launch_waves<D, false, true>(a, nw, st);
  else q16 ? launch_waves<D, true, false>(a, nw, st) : launch_waves<D, false, false>(a, nw, st);
}

}  // namespace

RowsPlan rows_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool s_f16, bool weights) {
  const int64_t rows = T * (Hq / Hkv), units = B * Hkv, tiles = (Sk + kTile - 1) / kTile;
  RowsPlan p;
  // eight waves (256 rows, one workgroup per CU), or four, two workgroups per
  // CU, where eight would leave four without rows. Key weights are of prompts,
  // with rows enough, and two terms take the LDS of eight waves' workgroup.
  p.nw = weights || s_f16 || (rows + 127) / 128 % 2 == 0 || rows > 1024 ? 8 : 4;
  p.row_chunks = (rows + 32 * p.nw - 1) / (32 * p.nw);
  // the split with the least estimate, in tiles' times (2.2 us): rounds of the
  // workgroups that are resident together, each its tiles and about six tiles'
  // time of prologue and epilogue; the partials' traffic (33 MB in 14 us) and a
  // merge's launch
  const int64_t wgs = units * p.row_chunks, slots = p.nw == 8 ? 256 : 512;
  p.n_split = 1;
  double best = 0.0;
  for (int64_t ns = 1; ns <= std::min<int64_t>(64, std::max<int64_t>(1, tiles / 4)); ++ns) {
    const double rounds = (double)((wgs * ns + slots - 1) / slots);
    const double cost = rounds * ((double)((tiles + ns - 1) / ns) + 6.0) +
                        (ns > 1 ? 2.5 + (double)(units * rows * ns) * (double)D / 1.2e6 : 0.0);
    if (ns == 1 || cost < best) {
      best = cost;
      p.n_split = ns;
    }
  }
  p.ml_bytes = p.o_bytes = 0;
  if (p.n_split > 1) {
    p.ml_bytes = (units * rows * p.n_split * 8 + 255) / 256 * 256;
    p.o_bytes = units * rows * p.n_split * D * 4;
  }
  return p;
}

int launch_rows(RowsArgs a, const RowsPlan& p, hipStream_t st) {
  if (p.row_chunks >= 65536 || a.m.b.Sk >= (int64_t(1) << 31)) return KVQ_EUNSUP;
  a.m.row_chunks = (int)p.row_chunks;
  a.m.n_split = (int)p.n_split;
  if (a.m.b.D == 128) launch_types<128>(a, p.nw, st);
  else launch_types<64>(a, p.nw, st);
  if (p.n_split > 1) launch_block_merge(a.m, st);
  return KVQ_OK;
}

}  // namespace kvq
