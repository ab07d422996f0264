// Arguments shared by the tree-attention and key-weight kernels
// (kvq_tree.hip, kvq_weights.hip): a block of T query rows over cached K/V,
// contiguous or paged, with the masks a block takes.
#pragma once

#include "kvq_common.h"

namespace kvq {

// Which of a sequence's len keys query row i of the block attends. The block's
// own rows are the last T keys (key len - T + t is row t's):
//   kMaskNone    every key
//   kMaskCausal  the keys before the block and those of rows t <= i
//   kMaskTree    the keys before the block and those of rows t with
//                mask[b][i][t] != 0
enum { kMaskNone = 0, kMaskCausal = 1, kMaskTree = 2 };

struct BlockArgs {
  const void* q;
  int64_t qs_b, qs_h, qs_s, qs_d;  // element strides
  const uint8_t* kp;
  int64_t kps_b, kps_h, kps_s;  // byte strides
  const void* ks;
  int64_t kss_b, kss_h, kss_s;  // element strides
  const uint8_t* vp;
  int64_t vps_b, vps_h, vps_s;
  const void* vs;
  int64_t vss_b, vss_h, vss_s;
  PageMap pm;  // (paged: batch strides 0)
  const uint8_t* mask;
  int64_t ms_b, ms_i, ms_t;
  void* out;
  int64_t os_b, os_h, os_s, os_d;
  // [B, Hkv, row] (m, 1 / l) of each row, weight j = 2^(s_j - m) / l, or null. A row
  // with no key has 1 / l = 0. The pair, not m + log2 l: at
  // scores in the thousands the sum's rounding alone is 2^-12 of a weight.
  float2* stats;
  const int32_t* seq_lens;
  int64_t Sk;
  int q_dt, s_dt, kind;
  int B, Hq, Hkv, ratio, T, D, G;
  float scale_log2;  // sm_scale * log2(e)
};

// Where `stats` has query row i of head h: row i * ratio + h % ratio of the KV head.
__device__ __forceinline__ int64_t stats_at(const BlockArgs& a, int b, int h, int i) {
  return ((int64_t)b * a.Hkv + h / a.ratio) * a.ratio * a.T + (int64_t)i * a.ratio + h % a.ratio;
}

// Keys of sequence b: its device length clamped to [0, Sk], or Sk.
__device__ __forceinline__ int64_t block_len(const BlockArgs& a, int b) {
  if (!a.seq_lens) return a.Sk;
  const int64_t n = a.seq_lens[b];
  return n < 0 ? 0 : (n > a.Sk ? a.Sk : n);
}

// Whether row i of sequence b attends key t of the block's own rows.
__device__ __forceinline__ bool block_sees(const BlockArgs& a, int b, int i, int64_t t) {
  if (a.kind == kMaskTree) return a.mask[b * a.ms_b + i * a.ms_i + t * a.ms_t] != 0;
  return a.kind == kMaskNone || t <= i;
}

// A score as the softmax takes it: NaN weighs nothing, and infinities are held
// at finite values far outside any other score, so that no difference of two
// scores is NaN.
__device__ __forceinline__ float block_score(float s) {
  return s == s ? fminf(fmaxf(s, -1.0e30f), 1.0e30f) : -__builtin_inff();
}

// Element d of a packed row: code - 8, exact in fp32.
__device__ __forceinline__ float code_at(const uint8_t* row, int d, int G) {
  const int g = d / G, e = d - g * G;
  const uint32_t byte = row[g * ((G + 1) / 2) + (e >> 1)];
  return (float)((int)((e & 1) ? byte >> 4 : byte & 15u) - 8);
}

struct BlockPaged {
  const int32_t* bt;
  int64_t bt_stride, bt_cols, n_blocks, page_size;
};

// Checks shared by the entry points, and the arguments they fill in; KVQ_OK,
// or a status with the error set. `what` names the entry point. Paged calls
// pass pool strides (head, row), contiguous ones (batch, head, row); v_* are
// null where the values are not read.
int fill_block_args(BlockArgs* a, const char* what, const void* q, int q_dtype, const int64_t* q_strides,
                    const void* k_packed, const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides,
                    const void* v_packed, const int64_t* vp_strides, const void* v_scales, const int64_t* vs_strides,
                    int scale_dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t group_size,
                    const int32_t* seq_lens, int64_t Sk, float sm_scale, const BlockPaged* pg);

// The plain kernel of kvq_tree.hip: one workgroup per query row, any dtype,
// group size and head dim up to kMaxBlockD. Writes a.out (unless null) and
// a.stats (unless null).
constexpr int kMaxBlockD = 256;
void launch_block_rows(const BlockArgs& a, hipStream_t st);

}  // namespace kvq
