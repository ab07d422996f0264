// The matrix-core kernel of kvq_block.hip: its arguments, plan and launch.
#pragma once

#include "kvq_block.h"

namespace kvq {

struct BlockMfmaArgs {
  BlockArgs b;
  int n_units, row_chunks, n_split;  // unit = batch * Hkv + KV head
  int ng, s_f16;                     // scales of a cache row; whether they are fp16
  int q_vec, o_vec;                  // 16-byte query pieces, 8-byte output pieces
  int tiles_max;
  float2* ws_ml;  // [unit][row][split] (max, sum)
  float* ws_o;    // [unit][row][split][D] unnormalised
  // key weights: scores in log2 units ([unit][tile][row][64], the keys of a
  // tile in the order 16 kb + g + 4 j at 16 kb + 4 g + j), or null, and the sums
  float* scores;
  float* weights;
  int64_t w_b, w_h, w_k;
};

constexpr int kMaxScoreRows = 32;  // query rows per KV head of a launch that keeps its scores

struct BlockPlan {
  int rb, nw;  // 16-row blocks a wave, waves a workgroup
  int64_t row_chunks, n_split, ml_bytes, o_bytes;
};

BlockPlan block_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk);

// Whether the matrix-core kernels take these arguments (else the plain ones);
// the first for kernels that read no values.
bool block_mfma_takes_keys(const BlockArgs& a);
bool block_mfma_takes(const BlockArgs& a);

// Attention by the kernel of few rows or of many; without the workspace for its
// split the launch does not split.
int64_t block_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool s_f16);
int launch_block_mfma(const BlockArgs& b, void* workspace, int64_t workspace_bytes, hipStream_t st);

// Attention that keeps its scores, and the key weights from them, for up to
// kMaxScoreRows rows per KV head; workspace bytes (0 for more rows).
int64_t block_scores_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk);
int launch_block_weights(const BlockArgs& b, float* weights, const int64_t* ws, void* workspace, hipStream_t st);

// Merges the splits' partials of a launch that leaves them in ws_ml and ws_o.
void launch_block_merge(const BlockMfmaArgs& a, hipStream_t st);
void fill_block_mfma(BlockMfmaArgs* a, const BlockArgs& b);

// The queries as matrix operands, kept for the key weights' second pass.
struct QueryImages {
  float* unit;  // [unit][row]: the power of two of the row
  uint4* img;   // [unit][32-row block][16-dim step][64]
  int* odd;     // [unit][32-row block]: a query is not finite
  int blocks;
};

// Many rows per KV head (kvq_rows.hip): the arguments of the kernel, its plan
// and launch. With qi.img it keeps the query operands and sums the softmax in
// full precision.
struct RowsArgs {
  BlockMfmaArgs m;
  QueryImages qi;
};

struct RowsPlan {
  int nw;
  int64_t row_chunks, n_split, ml_bytes, o_bytes;
};

// Trees of more rows per KV head than this take it. Where the keys fill the GPU
// it is faster from 65 rows (104 rows of 64 KV heads over 8K keys: 57 against 82
// us by kvq_block.hip), and never by more than 4 us slower (96 rows of 8 heads
// over 16K keys: 34.5 against 33.4; 256 rows: 45 against 54). With fp16 scales,
// two products each: 128 rows of 16 heads over 30K keys 94 against 80 us, 404
// rows 183 against 257.
inline int64_t rows_min(bool s_f16) { return s_f16 ? 128 : 64; }
RowsPlan rows_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool s_f16, bool weights);
int launch_rows(RowsArgs a, const RowsPlan& p, hipStream_t st);

// Key weights of blocks of any length (kvq_sums.hip), for what
// block_mfma_takes_keys takes of a contiguous cache.
// With `attend` the block's attention too, whose statistics the sums then take.
int64_t sums_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, bool s_f16, bool attend);
int launch_key_sums(const BlockArgs& b, bool attend, float* weights, const int64_t* ws, void* workspace, hipStream_t st);

// Dims d .. d + 3 of output row R (row R / ratio of the block, head R % ratio
// of the group), and the row's statistics, from a row's max, sum and
// unnormalised values.
template <bool QF16>
__device__ __forceinline__ void block_store_row(const BlockMfmaArgs& a, int b, int kvh, int R, int d, float m, float l,
                                                float4 o) {
  const int i = R / a.b.ratio, h = kvh * a.b.ratio + R % a.b.ratio;
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  if (a.b.stats && d == 0) a.b.stats[((int64_t)b * a.b.Hkv + kvh) * a.b.ratio * a.b.T + R] = make_float2(m, inv);
  if (!a.b.out) return;
  uint16_t* p = (uint16_t*)a.b.out + b * a.b.os_b + (int64_t)h * a.b.os_h + (int64_t)i * a.b.os_s + d;
  const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = QF16 ? f32_to_f16_bits(v[k]) : f32_to_bf16_bits(v[k]);
  if (a.o_vec) {
    *(uint2*)p = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = (uint16_t)w[k];
  }
}

}  // namespace kvq
