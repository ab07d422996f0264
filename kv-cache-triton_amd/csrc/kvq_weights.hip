// Key weights: how much attention each cached key has drawn (gfx950).
//
//   w[b, kvh, j] += sum over the KV head's query heads h and the block's rows i
//                   of 2^(c s[i, j] - m[i]) / l[i],   c = log2 e,
//                   m[i] = max_j c s[i, j],  l[i] = sum_j 2^(c s[i, j] - m[i])
//
// i.e. the softmax weights of a block of queries, summed over the rows that
// share the KV head, added to a running fp32 sum per key: what an eviction
// ranks the cache's rows by. A key's sum needs every row's m and l, so the
// scores are formed twice, by the same operations in the same order both times
// (a row's weights then add up to 1 however large its scores), or kept:
//   few rows with their attention   scores kept by kvq_block.hip
//   other 16-bit blocks             kvq_rows.hip, then kvq_sums.hip
//   the rest                        the plain kernels (the attention's, and below)
// Sums over rows are taken in a fixed order (no atomics), so equal calls give
// equal bits. The reference has no counterpart.
//
// Kept scores are 4 bytes a row and key, written and read: 134 MB for 8 sequences
// of 32K keys and 64 heads (102 us in all). A second pass over that cache would
// read as much and form the scores again.

#include <algorithm>

#include "kvq_block_mfma.h"

namespace kvq {
namespace {

constexpr int kWKeys = 64;      // keys per workgroup
constexpr int kWThreads = 256;  // four threads per key, each every fourth row

// The plain kernel: the codes and scales of 64 keys in LDS in fp32, every row
// of the KV head scored against them as block_rows_kernel does, with its
// statistics known. Right for every dtype, group size and stride.
__global__ __launch_bounds__(kWThreads) void key_weights_rows_kernel(const BlockArgs a, float* w, int64_t ws_b,
                                                                     int64_t ws_h, int64_t ws_k, int chunks) {
  __shared__ float k_lds[kWKeys * (kMaxBlockD + 1)];
  __shared__ float sums[kWThreads];
  const int tid = threadIdx.x, pitch = a.D + 1;
  const int chunk = blockIdx.x % chunks, unit = blockIdx.x / chunks;
  const int kvh = unit % a.Hkv, b = unit / a.Hkv;
  const int64_t len = block_len(a, b), base = len - a.T, j0 = (int64_t)chunk * kWKeys;
  if (j0 >= len) return;
  const uint8_t* kp = a.kp + b * a.kps_b + kvh * a.kps_h;
  const int64_t ks0 = b * a.kss_b + kvh * a.kss_h;
  for (int x = tid; x < kWKeys * a.D; x += kWThreads) {
    const int key = x / a.D, d = x % a.D;
    const int64_t j = j0 + key;
    k_lds[key * pitch + d] = j < len ? code_at(kp + j * a.kps_s, d, a.G) : 0.0f;
  }
  __syncthreads();
  const int key = tid % kWKeys, part = tid / kWKeys;
  const int64_t j = j0 + key;
  float sum = 0.0f;
  for (int R = part; R < a.ratio * a.T; R += kWThreads / kWKeys) {
    const int i = R / a.ratio, h = kvh * a.ratio + R % a.ratio;
    const float2 st = a.stats[stats_at(a, b, h, i)];
    if (st.y == 0.0f || j >= len || (j >= base && !block_sees(a, b, i, j - base))) continue;
    const int64_t q0 = b * a.qs_b + h * a.qs_h + i * a.qs_s;
    float s = 0.0f;
    for (int g = 0, d = 0; d < a.D; ++g) {
      float dot = 0.0f;
      for (int e = 0; e < a.G && d < a.D; ++e, ++d)
        dot = fmaf(load_as_f32(a.q, q0 + d * a.qs_d, a.q_dt) * a.scale_log2, k_lds[key * pitch + d], dot);
      s = fmaf(dot, load_as_f32(a.ks, ks0 + j * a.kss_s + g, a.s_dt), s);
    }
    sum = fmaf(exp2f(block_score(s) - st.x), st.y, sum);
  }
  sums[tid] = sum;
  __syncthreads();
  if (tid < kWKeys && j < len) {
    float* dst = w + b * ws_b + kvh * ws_h + j * ws_k;
    *dst += (sums[tid] + sums[tid + kWKeys]) + (sums[tid + 2 * kWKeys] + sums[tid + 3 * kWKeys]);
  }
}

void launch_key_weights_rows(const BlockArgs& a, float* w, const int64_t* ws, hipStream_t st) {
  const int64_t chunks = (a.Sk + kWKeys - 1) / kWKeys;
  if (chunks == 0) return;
  hipLaunchKernelGGL(key_weights_rows_kernel, dim3((unsigned)(chunks * a.B * a.Hkv)), dim3(kWThreads), 0, st, a, w,
                     ws[0], ws[1], ws[2], (int)chunks);
}

int64_t stats_bytes(int64_t B, int64_t Hq, int64_t T) { return (B * Hq * T * 8 + 255) / 256 * 256; }

// Whether a call with attention keeps its scores (launch_block_weights): few
// rows per KV head, as of decode tokens, and scores of at most 1 GiB.
bool takes_scores(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, int q_dt, int s_dt) {
  if (!(D == 64 || D == 128) || q_dt == KVQ_F32 || s_dt == KVQ_F32) return false;
  const int64_t n = block_scores_bytes(B, Hq, Hkv, T, D, Sk);
  return n > 0 && n <= (int64_t(1) << 30);
}

int64_t workspace_needed(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t Sk, int q_dt, int s_dt,
                         bool with_out) {
  int64_t n = stats_bytes(B, Hq, T);
  if (B == 0 || T == 0 || !(D == 64 || D == 128) || q_dt == KVQ_F32 || s_dt == KVQ_F32) return n;
  if (with_out && takes_scores(B, Hq, Hkv, T, D, Sk, q_dt, s_dt)) return std::max(n, block_scores_bytes(B, Hq, Hkv, T, D, Sk));
  n = std::max(n, sums_workspace_bytes(B, Hq, Hkv, T, D, Sk, s_dt == KVQ_F16, with_out));
  return n;
}

// Shared by the two entry points: with `out`, the block's attention too.
int weights_impl(const char* what, const void* q, int q_dtype, const int64_t* q_strides, const void* k_packed,
                 const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides, const void* v_packed,
                 const int64_t* vp_strides, const void* v_scales, const int64_t* vs_strides, int scale_dtype, void* out,
                 const int64_t* out_strides, float* weights, const int64_t* weight_strides, int64_t B, int64_t Hq,
                 int64_t Hkv, int64_t T, int64_t D, int64_t group_size, const int32_t* seq_lens, int64_t Sk,
                 int is_causal, float sm_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  KVQ_CHECK_ARG(weight_strides && (!vp_strides || out_strides), "%s: null stride array", what);
  BlockArgs a;
  const int rc = fill_block_args(&a, what, q, q_dtype, q_strides, k_packed, kp_strides, k_scales, ks_strides, v_packed,
                                 vp_strides, v_scales, vs_strides, scale_dtype, B, Hq, Hkv, T, D, group_size, seq_lens,
                                 Sk, sm_scale, nullptr);
  if (rc != KVQ_OK) return rc;
  if (B == 0 || T == 0) return KVQ_OK;
  KVQ_CHECK_ARG(B * Hkv * ((Sk + kWKeys - 1) / kWKeys) < (int64_t(1) << 31), "%s: too large", what);
  KVQ_CHECK_ARG(q && (!vp_strides || out) && (weights || Sk == 0), "%s: null data pointer", what);
  const int64_t need = workspace_needed(B, Hq, Hkv, T, D, Sk, q_dtype, scale_dtype, vp_strides != nullptr);
  if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0) {
    set_error("%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)need);
    return KVQ_ESPACE;
  }
  a.kind = is_causal ? kMaskCausal : kMaskNone;
  a.stats = (float2*)workspace;
  if (vp_strides) {
    a.out = out;
    a.os_b = out_strides[0]; a.os_h = out_strides[1]; a.os_s = out_strides[2]; a.os_d = out_strides[3];
  }
  hipStream_t st = (hipStream_t)stream;
  if (a.out && takes_scores(B, Hq, Hkv, T, D, Sk, q_dtype, scale_dtype) && block_mfma_takes(a)) {
    a.stats = nullptr;
    const int lc = launch_block_weights(a, weights, weight_strides, workspace, st);
    KVQ_CHECK_ARG(lc == KVQ_OK, "%s: too large", what);
    KVQ_CHECK_LAUNCH(what);
    return KVQ_OK;
  }
  if (block_mfma_takes_keys(a)) {
    a.stats = nullptr;
    const bool attend = a.out && block_mfma_takes(a);
    if (a.out && !attend) launch_block_rows(a, st);
    const int lc = launch_key_sums(a, attend, weights, weight_strides, workspace, st);
    KVQ_CHECK_ARG(lc == KVQ_OK, "%s: too large", what);
  } else {
    launch_block_rows(a, st);
    launch_key_weights_rows(a, weights, weight_strides, st);
  }
  KVQ_CHECK_LAUNCH(what);
  return KVQ_OK;
}

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_attn_key_weights(const void* q, int q_dtype, const int64_t* q_strides, const void* k_packed,
                                    const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides,
                                    const void* v_packed, const int64_t* vp_strides, const void* v_scales,
                                    const int64_t* vs_strides, int scale_dtype, void* out, const int64_t* out_strides,
                                    float* weights, const int64_t* weight_strides, int64_t B, int64_t Hq, int64_t Hkv,
                                    int64_t Sq, int64_t D, int64_t group_size, const int32_t* seq_lens, int64_t Sk,
                                    int is_causal, float sm_scale, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  clear_error();
  KVQ_CHECK_ARG(vp_strides && vs_strides, "kvq_attn_key_weights: null stride array");
  return weights_impl("kvq_attn_key_weights", q, q_dtype, q_strides, k_packed, kp_strides, k_scales, ks_strides,
                      v_packed, vp_strides, v_scales, vs_strides, scale_dtype, out, out_strides, weights,
                      weight_strides, B, Hq, Hkv, Sq, D, group_size, seq_lens, Sk, is_causal, sm_scale, workspace,
                      workspace_bytes, stream);
}

extern "C" int kvq_add_key_weights(const void* q, int q_dtype, const int64_t* q_strides, const void* k_packed,
                                   const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides,
                                   int scale_dtype, float* weights, const int64_t* weight_strides, int64_t B,
                                   int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, int64_t group_size,
                                   const int32_t* seq_lens, int64_t Sk, int is_causal, float sm_scale, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  return weights_impl("kvq_add_key_weights", q, q_dtype, q_strides, k_packed, kp_strides, k_scales, ks_strides, nullptr,
                      nullptr, nullptr, nullptr, scale_dtype, nullptr, nullptr, weights, weight_strides, B, Hq, Hkv, Sq,
                      D, group_size, seq_lens, Sk, is_causal, sm_scale, workspace, workspace_bytes, stream);
}

extern "C" int64_t kvq_key_weights_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D,
                                                   int64_t group_size, int64_t Sk, int q_dtype, int scale_dtype,
                                                   int with_attention) {
  clear_error();
  if (B < 0 || Hq < 1 || Hkv < 1 || Sq < 0 || Sk < 0 || D < 1 || group_size < 1 || Hq % Hkv != 0 ||
      !dtype_ok(q_dtype) || !dtype_ok(scale_dtype)) {
    set_error("kvq_key_weights_workspace_bytes: bad shape or dtype");
    return KVQ_EINVAL;
  }
  return workspace_needed(B, Hq, Hkv, Sq, D, Sk, q_dtype, scale_dtype, with_attention != 0);
}
