// Tree attention: a block of T drafted tokens, which form a tree, over the
// INT4 cache that already holds their rows (gfx950).
//
//   s[i, j] = sm_scale * q_i . k_j                       (query head h reads KV head h / ratio)
//   o_i     = sum_j 2^(c s[i, j] - m_i) v_j / sum_j 2^(c s[i, j] - m_i),   c = log2 e
//
// over the keys j that row i attends: all before the block, and of the block's
// own rows those of its ancestors and itself (a mask). A row that attends no
// key is zero. The reference has no counterpart (its kernel masks causally,
// kernels/llama3/attention_quant.py:91-97).

#include "kvq_block_mfma.h"

namespace kvq {

int fill_block_args(BlockArgs* a, const char* what, const void* q, int q_dtype, const int64_t* q_strides,
                    const void* k_packed, const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides,
                    const void* v_packed, const int64_t* vp_strides, const void* v_scales, const int64_t* vs_strides,
                    int scale_dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t group_size,
                    const int32_t* seq_lens, int64_t Sk, float sm_scale, const BlockPaged* pg) {
  KVQ_CHECK_ARG(q_strides && kp_strides && ks_strides && (vp_strides != nullptr) == (vs_strides != nullptr),
                "%s: null stride array", what);
  KVQ_CHECK_ARG(dtype_ok(q_dtype) && dtype_ok(scale_dtype), "%s: unknown dtype code", what);
  KVQ_CHECK_ARG(B >= 0 && Hq >= 1 && Hkv >= 1 && T >= 0 && Sk >= 0 && D >= 1 && group_size >= 1,
                "%s: bad shape (B=%lld Hq=%lld Hkv=%lld T=%lld Sk=%lld D=%lld G=%lld)", what, (long long)B,
                (long long)Hq, (long long)Hkv, (long long)T, (long long)Sk, (long long)D, (long long)group_size);
  KVQ_CHECK_ARG(Hq % Hkv == 0, "%s: Hq (%lld) must be a multiple of Hkv (%lld)", what, (long long)Hq, (long long)Hkv);
  if (D > kMaxBlockD) {
    set_error("%s: head dims up to %d (got %lld)", what, kMaxBlockD, (long long)D);
    return KVQ_EUNSUP;
  }
  KVQ_CHECK_ARG(B < (1 << 24) && T < (1 << 24) && Sk < (int64_t(1) << 31) && Hq <= 65536 && B * Hq * T < (int64_t(1) << 31),
                "%s: too large", what);
  const int64_t groups = (D + group_size - 1) / group_size, width = groups * ((group_size + 1) / 2);
  const int sd = pg ? 1 : 2;  // place of the row stride
  KVQ_CHECK_ARG(kp_strides[sd] >= width && ks_strides[sd] >= groups &&
                    (!vp_strides || (vp_strides[sd] >= width && vs_strides[sd] >= groups)),
                "%s: cache rows narrower than the codes or scales of D = %lld, G = %lld", what, (long long)D,
                (long long)group_size);
  *a = BlockArgs{};
  if (pg) {
    KVQ_CHECK_ARG(pg->page_size >= 1 && (pg->page_size & (pg->page_size - 1)) == 0 && pg->page_size <= (1 << 20),
                  "%s: page_size must be a power of two (got %lld)", what, (long long)pg->page_size);
    KVQ_CHECK_ARG(pg->n_blocks >= 0 && pg->n_blocks < (int64_t(1) << 31) && pg->bt_cols >= 0 &&
                      pg->bt_stride >= pg->bt_cols && Sk <= pg->bt_cols * pg->page_size,
                  "%s: bad block table geometry or length past the table", what);
    KVQ_CHECK_ARG(pg->bt != nullptr || pg->bt_cols == 0 || B == 0, "%s: null block table", what);
    int shift = 0;
    while ((int64_t(1) << shift) < pg->page_size) ++shift;
    a->pm = PageMap{1, pg->bt, pg->bt_stride, pg->bt_cols, pg->n_blocks, shift};
  }
  const bool reads = B > 0 && T > 0 && Sk > 0;
  KVQ_CHECK_ARG(!reads || (q && k_packed && k_scales && (!vp_strides || (v_packed && v_scales))),
                "%s: null data pointer", what);
  a->q = q;
  a->qs_b = q_strides[0]; a->qs_h = q_strides[1]; a->qs_s = q_strides[2]; a->qs_d = q_strides[3];
  auto three = [&](const int64_t* s, int64_t* b, int64_t* h, int64_t* r) {
    *b = pg ? 0 : s[0];
    *h = s[sd - 1];
    *r = s[sd];
  };
  a->kp = (const uint8_t*)k_packed;
  a->ks = k_scales;
  three(kp_strides, &a->kps_b, &a->kps_h, &a->kps_s);
  three(ks_strides, &a->kss_b, &a->kss_h, &a->kss_s);
  if (vp_strides) {
    a->vp = (const uint8_t*)v_packed;
    a->vs = v_scales;
    three(vp_strides, &a->vps_b, &a->vps_h, &a->vps_s);
    three(vs_strides, &a->vss_b, &a->vss_h, &a->vss_s);
  }
  a->seq_lens = seq_lens;
  a->Sk = Sk;
  a->q_dt = q_dtype; a->s_dt = scale_dtype; a->kind = kMaskNone;
  a->B = (int)B; a->Hq = (int)Hq; a->Hkv = (int)Hkv; a->ratio = (int)(Hq / Hkv); a->T = (int)T;
  a->D = (int)D; a->G = (int)group_size;
  a->scale_log2 = sm_scale * 1.4426950408889634f;
  return KVQ_OK;
}

namespace {

constexpr int kRowThreads = 256;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

// One workgroup per query row: 256 keys at a time, a thread scores a key in
// fp32; then a thread owns a dim (256 / D keys' parts side by side) of the
// weighted values. Right for every dtype, group size, stride and page; a key
// that is not attended is never multiplied in, so what it holds does not
// matter.
__global__ __launch_bounds__(kRowThreads) void block_rows_kernel(const BlockArgs a) {
  __shared__ float q_lds[kMaxBlockD];
  __shared__ float p_lds[kRowThreads];
  __shared__ int64_t row_lds[kRowThreads];
  __shared__ float red[kRowThreads / 64];
  __shared__ float o_lds[kRowThreads];
  const int tid = threadIdx.x, wave = tid >> 6;
  int wg = blockIdx.x;
  const int i = wg % a.T;
  wg /= a.T;
  const int h = wg % a.Hq, b = wg / a.Hq, kvh = h / a.ratio;
  const int64_t len = block_len(a, b), base = len - a.T;

  if (tid < a.D)
    q_lds[tid] = load_as_f32(a.q, b * a.qs_b + h * a.qs_h + i * a.qs_s + tid * a.qs_d, a.q_dt) * a.scale_log2;
  __syncthreads();

  const uint8_t* kp = a.kp + b * a.kps_b + kvh * a.kps_h;
  const uint8_t* vp = a.vp + b * a.vps_b + kvh * a.vps_h;
  const int64_t ks0 = b * a.kss_b + kvh * a.kss_h, vs0 = b * a.vss_b + kvh * a.vss_h;
  const int parts = kRowThreads / a.D;  // threads per dim (D <= 256)
  const int d = tid % a.D, part = tid / a.D;
  const int vg = d / a.G;
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
  for (int64_t j0 = 0; j0 < len; j0 += kRowThreads) {
    const int64_t j = j0 + tid;
    bool on = j < len && (j < base || block_sees(a, b, i, j - base));
    int64_t r = -1;
    if (on) {
      r = a.pm.paged ? page_row(a.pm, b, j) : j;
      on = r >= 0;
    }
    float s = -__builtin_inff();
    if (on) {
      float dot = 0.0f;
      for (int g = 0, x = 0; x < a.D; ++g) {
        float part_dot = 0.0f;
        for (int e = 0; e < a.G && x < a.D; ++e, ++x) part_dot = fmaf(q_lds[x], code_at(kp + r * a.kps_s, x, a.G), part_dot);
        dot = fmaf(part_dot, load_as_f32(a.ks, ks0 + r * a.kss_s + g, a.s_dt), dot);
      }
      s = block_score(dot);
    }
    float mx = wave_max(s);
    if ((tid & 63) == 0) red[wave] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowThreads / 64; ++w) mx = fmaxf(mx, red[w]);
    const float m_new = fmaxf(m, mx);
    const float alpha = m == m_new ? 1.0f : exp2f(m - m_new);
    const float p = s == -__builtin_inff() ? 0.0f : exp2f(s - m_new);
    m = m_new;
    p_lds[tid] = p;
    row_lds[tid] = r;
    __syncthreads();
    l = l * alpha + p;  // this thread's keys
    if (a.out && part < parts) {
      o *= alpha;
      for (int x = part; x < kRowThreads; x += parts) {
        const float w = p_lds[x];
        if (w == 0.0f) continue;
        const int64_t rr = row_lds[x];
        o = fmaf(w, code_at(vp + rr * a.vps_s, d, a.G) * load_as_f32(a.vs, vs0 + rr * a.vss_s + vg, a.s_dt), o);
      }
    }
  }
  l = wave_sum(l);
  __syncthreads();
  if ((tid & 63) == 0) red[wave] = l;
  o_lds[tid] = o;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) l += red[w];
  if (a.stats && tid == 0)
    a.stats[stats_at(a, b, h, i)] = make_float2(m, l > 0.0f ? 1.0f / l : 0.0f);
  if (a.out && tid < a.D) {
    float x = 0.0f;
    for (int w = 0; w < parts; ++w) x += o_lds[w * a.D + tid];
    store_from_f32(a.out, b * a.os_b + h * a.os_h + i * a.os_s + tid * a.os_d, a.q_dt, l > 0.0f ? x / l : 0.0f);
  }
}

// The same where groups are whole code words (G a multiple of 8, D too, and
// rows aligned for 4-byte loads): a thread scores a key eight dims at a time,
// and weighs eight dims of every (NT / (D / 8))-th key, so that no index is
// divided in a loop and a chunk's loads are in flight together. (96 rows of
// GPT-2 small over 1000 keys: 105 us above, 23 with 256 threads, 13 with 1024.)
template <int NT>
__global__ __launch_bounds__(NT) void block_rows8_kernel(const BlockArgs a) {
  __shared__ __align__(16) float q_lds[kMaxBlockD];
  __shared__ float p_lds[NT];
  __shared__ int64_t row_lds[NT];
  __shared__ float red[NT / 64];
  __shared__ __align__(16) float o_lds[NT * 8];
  const int tid = threadIdx.x, wave = tid >> 6;
  int wg = blockIdx.x;
  const int i = wg % a.T;
  wg /= a.T;
  const int h = wg % a.Hq, b = wg / a.Hq, kvh = h / a.ratio;
  const int64_t len = block_len(a, b), base = len - a.T;
  const int words = a.D / 8, gw = a.G / 8;  // code words of a row, of a group

  if (tid < a.D)
    q_lds[tid] = load_as_f32(a.q, b * a.qs_b + h * a.qs_h + i * a.qs_s + tid * a.qs_d, a.q_dt) * a.scale_log2;
  __syncthreads();

  const uint8_t* kp = a.kp + b * a.kps_b + kvh * a.kps_h;
  const uint8_t* vp = a.vp + b * a.vps_b + kvh * a.vps_h;
  const int64_t ks0 = b * a.kss_b + kvh * a.kss_h, vs0 = b * a.vss_b + kvh * a.vss_h;
  const int word = tid % words, part = tid / words, parts = NT / words;
  float m = -__builtin_inff(), l = 0.0f;
  float o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t j0 = 0; j0 < len; j0 += NT) {
    const int64_t j = j0 + tid;
    bool on = j < len && (j < base || block_sees(a, b, i, j - base));
    int64_t r = -1;
    if (on) {
      r = a.pm.paged ? page_row(a.pm, b, j) : j;
      on = r >= 0;
    }
    float s = -__builtin_inff();
    if (on) {
      const uint32_t* row = (const uint32_t*)(kp + r * a.kps_s);
      float dot = 0.0f;
      for (int g = 0, x = 0; x < words; ++g) {
        float part_dot = 0.0f;
#pragma unroll 4
        for (int e = 0; e < gw; ++e, ++x) {
          const uint32_t w = row[x];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            part_dot = fmaf(q_lds[8 * x + k], (float)((int)((w >> (4 * k)) & 15u) - 8), part_dot);
        }
        dot = fmaf(part_dot, load_as_f32(a.ks, ks0 + r * a.kss_s + g, a.s_dt), dot);
      }
      s = block_score(dot);
    }
    float mx = wave_max(s);
    if ((tid & 63) == 0) red[wave] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) mx = fmaxf(mx, red[w]);
    const float m_new = fmaxf(m, mx);
    const float alpha = m == m_new ? 1.0f : exp2f(m - m_new);
    const float p = s == -__builtin_inff() ? 0.0f : exp2f(s - m_new);
    m = m_new;
    p_lds[tid] = p;
    row_lds[tid] = r;
    __syncthreads();
    l = l * alpha + p;  // this thread's keys
    if (a.out && part < parts) {
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] *= alpha;
      for (int x0 = part; x0 < NT; x0 += 8 * parts) {
        uint32_t w[8];
        float sc[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {  // (a key without weight is not read)
          const int x = x0 + y * parts;
          const float p8 = x < NT ? p_lds[x] : 0.0f;
          w[y] = 0u;
          sc[y] = 0.0f;
          if (p8 != 0.0f) {
            const int64_t rr = row_lds[x];
            w[y] = ((const uint32_t*)(vp + rr * a.vps_s))[word];
            sc[y] = load_as_f32(a.vs, vs0 + rr * a.vss_s + word / gw, a.s_dt);
          }
        }
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const int x = x0 + y * parts;
          const float p8 = x < NT ? p_lds[x] : 0.0f;
          if (p8 != 0.0f) {
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = fmaf(p8, (float)((int)((w[y] >> (4 * k)) & 15u) - 8) * sc[y], o[k]);
          }
        }
      }
    }
  }
  l = wave_sum(l);
  __syncthreads();
  if ((tid & 63) == 0) red[wave] = l;
#pragma unroll
  for (int k = 0; k < 8; ++k) o_lds[tid * 8 + k] = o[k];
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) l += red[w];
  if (a.stats && tid == 0)
    a.stats[stats_at(a, b, h, i)] = make_float2(m, l > 0.0f ? 1.0f / l : 0.0f);
  if (!a.out) return;
  // dim d's parts: first every (NT / D)-th of them, then those sums
  const int d = tid % a.D, first = tid / a.D, step = NT / a.D;
  float x = 0.0f;
  if (first < step)
    for (int y = first; y < parts; y += step) x += o_lds[(y * words) * 8 + d];
  __syncthreads();
  if (first < step) o_lds[tid] = x;
  __syncthreads();
  if (tid < a.D) {
    x = 0.0f;
    for (int y = 0; y < step; ++y) x += o_lds[y * a.D + tid];
    store_from_f32(a.out, b * a.os_b + h * a.os_h + i * a.os_s + tid * a.os_d, a.q_dt, l > 0.0f ? x / l : 0.0f);
  }
}

}  // namespace

void launch_block_rows(const BlockArgs& a, hipStream_t st) {
  const int64_t n = (int64_t)a.B * a.Hq * a.T;
  auto words = [](const void* p, int64_t b, int64_t h, int64_t s) {
    return (uintptr_t)p % 4 == 0 && b % 4 == 0 && h % 4 == 0 && s % 4 == 0;
  };
  if (a.D % 8 == 0 && a.G % 8 == 0 && a.D % a.G == 0 && words(a.kp, a.kps_b, a.kps_h, a.kps_s) &&
      words(a.vp, a.vps_b, a.vps_h, a.vps_s))
    // 1024 keys at a time while all rows' workgroups are resident together (512):
    // latency counts (fp32, 96 rows of 64 dims: 1000 keys 12.8 against 23.0 us,
    // 4096 keys 32 against 78). More rows fill the GPU with 256 threads each (1536
    // rows, 1000 keys: 54 against 71 us).
    if (a.Sk > kRowThreads && n <= 512) hipLaunchKernelGGL((block_rows8_kernel<1024>), dim3((unsigned)n), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((block_rows8_kernel<256>), dim3((unsigned)n), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(block_rows_kernel, dim3((unsigned)n), dim3(kRowThreads), 0, st, a);
}

}  // namespace kvq

using namespace kvq;

namespace {

int tree_impl(const char* what, const void* q, int q_dtype, const int64_t* q_strides, const void* k_packed,
              const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides, const void* v_packed,
              const int64_t* vp_strides, const void* v_scales, const int64_t* vs_strides, int scale_dtype,
              const void* mask, const int64_t* mask_strides, void* out, const int64_t* out_strides, int64_t B,
              int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t group_size, const int32_t* seq_lens, int64_t Sk,
              float sm_scale, void* workspace, int64_t workspace_bytes, void* stream, const BlockPaged* pg) {
  clear_error();
  KVQ_CHECK_ARG(mask_strides && out_strides && vp_strides && vs_strides, "%s: null stride array", what);
  BlockArgs a;
  const int rc = fill_block_args(&a, what, q, q_dtype, q_strides, k_packed, kp_strides, k_scales, ks_strides, v_packed,
                                 vp_strides, v_scales, vs_strides, scale_dtype, B, Hq, Hkv, T, D, group_size, seq_lens,
                                 Sk, sm_scale, pg);
  if (rc != KVQ_OK) return rc;
  if (B == 0 || T == 0) return KVQ_OK;
  KVQ_CHECK_ARG(q && out && mask, "%s: null data pointer", what);
  a.kind = kMaskTree;
  a.mask = (const uint8_t*)mask;
  a.ms_b = mask_strides[0]; a.ms_i = mask_strides[1]; a.ms_t = mask_strides[2];
  a.out = out;
  a.os_b = out_strides[0]; a.os_h = out_strides[1]; a.os_s = out_strides[2]; a.os_d = out_strides[3];
  if (block_mfma_takes(a)) {
    const int lc = launch_block_mfma(a, workspace, workspace_bytes, (hipStream_t)stream);
    KVQ_CHECK_ARG(lc == KVQ_OK, "%s: too large", what);
  } else {
    launch_block_rows(a, (hipStream_t)stream);
  }
  KVQ_CHECK_LAUNCH(what);
  return KVQ_OK;
}

}  // namespace

extern "C" int kvq_tree_attn(const void* q, int q_dtype, const int64_t* q_strides, const void* k_packed,
                             const int64_t* kp_strides, const void* k_scales, const int64_t* ks_strides,
                             const void* v_packed, const int64_t* vp_strides, const void* v_scales,
                             const int64_t* vs_strides, int scale_dtype, const void* mask, const int64_t* mask_strides,
                             void* out, const int64_t* out_strides, int64_t B, int64_t Hq, int64_t Hkv, int64_t T,
                             int64_t D, int64_t group_size, const int32_t* seq_lens, int64_t Sk, float sm_scale,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  return tree_impl("kvq_tree_attn", q, q_dtype, q_strides, k_packed, kp_strides, k_scales, ks_strides, v_packed,
                   vp_strides, v_scales, vs_strides, scale_dtype, mask, mask_strides, out, out_strides, B, Hq, Hkv, T, D,
                   group_size, seq_lens, Sk, sm_scale, workspace, workspace_bytes, stream, nullptr);
}

extern "C" int kvq_tree_attn_paged(const void* q, int q_dtype, const int64_t* q_strides, const void* k_pool,
                                   const int64_t* kp_strides, const void* k_scale_pool, const int64_t* ks_strides,
                                   const void* v_pool, const int64_t* vp_strides, const void* v_scale_pool,
                                   const int64_t* vs_strides, int scale_dtype, const int32_t* block_table,
                                   int64_t table_stride, int64_t table_cols, int64_t num_blocks, int64_t page_size,
                                   const void* mask, const int64_t* mask_strides, void* out, const int64_t* out_strides,
                                   int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t group_size,
                                   const int32_t* seq_lens, int64_t Sk, float sm_scale, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const BlockPaged pg{block_table, table_stride, table_cols, num_blocks, page_size};
  return tree_impl("kvq_tree_attn_paged", q, q_dtype, q_strides, k_pool, kp_strides, k_scale_pool, ks_strides, v_pool,
                   vp_strides, v_scale_pool, vs_strides, scale_dtype, mask, mask_strides, out, out_strides, B, Hq, Hkv,
                   T, D, group_size, seq_lens, Sk, sm_scale, workspace, workspace_bytes, stream, &pg);
}

extern "C" int64_t kvq_tree_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D,
                                                 int64_t group_size, int64_t Sk, int q_dtype, int scale_dtype) {
  clear_error();
  if (B < 0 || Hq < 1 || Hkv < 1 || T < 0 || Sk < 0 || D < 1 || group_size < 1 || Hq % Hkv != 0 || !dtype_ok(q_dtype) ||
      !dtype_ok(scale_dtype)) {
    set_error("kvq_tree_attn_workspace_bytes: bad shape or dtype");
    return KVQ_EINVAL;
  }
  if (B == 0 || T == 0 || !(D == 64 || D == 128) || q_dtype == KVQ_F32 || scale_dtype == KVQ_F32) return 0;
  return block_workspace_bytes(B, Hq, Hkv, T, D, Sk, scale_dtype == KVQ_F16);
}
