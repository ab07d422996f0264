// Eviction: which rows of a cache to keep, and moving them (gfx950).
//
// select: per (sequence, KV head) of n keys, the first `sink`, the last
// `recent` and, of the others, those of the greatest weight, `keep` in all,
// as ascending row numbers. Equal weights go to the lowest row; a NaN ranks
// above every number, -0 with +0. The order is that of the weights' bits,
// mapped to unsigned integers that compare as the floats do.
// move: destination row first + i of each tensor is source row index[i].
//
// The reference's cache drops nothing (models/llama3/kv_cache.py:76-105).

#include "kvq_common.h"

namespace kvq {
namespace {

// ---------------------------------------------------------------------------
// select

struct SelectArgs {
  const float* w;
  int64_t ws_b, ws_h, ws_k;
  int32_t* index;  // [B, H, keep], contiguous
  const int32_t* seq_lens;
  int64_t S;
  int H;
  int keep, sink, recent;
};

constexpr int kSelThreads = 1024;

// Weights in the order of their floats: NaN above everything, -0 as +0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int wave_count(bool x) { return __builtin_popcountll(__builtin_amdgcn_ballot_w64(x)); }

// One workgroup per (sequence, KV head). The rank of the k-th largest weight
// is built bit by bit from the top (32 counts over the candidates), then one
// ordered pass writes the rows above it and the first of those that equal it.
__global__ __launch_bounds__(kSelThreads) void select_keys_kernel(const SelectArgs a) {
  __shared__ int counts[2][kSelThreads / 64];
  __shared__ int above[kSelThreads / 64], equal[kSelThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % a.H, b = blockIdx.x / a.H;
  int64_t n64 = a.S;
  if (a.seq_lens) {
    n64 = a.seq_lens[b];
    n64 = n64 < 0 ? 0 : (n64 > a.S ? a.S : n64);
  }
  const int n = (int)n64;
  const float* w = a.w + b * a.ws_b + h * a.ws_h;
  int32_t* out = a.index + ((int64_t)b * a.H + h) * a.keep;
  if (n <= a.keep) {
    for (int i = tid; i < a.keep; i += kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int lo = a.sink, hi = n - a.recent;  // candidates [lo, hi): keep > sink + recent or none is taken
  const int want = a.keep - a.sink - a.recent;
  uint32_t t = 0;  // the want-th largest rank
  if (want > 0) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = t | (1u << bit);
      int c = 0;
      for (int j = lo + tid; j - tid < hi; j += kSelThreads)
        c += wave_count(j < hi && rank_of(w[(int64_t)j * a.ws_k]) >= cand);
      int* slot = counts[bit & 1];
      if (lane == 0) slot[wave] = c;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int x = 0; x < kSelThreads / 64; ++x) total += slot[x];
      if (total >= want) t = cand;
    }
  } else {
    t = 0xffffffffu;
  }
  // rows in order, 1024 at a time: [0, sink) and [hi, n) always, a candidate
  // above t, and of those equal to t the first `ties`
  int n_above = 0;
  for (int j = lo + tid; j - tid < hi; j += kSelThreads)
    n_above += wave_count(j < hi && want > 0 && rank_of(w[(int64_t)j * a.ws_k]) > t);
  __syncthreads();
  if (lane == 0) counts[0][wave] = n_above;
  __syncthreads();
  int ties = want;
#pragma unroll
  for (int x = 0; x < kSelThreads / 64; ++x) ties -= counts[0][x];
  int done = 0, taken = 0;  // rows written, ties taken, before this chunk
  for (int j0 = 0; j0 < n; j0 += kSelThreads) {
    const int j = j0 + tid;
    const bool cand = want > 0 && j >= lo && j < hi;
    const uint32_t r = cand ? rank_of(w[(int64_t)j * a.ws_k]) : 0u;
    const bool sure = j < n && (j < lo || j >= hi || (cand && r > t)), tie = cand && r == t;
    const uint64_t mt = __builtin_amdgcn_ballot_w64(tie);
    if (lane == 0) equal[wave] = __builtin_popcountll(mt);
    __syncthreads();
    int before = taken, all = taken;
    for (int x = 0; x < kSelThreads / 64; ++x) {
      if (x < wave) before += equal[x];
      all += equal[x];
    }
    before += __builtin_popcountll(mt & ((1ull << lane) - 1));
    const bool on = sure || (tie && before < ties);
    const uint64_t mo = __builtin_amdgcn_ballot_w64(on);
    if (lane == 0) above[wave] = __builtin_popcountll(mo);
    __syncthreads();
    int at = done, sum = done;
    for (int x = 0; x < kSelThreads / 64; ++x) {
      if (x < wave) at += above[x];
      sum += above[x];
    }
    at += __builtin_popcountll(mo & ((1ull << lane) - 1));
    if (on && at < a.keep) out[at] = j;
    done = sum;
    taken = all;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// move

constexpr int kMoveMax = 5;  // tensors of one call: K and V codes and scales, weights

struct MoveTensor {
  const uint8_t* src;
  uint8_t* dst;
  int64_t ss_b, ss_h, ss_s, ds_b, ds_h, ds_s;  // byte strides
  int width;                                   // bytes of a row
  int unit;                                    // bytes moved at a time (16, 8, 4, 2 or 1)
  int lpr;                                     // units of a row
};

struct MoveArgs {
  MoveTensor t[kMoveMax];
  const int32_t* index;
  int64_t is_b, is_h, is_i;
  const int32_t* first;  // device [B] first destination rows, or null
  int64_t first0;
  int64_t S, dst_rows;
  PageMap pm;  // paged: source and destination rows go through the table
  int H, n;
};

__device__ __forceinline__ int64_t move_first(const MoveArgs& a, int b) { return a.first ? a.first[b] : a.first0; }

// Source and destination row of item i, or source -1 (nothing moves): an index
// outside [0, S), a destination outside its rows, a page without a block.
__device__ __forceinline__ void move_rows_of(const MoveArgs& a, int b, int h, int i, int64_t* src, int64_t* dst) {
  const int64_t from = a.index[b * a.is_b + h * a.is_h + i * a.is_i];
  const int64_t to = move_first(a, b) + i;
  *src = -1;
  *dst = to;
  if (from < 0 || from >= a.S || to < 0 || to >= a.dst_rows) return;
  if (!a.pm.paged) {
    *src = from;
    return;
  }
  const int64_t s = page_row(a.pm, b, from), d = page_row(a.pm, b, to);
  if (s < 0 || d < 0) return;
  *src = s;
  *dst = d;
}

__device__ __forceinline__ uint4 move_load(const uint8_t* p, int unit) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (unit == 16) v = *(const uint4*)p;
  else if (unit == 8) { const uint2 x = *(const uint2*)p; v.x = x.x; v.y = x.y; }
  else if (unit == 4) v.x = *(const uint32_t*)p;
  else if (unit == 2) v.x = *(const uint16_t*)p;
  else v.x = *p;
  return v;
}
__device__ __forceinline__ void move_store(uint8_t* p, int unit, uint4 v) {
  if (unit == 16) *(uint4*)p = v;
  else if (unit == 8) *(uint2*)p = make_uint2(v.x, v.y);
  else if (unit == 4) *(uint32_t*)p = v.x;
  else if (unit == 2) *(uint16_t*)p = (uint16_t)v.x;
  else *p = (uint8_t)v.x;
}

constexpr int kMoveThreads = 256;

// Into other buffers: a thread moves one piece of one row; blockIdx.y is the
// tensor, blockIdx.z the (sequence, head).
__global__ __launch_bounds__(kMoveThreads) void move_rows_kernel(const MoveArgs a) {
  const MoveTensor t = a.t[blockIdx.y];
  const int h = blockIdx.z % a.H, b = blockIdx.z / a.H;
  const int64_t x = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x;
  const int64_t i = x / t.lpr;
  if (i >= a.n) return;
  const int at = (int)(x % t.lpr) * t.unit;
  int64_t s, d;
  move_rows_of(a, b, h, (int)i, &s, &d);
  if (s < 0) return;
  move_store(t.dst + b * t.ds_b + h * t.ds_h + d * t.ds_s + at, t.unit,
             move_load(t.src + b * t.ss_b + h * t.ss_h + s * t.ss_s + at, t.unit));
}

// In place: one workgroup per tensor, sequence and head reads every row that
// moves into LDS, then writes them, so that any index is right.
constexpr int kMoveLds = 65536;

__global__ __launch_bounds__(kMoveThreads) void move_rows_in_place_kernel(const MoveArgs a) {
  __shared__ __align__(16) uint8_t lds[kMoveLds];
  const MoveTensor t = a.t[blockIdx.y];
  const int h = blockIdx.z % a.H, b = blockIdx.z / a.H;
  const int pieces = a.n * t.lpr;
  for (int x = threadIdx.x; x < pieces; x += kMoveThreads) {
    int64_t s, d;
    move_rows_of(a, b, h, x / t.lpr, &s, &d);
    if (s < 0) continue;
    move_store(lds + (int64_t)x * t.unit, t.unit,
               move_load(t.src + b * t.ss_b + h * t.ss_h + s * t.ss_s + (x % t.lpr) * t.unit, t.unit));
  }
  __syncthreads();
  for (int x = threadIdx.x; x < pieces; x += kMoveThreads) {
    int64_t s, d;
    move_rows_of(a, b, h, x / t.lpr, &s, &d);
    if (s < 0) continue;
    move_store(t.dst + b * t.ds_b + h * t.ds_h + d * t.ds_s + (x % t.lpr) * t.unit, t.unit,
               move_load(lds + (int64_t)x * t.unit, t.unit));
  }
}

int move_impl(const char* what, int64_t n_tensors, const void* const* src, const int64_t* src_strides, void* const* dst,
              const int64_t* dst_strides, const int64_t* widths, const int32_t* index, const int64_t* index_strides,
              int64_t B, int64_t H, int64_t S, int64_t n, int64_t dst_rows, const int32_t* first, int64_t first0,
              void* stream, const PageMap* pm, bool in_place) {
  clear_error();
  KVQ_CHECK_ARG(n_tensors >= 1 && n_tensors <= kMoveMax, "%s: 1 to %d tensors (got %lld)", what, kMoveMax,
                (long long)n_tensors);
  KVQ_CHECK_ARG(src && src_strides && dst && dst_strides && widths && index_strides, "%s: null argument array", what);
  KVQ_CHECK_ARG(B >= 0 && H >= 1 && S >= 0 && n >= 0 && dst_rows >= 0 && B * H < 65536 && S < (int64_t(1) << 31) &&
                    n < (int64_t(1) << 24),
                "%s: bad shape (B=%lld H=%lld S=%lld n=%lld)", what, (long long)B, (long long)H, (long long)S,
                (long long)n);
  MoveArgs a = {};
  int64_t most = 0;
  for (int k = 0; k < n_tensors; ++k) {
    const int64_t* ss = src_strides + 3 * k;
    const int64_t* ds = dst_strides + 3 * k;
    KVQ_CHECK_ARG(widths[k] >= 1 && widths[k] <= (1 << 20), "%s: row of %lld bytes", what, (long long)widths[k]);
    KVQ_CHECK_ARG(B == 0 || n == 0 || (dst[k] && (src[k] || S == 0)), "%s: null data pointer", what);
    MoveTensor& t = a.t[k];
    t.src = (const uint8_t*)src[k];
    t.dst = (uint8_t*)dst[k];
    t.ss_b = ss[0]; t.ss_h = ss[1]; t.ss_s = ss[2];
    t.ds_b = ds[0]; t.ds_h = ds[1]; t.ds_s = ds[2];
    t.width = (int)widths[k];
    // the widest piece that divides the row and that every row is aligned for
    t.unit = 16;
    auto fits = [&](int u) {
      return widths[k] % u == 0 && (uintptr_t)src[k] % u == 0 && (uintptr_t)dst[k] % u == 0 && ss[0] % u == 0 &&
             ss[1] % u == 0 && ss[2] % u == 0 && ds[0] % u == 0 && ds[1] % u == 0 && ds[2] % u == 0;
    };
    while (t.unit > 1 && !fits(t.unit)) t.unit >>= 1;
    t.lpr = t.width / t.unit;
    if (in_place) KVQ_CHECK_ARG(n * widths[k] <= kMoveLds, "%s: in place, at most %d bytes of rows a head move (got %lld)",
                                what, kMoveLds, (long long)(n * widths[k]));
    most = n * t.lpr > most ? n * t.lpr : most;
  }
  if (B == 0 || n == 0) return KVQ_OK;
  KVQ_CHECK_ARG(index, "%s: null index", what);
  a.index = index;
  a.is_b = index_strides[0]; a.is_h = index_strides[1]; a.is_i = index_strides[2];
  a.first = first;
  a.first0 = first0;
  a.S = S;
  a.dst_rows = dst_rows;
  a.H = (int)H;
  a.n = (int)n;
  if (pm) a.pm = *pm;
  hipStream_t st = (hipStream_t)stream;
  if (in_place) {
    hipLaunchKernelGGL(move_rows_in_place_kernel, dim3(1, (unsigned)n_tensors, (unsigned)(B * H)), dim3(kMoveThreads), 0,
                       st, a);
  } else {
    const int64_t wgs = (most + kMoveThreads - 1) / kMoveThreads;
    KVQ_CHECK_ARG(wgs < (int64_t(1) << 31), "%s: too large", what);
    hipLaunchKernelGGL(move_rows_kernel, dim3((unsigned)wgs, (unsigned)n_tensors, (unsigned)(B * H)), dim3(kMoveThreads),
                       0, st, a);
  }
  KVQ_CHECK_LAUNCH(what);
  return KVQ_OK;
}

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_select_keys(const float* weights, const int64_t* weight_strides, int64_t B, int64_t H, int64_t S,
                               const int32_t* seq_lens, int64_t n_keep, int64_t sink, int64_t recent, int32_t* index,
                               void* stream) {
  clear_error();
  KVQ_CHECK_ARG(weight_strides, "kvq_select_keys: null stride array");
  KVQ_CHECK_ARG(B >= 0 && H >= 1 && S >= 0 && S < (int64_t(1) << 30) && B * H < (int64_t(1) << 31),
                "kvq_select_keys: bad shape (B=%lld H=%lld S=%lld)", (long long)B, (long long)H, (long long)S);
  KVQ_CHECK_ARG(sink >= 0 && recent >= 0 && n_keep >= 0 && n_keep < (int64_t(1) << 30) && sink <= n_keep &&
                    recent <= n_keep - sink,
                "kvq_select_keys: n_keep (%lld) must hold sink (%lld) and recent (%lld)", (long long)n_keep,
                (long long)sink, (long long)recent);
  if (B == 0 || n_keep == 0) return KVQ_OK;
  KVQ_CHECK_ARG(index && (weights || S == 0), "kvq_select_keys: null data pointer");
  const SelectArgs a = {weights, weight_strides[0], weight_strides[1], weight_strides[2], index, seq_lens, S, (int)H,
                        (int)n_keep, (int)sink, (int)recent};
  hipLaunchKernelGGL(select_keys_kernel, dim3((unsigned)(B * H)), dim3(kSelThreads), 0, (hipStream_t)stream, a);
  KVQ_CHECK_LAUNCH("kvq_select_keys");
  return KVQ_OK;
}

extern "C" int kvq_move_rows(int64_t n_tensors, const void* const* src, const int64_t* src_strides, void* const* dst,
                             const int64_t* dst_strides, const int64_t* row_bytes, const int32_t* index,
                             const int64_t* index_strides, int64_t B, int64_t H, int64_t S, int64_t n, int64_t dst_rows,
                             const int32_t* first, int64_t first0, int in_place, void* stream) {
  return move_impl("kvq_move_rows", n_tensors, src, src_strides, dst, dst_strides, row_bytes, index, index_strides, B, H,
                   S, n, dst_rows, first, first0, stream, nullptr, in_place != 0);
}

extern "C" int kvq_move_rows_paged(int64_t n_tensors, void* const* pools, const int64_t* pool_strides,
                                   const int64_t* row_bytes, const int32_t* block_table, int64_t table_stride,
                                   int64_t table_cols, int64_t num_blocks, int64_t page_size, const int32_t* index,
                                   const int64_t* index_strides, int64_t B, int64_t H, int64_t n, const int32_t* first,
                                   int64_t first0, void* stream) {
  clear_error();
  KVQ_CHECK_ARG(page_size >= 1 && (page_size & (page_size - 1)) == 0 && page_size <= (1 << 20),
                "kvq_move_rows_paged: page_size must be a power of two (got %lld)", (long long)page_size);
  KVQ_CHECK_ARG(num_blocks >= 0 && num_blocks < (int64_t(1) << 31) && table_cols >= 0 && table_stride >= table_cols &&
                    (block_table || table_cols == 0 || B == 0),
                "kvq_move_rows_paged: bad block table geometry");
  KVQ_CHECK_ARG(pool_strides, "kvq_move_rows_paged: null argument array");
  KVQ_CHECK_ARG(n_tensors >= 1 && n_tensors <= kMoveMax, "kvq_move_rows_paged: 1 to %d tensors (got %lld)", kMoveMax,
                (long long)n_tensors);
  int64_t st[3 * kMoveMax];
  for (int k = 0; k < n_tensors; ++k) {
    st[3 * k] = 0;
    st[3 * k + 1] = pool_strides[2 * k];
    st[3 * k + 2] = pool_strides[2 * k + 1];
  }
  int shift = 0;
  while ((int64_t(1) << shift) < page_size) ++shift;
  const PageMap pm{1, block_table, table_stride, table_cols, num_blocks, shift};
  const int64_t rows = table_cols * page_size;
  return move_impl("kvq_move_rows_paged", n_tensors, (const void* const*)pools, st, pools, st, row_bytes, index,
                   index_strides, B, H, rows, n, rows, first, first0, stream, &pm, true);
}
