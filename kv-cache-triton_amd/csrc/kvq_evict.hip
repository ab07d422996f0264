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

struct SelectUnit {
  const float* w;
  int32_t* out;
  int n, lo, hi, want;  // candidates [lo, hi), of which `want` are kept
};

__device__ __forceinline__ SelectUnit select_unit(const SelectArgs& a) {
  const int h = blockIdx.x % a.H, b = blockIdx.x / a.H;
  int64_t n = a.S;
  if (a.seq_lens) {
    n = a.seq_lens[b];
    n = n < 0 ? 0 : (n > a.S ? a.S : n);
  }
  SelectUnit u;
  u.w = a.w + b * a.ws_b + h * a.ws_h;
  u.out = a.index + ((int64_t)b * a.H + h) * a.keep;
  u.n = (int)n;
  u.lo = a.sink;
  u.hi = u.n - a.recent;
  u.want = a.keep - a.sink - a.recent;
  return u;
}

// A sequence that keeps everything.
__device__ __forceinline__ void select_all(const SelectArgs& a, const SelectUnit& u) {
  for (int i = threadIdx.x; i < a.keep; i += kSelThreads) u.out[i] = i < u.n ? i : -1;
}

// Sum over the workgroup's waves of a value uniform in each wave; `slot`
// alternates between two calls' buffers, so that one barrier is enough.
__device__ __forceinline__ int block_sum(int x, int* slot) {
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = x;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 64; ++w) total += slot[w];
  return total;
}

// One workgroup per (sequence, KV head), its ranks in registers (NE a thread;
// each wave holds 64 NE consecutive rows, so that its kept rows are counted
// and written in order). The rank of the want-th largest is built bit by bit
// from the top: a bit is set if that many candidates are at least the rank so
// formed, counted with one compare a register and ballots (a histogram in LDS
// would put most of a wave's lanes on the same few exponents). It stops as soon
// as exactly `want` candidates are at or above it. Bound by those compares and a
// barrier a bit, about 0.2 us a bit at 16K keys.
template <int NE>
__global__ __launch_bounds__(kSelThreads) void select_keys_kernel(const SelectArgs a) {
  __shared__ int counts[2][kSelThreads / 64];
  const SelectUnit u = select_unit(a);
  if (u.n <= a.keep) {
    select_all(a, u);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j0 = wave * (64 * NE) + lane;
  uint32_t r[NE];  // ranks of rows j0 + 64 e; 0 (below every rank) outside the candidates
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const int j = j0 + 64 * e;
    r[e] = j >= u.lo && j < u.hi ? rank_of(u.w[(int64_t)j * a.ws_k]) : 0u;
  }
  uint32_t t = 0;
  bool exact = u.want == 0;  // whether the candidates at or above t are just those kept
  if (!exact) {
#pragma unroll 1
    for (int bit = 31; bit >= 0 && !exact; --bit) {
      const uint32_t cand = t | (1u << bit);
      int c = 0;
#pragma unroll
      for (int e = 0; e < NE; ++e) c += wave_count(r[e] >= cand);
      const int total = block_sum(c, counts[bit & 1]);
      if (total >= u.want) {
        t = cand;
        exact = total == u.want;
      }
    }
  } else {
    t = 0xffffffffu;
  }
  // of the candidates that equal t, the first `ties` (exact: all of them)
  int above = 0, equal = 0;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    above += wave_count(r[e] > t);
    equal += wave_count(r[e] == t && t != 0u);
  }
  if (u.want == 0) above = equal = 0;
  __syncthreads();
  const int all_above = block_sum(above, counts[0]);
  int ties = u.want - all_above, before = 0;
  (void)block_sum(equal, counts[1]);
#pragma unroll
  for (int w = 0; w < kSelThreads / 64; ++w) before += w < wave ? counts[1][w] : 0;
  // rows kept in this wave, its place among the waves', then the rows again
  auto keeps = [&](int e, int& seen) {  // the wave's kept rows among its e-th 64; seen: ties so far
    const int j = j0 + 64 * e;
    const bool cand = u.want > 0 && j >= u.lo && j < u.hi;
    const bool tie = cand && r[e] == t;
    const uint64_t mt = __builtin_amdgcn_ballot_w64(tie);
    const bool keep = (j < u.n && (j < u.lo || j >= u.hi)) || (cand && r[e] > t) ||
                      (tie && seen + __builtin_popcountll(mt & ((1ull << lane) - 1)) < ties);
    seen += __builtin_popcountll(mt);
    return __builtin_amdgcn_ballot_w64(keep);
  };
  int mine = 0, seen = before;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    mine += __builtin_popcountll(keeps(e, seen));
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  (void)block_sum(mine, counts[0]);
  int at = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 64; ++w) at += w < wave ? counts[0][w] : 0;
  seen = before;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const uint64_t on = keeps(e, seen);
    const int i = at + __builtin_popcountll(on & ((1ull << lane) - 1));
    if (((on >> lane) & 1) && i < a.keep) u.out[i] = j0 + 64 * e;
    at += __builtin_popcountll(on);
    __builtin_amdgcn_sched_barrier(0);  // (one mask at a time)
  }
}

// The same for sequences that registers do not hold: the weights are read
// again for every bit.
__global__ __launch_bounds__(kSelThreads) void select_long_kernel(const SelectArgs a) {
  __shared__ int counts[2][kSelThreads / 64];
  __shared__ int above[kSelThreads / 64], equal[kSelThreads / 64];
  const SelectUnit u = select_unit(a);
  if (u.n <= a.keep) {
    select_all(a, u);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t t = 0xffffffffu;
  if (u.want > 0) {
    t = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = t | (1u << bit);
      int c = 0;
      for (int j = u.lo + tid; j - tid < u.hi; j += kSelThreads)
        c += wave_count(j < u.hi && rank_of(u.w[(int64_t)j * a.ws_k]) >= cand);
      if (block_sum(c, counts[bit & 1]) >= u.want) t = cand;
    }
  }
  int c = 0;
  for (int j = u.lo + tid; j - tid < u.hi; j += kSelThreads)
    c += wave_count(j < u.hi && u.want > 0 && rank_of(u.w[(int64_t)j * a.ws_k]) > t);
  __syncthreads();
  const int ties = u.want - block_sum(c, counts[0]);
  // rows in order, 1024 at a time
  int done = 0, taken = 0;  // rows written, ties taken, before this chunk
  for (int r0 = 0; r0 < u.n; r0 += kSelThreads) {
    const int j = r0 + tid;
    const bool cand = u.want > 0 && j >= u.lo && j < u.hi;
    const uint32_t r = cand ? rank_of(u.w[(int64_t)j * a.ws_k]) : 0u;
    const bool sure = j < u.n && (j < u.lo || j >= u.hi || (cand && r > t)), tie = cand && r == t;
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
    if (on && at < a.keep) u.out[at] = j;
    done = sum;
    taken = all;
    __syncthreads();
  }
}

template <int NE>
void launch_select(const SelectArgs& a, unsigned units, hipStream_t st) {
  hipLaunchKernelGGL((select_keys_kernel<NE>), dim3(units), dim3(kSelThreads), 0, st, a);
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
  FastDiv div;                                 // by lpr
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
  uint32_t wg0[kMoveMax];  // first workgroup of each tensor (none: past the last)
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
constexpr int kMovePer = 4;  // pieces a thread moves, all loads before the stores

// Into other buffers: a thread moves pieces of rows; a workgroup's tensor is
// found from the workgroups of those before it, blockIdx.y is the (sequence,
// head). Memory-bound, in pieces of up to 16 bytes of rows that lie apart.
__global__ __launch_bounds__(kMoveThreads) void move_rows_kernel(const MoveArgs a) {
  int k = 0;
#pragma unroll
  for (int x = 1; x < kMoveMax; ++x) k = blockIdx.x >= a.wg0[x] ? x : k;
  const MoveTensor& t = a.t[k];
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H;
  const uint32_t x0 = (blockIdx.x - a.wg0[k]) * (kMoveThreads * kMovePer) + threadIdx.x;
  const uint32_t pieces = (uint32_t)a.n * (uint32_t)t.lpr;
  int64_t s[kMovePer], d[kMovePer];
  int at[kMovePer];
#pragma unroll
  for (int y = 0; y < kMovePer; ++y) {
    const uint32_t x = x0 + y * kMoveThreads, i = fdiv(x, t.div);
    at[y] = (int)(x - i * (uint32_t)t.lpr) * t.unit;
    s[y] = -1;
    if (x < pieces) move_rows_of(a, b, h, (int)i, &s[y], &d[y]);
  }
  const uint8_t* src = t.src + b * t.ss_b + h * t.ss_h;
  uint8_t* dst = t.dst + b * t.ds_b + h * t.ds_h;
  uint4 v[kMovePer];
#pragma unroll
  for (int y = 0; y < kMovePer; ++y)
    if (s[y] >= 0) v[y] = move_load(src + s[y] * t.ss_s + at[y], t.unit);
#pragma unroll
  for (int y = 0; y < kMovePer; ++y)
    if (s[y] >= 0) move_store(dst + d[y] * t.ds_s + at[y], t.unit, v[y]);
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
  int64_t wgs = 0;
  for (int k = 0; k < kMoveMax; ++k) a.wg0[k] = 0xffffffffu;
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
    t.div = make_fastdiv((uint32_t)t.lpr);
    if (in_place) KVQ_CHECK_ARG(n * widths[k] <= kMoveLds, "%s: in place, at most %d bytes of rows a head move (got %lld)",
                                what, kMoveLds, (long long)(n * widths[k]));
    KVQ_CHECK_ARG(n * t.lpr < (int64_t(1) << 31), "%s: too large", what);
    a.wg0[k] = (uint32_t)wgs;
    wgs += (n * t.lpr + kMoveThreads * kMovePer - 1) / (kMoveThreads * kMovePer);
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
    KVQ_CHECK_ARG(wgs < (int64_t(1) << 31), "%s: too large", what);
    hipLaunchKernelGGL(move_rows_kernel, dim3((unsigned)wgs, (unsigned)(B * H)), dim3(kMoveThreads), 0, st, a);
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
  const unsigned units = (unsigned)(B * H);
  hipStream_t st = (hipStream_t)stream;
  if (S <= 2 * kSelThreads) launch_select<2>(a, units, st);
  else if (S <= 8 * kSelThreads) launch_select<8>(a, units, st);
  else if (S <= 16 * kSelThreads) launch_select<16>(a, units, st);
  else if (S <= 32 * kSelThreads) launch_select<32>(a, units, st);
  else if (S <= 64 * kSelThreads) launch_select<64>(a, units, st);
  else hipLaunchKernelGGL(select_long_kernel, dim3(units), dim3(kSelThreads), 0, st, a);
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
