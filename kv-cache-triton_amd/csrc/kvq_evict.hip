// Eviction: which rows of a cache to keep, and moving them (gfx950).
//
// select: per (sequence, KV head) of n keys, the first `sink`, the last
// `recent` and, of the others, those of the greatest weight, `keep` in all,
// as ascending row numbers. Equal weights go to the lowest row; a NaN ranks
// above every number, -0 with +0. The order is that of the weights' bits,
// mapped to unsigned integers that compare as the floats do.
// move: destination row first + i of each tensor is source row index[i].
//
// Measured: 8 heads of 16K rows cut to 2K 13.4 + 3.5 us, 400 heads of 1,100 rows
// 11.5 + 9, 64 heads of 32K rows cut to 8K 23 + 50. The selection is bound by the
// latency of its rounds (one workgroup per head), the move by memory: its rows
// of 64 bytes of codes lie apart, and each fetches a line of 128.
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

// Weights in the order of their floats: NaN above every number, -0 as +0. No
// weight has rank 0 (no row) or 0xffffffff (a row that is always kept).
__device__ __forceinline__ uint32_t rank_of(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

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
template <int NT>
__device__ __forceinline__ void select_all(const SelectArgs& a, const SelectUnit& u) {
  for (int i = threadIdx.x; i < a.keep; i += NT) u.out[i] = i < u.n ? i : -1;
}

// x + the value `lanes` lanes below, by DPP (0 where there is none): control
// words row_shr 1, 2, 4, 8 (within 16 lanes), then row 15's and row 31's last
// lane to the rows above.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int row_prefix(int x) {  // inclusive sum over each 16 lanes
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  return dpp_add<0x118, 0xf>(x);
}
__device__ __forceinline__ int wave_prefix(int x) {  // over the wave
  x = dpp_add<0x142, 0xa>(row_prefix(x));
  return dpp_add<0x143, 0xc>(x);
}

// One workgroup of NT threads per (sequence, KV head). The rank of the last row
// kept is found six bits a round from the top: the rows that share its bits so
// far are counted by their next six, in LDS, in 16 columns (a wave's lanes mostly
// have the same few exponents; in one counter they would wait for each other),
// and the columns added up. It stops as soon as a count
// is exactly what is wanted: after four rounds for weights that spread over the
// floats. Then the kept rows are counted and written in order, each wave a run
// of consecutive rows. Ranks are kept in LDS between the passes (up to CAP
// rows; CAP 0: formed again from the weights each time). Loops stay rolled: a
// few workgroups run this code once, and unrolled over ranks in registers most
// of the time went by until the instructions arrived (16K rows: 31 us so, of
// which the last pass alone took 20).
constexpr int kBits = 6, kBins = 1 << kBits;

template <int NT, int CAP>
__global__ __launch_bounds__(NT) void select_keys_kernel(const SelectArgs a) {
  constexpr int NW = NT / 64;
  __shared__ uint32_t ranks[CAP > 0 ? CAP : 1];
  __shared__ int hist[kBins * 16];
  __shared__ int totals[kBins];
  __shared__ int counts[2][NW];
  const SelectUnit u = select_unit(a);
  if (u.n <= a.keep) {
    select_all<NT>(a, u);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the rank of row j; always kept: the largest, past the sequence: 0
  auto rank_from = [&](int j, float w) {
    const uint32_t x = j < u.lo || j >= u.hi ? 0xffffffffu : rank_of(w);
    return j < u.n ? x : 0u;
  };
  auto load = [&](int j) { return u.w[(int64_t)min(j, u.n - 1) * a.ws_k]; };
  const int per = (u.n + NT - 1) / NT;  // 64-row pieces of a wave
  const int j0 = wave * (64 * per) + lane;
  for (int x = threadIdx.x; x < kBins * 16; x += NT) hist[x] = 0;
  if constexpr (CAP > 0) {
    int e = 0;
    for (; e + 8 <= per; e += 8) {  // (eight loads in flight)
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = load(j0 + 64 * (e + k));
#pragma unroll
      for (int k = 0; k < 8; ++k) ranks[j0 + 64 * (e + k)] = rank_from(j0 + 64 * (e + k), w[k]);
    }
    for (; e < per; ++e) ranks[j0 + 64 * e] = rank_from(j0 + 64 * e, load(j0 + 64 * e));
  }
  auto rank_at = [&](int e) {
    const int j = j0 + 64 * e;
    if constexpr (CAP > 0) return ranks[j];
    else return rank_from(j, load(j));
  };
  __syncthreads();
  uint32_t t = 0;       // the rank's bits so far
  int need = a.keep;    // rows to keep among those that share them
  bool exact = false;   // whether all of those are kept
#pragma unroll 1
  for (int shift = 32 - kBits; !exact; shift -= kBits) {
    const int sh = shift > 0 ? shift : 0;
    const uint32_t low = shift > 0 ? kBins - 1 : (1u << (kBits + shift)) - 1;  // (fewer bits in the last round)
#pragma unroll 4
    for (int e = 0; e < per; ++e) {
      const uint32_t x = rank_at(e) >> sh;
      if (((x ^ (t >> sh)) & ~low) == 0) atomicAdd(&hist[(x & low) * 16 + (lane & 15)], 1);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < kBins * 16; x += NT) {
      const int v = row_prefix(hist[x]);
      hist[x] = 0;
      if ((x & 15) == 15) totals[x >> 4] = v;
    }
    __syncthreads();
    const int mine = totals[kBins - 1 - lane];  // bins from the top
    const int sum = wave_prefix(mine);
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum >= need));
    const int bin = __builtin_amdgcn_readlane(mine, at);
    need -= __builtin_amdgcn_readlane(sum, at) - bin;
    t |= (uint32_t)(kBins - 1 - at) << sh;
    exact = need == bin;
    if (shift <= 0) break;
  }
  // kept: ranks over t, and `need` of those equal to it (exact: t is lowered so
  // that all its rows are over it; no rank of a row is 0)
  if (exact) t -= 1;
  int above = 0, equal = 0;
#pragma unroll 4
  for (int e = 0; e < per; ++e) {
    const uint32_t r = rank_at(e);
    above += r > t ? 1 : 0;
    equal += r == t ? 1 : 0;
  }
  above = __builtin_amdgcn_readlane(wave_prefix(above), 63);
  equal = exact ? 0 : __builtin_amdgcn_readlane(wave_prefix(equal), 63);
  if (lane == 0) {
    counts[0][wave] = above;
    counts[1][wave] = equal;
  }
  __syncthreads();
  int at = 0, seen = 0;  // rows kept, and rows equal to t, before this wave's
  for (int x = 0; x < wave; ++x) {
    at += counts[0][x];
    seen += counts[1][x];
  }
  at = __builtin_amdgcn_readfirstlane(at + min(seen, need));
  seen = __builtin_amdgcn_readfirstlane(seen);
#pragma unroll 2
  for (int e = 0; e < per; ++e) {
    const uint32_t r = rank_at(e);
    bool on = r > t;
    if (!exact) {
      const uint64_t m = __builtin_amdgcn_ballot_w64(r == t);
      on = on || (r == t && seen + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0)) < need);
      seen += __builtin_popcountll(m);
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(on);
    const int i = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    if (on && i < a.keep) u.out[i] = j0 + 64 * e;
    at += __builtin_popcountll(m);
  }
}

template <int NT, int CAP>
void launch_select(const SelectArgs& a, unsigned units, hipStream_t st) {
  hipLaunchKernelGGL((select_keys_kernel<NT, CAP>), dim3(units), dim3(NT), 0, st, a);
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

// Source and destination row of an item, or source -1 (nothing moves): an index
// outside [0, S), a destination outside its rows, a page without a block.
__device__ __forceinline__ void move_rows_of(const MoveArgs& a, int b, int64_t from, int64_t to, int64_t* src, int64_t* dst) {
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

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Pieces of V's size: every load is issued before the first store, and none
// under a condition (a piece that does not move reads row 0), so that all are in
// flight together.
template <typename V>
__device__ __forceinline__ void move_pieces(const MoveArgs& a, const MoveTensor& t, int b, int h, uint32_t x0) {
  const uint32_t pieces = (uint32_t)a.n * (uint32_t)t.lpr;
  const int32_t* index = a.index + b * a.is_b + h * a.is_h;
  const int64_t first = move_first(a, b);
  int64_t s[kMovePer], d[kMovePer];
  int at[kMovePer];
  bool on[kMovePer];
#pragma unroll
  for (int y = 0; y < kMovePer; ++y) {
    const uint32_t x = x0 + y * kMoveThreads, xc = x < pieces ? x : pieces - 1, i = fdiv(xc, t.div);
    at[y] = (int)(xc - i * (uint32_t)t.lpr) * (int)sizeof(V);
    s[y] = index[i * a.is_i];
    d[y] = first + i;
    on[y] = x < pieces;
  }
#pragma unroll
  for (int y = 0; y < kMovePer; ++y) {
    int64_t from, to;
    move_rows_of(a, b, s[y], d[y], &from, &to);
    on[y] = on[y] & (from >= 0);
    s[y] = from < 0 ? 0 : from;
    d[y] = to;
  }
  const uint8_t* src = t.src + b * t.ss_b + h * t.ss_h;
  uint8_t* dst = t.dst + b * t.ds_b + h * t.ds_h;
  V v[kMovePer];
#pragma unroll
  for (int y = 0; y < kMovePer; ++y) v[y] = *(const V*)(src + s[y] * t.ss_s + at[y]);
#pragma unroll
  for (int y = 0; y < kMovePer; ++y)
    if (on[y]) *(V*)(dst + d[y] * t.ds_s + at[y]) = v[y];
}

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
  if (t.unit == 16) move_pieces<u32x4_t>(a, t, b, h, x0);
  else if (t.unit == 8) move_pieces<u32x2_t>(a, t, b, h, x0);
  else if (t.unit == 4) move_pieces<uint32_t>(a, t, b, h, x0);
  else if (t.unit == 2) move_pieces<uint16_t>(a, t, b, h, x0);
  else move_pieces<uint8_t>(a, t, b, h, x0);
}

// In place: one workgroup per tensor, sequence and head reads every row that
// moves into LDS, then writes them, so that any index is right.
constexpr int kMoveLds = 65536;

__global__ __launch_bounds__(kMoveThreads) void move_rows_in_place_kernel(const MoveArgs a) {
  __shared__ __align__(16) uint8_t lds[kMoveLds];
  const MoveTensor t = a.t[blockIdx.y];
  const int h = blockIdx.z % a.H, b = blockIdx.z / a.H;
  const int pieces = a.n * t.lpr;
  const int32_t* index = a.index + b * a.is_b + h * a.is_h;
  const int64_t first = move_first(a, b);
  for (int x = threadIdx.x; x < pieces; x += kMoveThreads) {
    int64_t s, d;
    move_rows_of(a, b, index[(x / t.lpr) * a.is_i], first + x / t.lpr, &s, &d);
    if (s < 0) continue;
    move_store(lds + (int64_t)x * t.unit, t.unit,
               move_load(t.src + b * t.ss_b + h * t.ss_h + s * t.ss_s + (x % t.lpr) * t.unit, t.unit));
  }
  __syncthreads();
  for (int x = threadIdx.x; x < pieces; x += kMoveThreads) {
    int64_t s, d;
    move_rows_of(a, b, index[(x / t.lpr) * a.is_i], first + x / t.lpr, &s, &d);
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
    if (!in_place) {  // no destination may overlap a source
      auto last = [](const int64_t* st, int64_t B, int64_t H, int64_t rows, int64_t width) {
        return (B - 1) * st[0] + (H - 1) * st[1] + (rows - 1) * st[2] + width;
      };
      for (int x = 0; x < n_tensors && B > 0 && S > 0 && n > 0 && dst_rows > 0; ++x) {
        const uint8_t* s0 = (const uint8_t*)src[x];
        const uint8_t* d0 = (const uint8_t*)dst[k];
        KVQ_CHECK_ARG(d0 + last(ds, B, H, dst_rows, widths[k]) <= s0 ||
                          s0 + last(src_strides + 3 * x, B, H, S, widths[x]) <= d0,
                      "%s: a destination overlaps a tensor that is read (in_place moves within one)", what);
      }
    }
    if (in_place) KVQ_CHECK_ARG(n * widths[k] <= kMoveLds, "%s: in place, at most %d bytes of rows a head move (got %lld)",
                                what, kMoveLds, (long long)(n * widths[k]));
    KVQ_CHECK_ARG(n * t.lpr < (int64_t(1) << 31), "%s: too large", what);
    a.wg0[k] = (uint32_t)wgs;
    wgs += (n * t.lpr + kMoveThreads * kMovePer - 1) / (kMoveThreads * kMovePer);
  }
  if (B == 0 || n == 0) return KVQ_OK;
  KVQ_CHECK_ARG(index, "%s: null index", what);
  if (S == 0 || (pm && pm->n_blocks == 0)) return KVQ_OK;  // no row to move
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
  // as few waves as keep a few rows each busy (every wave repeats the rounds'
  // bookkeeping), and no more LDS than the rows need
  if (S <= 2048) launch_select<256, 2048>(a, units, st);
  else if (S <= 8192) launch_select<512, 8192>(a, units, st);
  else if (S <= 32768) launch_select<1024, 32768>(a, units, st);
  else launch_select<1024, 0>(a, units, st);
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
