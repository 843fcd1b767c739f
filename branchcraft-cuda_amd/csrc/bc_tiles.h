// Attention of chunks of new tokens over the paged cache, for gfx950: the
// kernels of bc_chunk_attention and the host code that cuts and launches them.
// Each source file that includes this has its own copies.
#pragma once

#include <type_traits>

#include "bc_device.h"
#include "bc_host.h"
#include "bc_rules.h"

using namespace bcd;

namespace {

constexpr int kThreads = 256;
// Most workgroups of a launch's first dimension: HIP takes fewer than 2^32
// threads.  Work that may need more is gone over in turns.
constexpr int kMostGroups = (1 << 24) - 1;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---------------------------------------------------------------------------
// Attention

struct ChunkParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* pages;
  const int32_t* lengths;
  const int32_t* starts;
  const float* slopes;
  const int32_t* prefix;
  const int32_t* first;
  uint16_t* out;
  long long qt, qh;          // query token and head strides
  long long kp, ks, kh;      // K page, slot and head strides
  long long vp, vs, vh;      // V's
  int tokens, batch, hq, hkv, group, max_pages, phys_pages;
  int causal, window;
  unsigned group_mul;        // ceil(2^32 / group), or 0: see divide
  unsigned hkv_mul;          // the same of hkv
  float scale, cap;
};

struct TileParams {
  ChunkParams c;
  float* part_acc;  // [partial row][Hkv][D]; null: nothing is split
  float* part_ml;   // [partial row][Hkv][2]: maximum and sum
  int4* records;    // two counts, then two int4 per split tile and narrow request
  int target;       // workgroups that a batch's work is cut for
  int waves;        // ranges of the narrow requests' tiles, at most, per KV head
  int most_parts;   // parts of split tiles, at most, per KV head
  int part_rows;    // rows of such a part
  int narrow_rows;  // partial rows of the narrow requests; the others' follow
};

// What the kernels of an 8-bit cache and of groups take on top.  Theirs alone have it
// among their arguments: 48 bytes more there put those that the grid's size follows on
// into another line, and a call of one token over 512 took 8.2 us in place of 7.9.
struct MoreParams {
  TileParams t;
  const uint8_t* k_scale;  // of an 8-bit cache, whose k, v and their strides are in bytes
  const uint8_t* v_scale;
  const int32_t* groups;   // of requests that begin with the same pages
  const int32_t* shared;
  int group_count;
  // With groups, see the entries below: records are one int4 each, of every entry's
  // tiles (the groups' from own_records on), and behind the parts lie the partial
  // rows of tiles in one piece, first those of the requests, then the groups'.
  int single_rows;         // where these begin
  int total_rows;          // all partial rows
  int own_records;
};

template <bool FP8>
using Taken = std::conditional_t<FP8, MoreParams, TileParams>;

template <bool FP8>
const Taken<FP8>& taken(const MoreParams& M) {
  if constexpr (FP8)
    return M;
  else
    return M.t;
}

// Of a kernel that takes them; its ChunkParams begin them.
__device__ __forceinline__ const MoreParams& more(const ChunkParams& C) {
  return reinterpret_cast<const MoreParams&>(C);
}

__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }

template <typename T>
__device__ __forceinline__ float load_elem(const uint16_t* p) {
  return to_float(__builtin_bit_cast(T, *p));
}

template <typename T>
__device__ __forceinline__ uint16_t round_to(float x) {
  return __builtin_bit_cast(uint16_t, (T)x);  // to nearest, ties to even
}

// Two e4m3 codes of a word (its low half, or its high one) times a power of two
// of which `scale` has the exponent, as two values of T in one instruction.
template <typename T, bool HIGH>
__device__ __forceinline__ uint32_t values2(uint32_t codes, float scale) {
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

// The power of two whose biased exponent a byte of an 8-bit cache's scales is.
__device__ __forceinline__ float power_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

constexpr int kFp8Block = BC_FP8_BLOCK;

// Where the scales of a slot and head start, [P][Hkv][16][D / 32].
template <int D>
__device__ __forceinline__ size_t scale_at(const ChunkParams& P, int page, int kvh, int slot) {
  return (((size_t)page * P.hkv + kvh) * BC_PAGE_SIZE + slot) * (D / kFp8Block);
}

// tanh in terms of one exponential, 1 - 2 / (e^2x + 1), which is off by a few
// 2^-24 and so loses small arguments; those take the first terms of the
// series, whose next one is below 2^-24 of x for |x| < 0.3.
__device__ __forceinline__ float tanh_of(float x) {
  const float y = x * x;
  const float small =
      x + x * y * (-1.f / 3.f + y * (2.f / 15.f + y * (-17.f / 315.f + y * (62.f / 2835.f))));
  const float large = 1.f - 2.f * __builtin_amdgcn_rcpf(fast_exp2(x * (2.f * kLog2e)) + 1.f);
  return __builtin_fabsf(x) < 0.3f ? small : large;
}

// The request that row t belongs to: the number of ends at or below t, for
// the whole wave; -1 for a row of none.
__device__ __forceinline__ int request_of(const ChunkParams& P, int t, int lane) {
  int b = 0;
  for (int i = lane; i - lane < P.batch; i += 64) {
    const bool ended = i < P.batch && P.starts[i + 1] <= t;
    b += __popcll(__builtin_amdgcn_ballot_w64(ended));
  }
  return b < P.batch && P.starts[b] <= t ? b : -1;
}

// x / by, as a multiply-high where the host has passed mul = ceil(2^32 / by),
// having seen that it is exact (x * by below 2^32).
__device__ __forceinline__ int divide(int x, int by, unsigned mul) {
  return by == 1 ? x : mul ? (int)__umulhi((unsigned)x, mul) : x / by;
}

__device__ __forceinline__ int by_group(const ChunkParams& P, int r) {
  return divide(r, P.group, P.group_mul);
}

// Inside the table's row, and so a few steps below 2^31 (BC_MAX_TABLE_PAGES).
__device__ __forceinline__ int clamp_len(const ChunkParams& P, int b) {
  return min(max(P.lengths[b], 0), P.max_pages * BC_PAGE_SIZE);
}

// The tokens lo .. hi that row t at position pos of request b sees.
__device__ __forceinline__ int2 row_range(const ChunkParams& P, int b, int t, int pos, int len) {
  int lo = 0, hi = len - 1;
  if (P.causal) hi = min(hi, P.prefix ? max(pos, max(P.prefix[b], 0) - 1) : pos);
  if (P.window > 0) lo = max(lo, max(pos, 0) - P.window + 1);
  if (P.first) lo = max(lo, P.first[t]);
  return pos < 0 ? make_int2(0, -1) : make_int2(lo, hi);
}

// The plain form of the operator, for tensors whose addresses or strides rule
// out 16-byte loads.  One wave per (row, query head): lane j scores token j
// of 64, the online softmax's maximum and sum stay in the wave, and each lane
// keeps D / 64 dimensions of the output.  Tokens that the row does not see
// are never multiplied, whatever their K and V hold.
template <typename T, int D, bool FP8>
__device__ __forceinline__ void attend_row(const ChunkParams& P, int t, int h, int lane) {
  constexpr int R = D / 64;
  const int b = request_of(P, t, lane);
  float acc[R] = {}, m = kNegInf, l = 0.f;
  if (b >= 0) {
    const int len = clamp_len(P, b);
    const int pos = max(P.lengths[b], 0) - (min(P.starts[b + 1], P.tokens) - t);
    const int2 seen = row_range(P, b, t, pos, len);
    const int kvh = h / P.group;
    const uint16_t* const q = P.q + t * P.qt + h * P.qh;
    const int32_t* const row = P.pages + (size_t)b * P.max_pages;
    const float slope = P.slopes ? P.slopes[h] * kLog2e : 0.f;
    // Value e of slot `slot` of a page of K or V.
    auto value = [&](const uint16_t* pool, const uint8_t* scales, long long at, int page, int slot, int e) {
      if constexpr (FP8) {
        const uint8_t code = reinterpret_cast<const uint8_t*>(pool)[at + e];
        const uint8_t power = scales[scale_at<D>(P, page, kvh, slot) + e / kFp8Block];
        return to_float(__builtin_bit_cast(T, (uint16_t)values2<T, false>(code, power_of(power))));
      } else {
        return load_elem<T>(pool + at + e);
      }
    };
    for (int j0 = seen.x & ~63; j0 <= seen.y; j0 += 64) {
      const int j = j0 + lane;
      const int id = j >= seen.x && j <= seen.y ? row[j >> 4] : -1;
      const bool ok = (unsigned)id < (unsigned)P.phys_pages;
      float s = kNegInf;
      if (ok) {
        const long long k = id * P.kp + (j & 15) * P.ks + kvh * P.kh;
        float dot = 0.f;
        for (int d = 0; d < D; ++d) dot += load_elem<T>(q + d) * value(P.k, more(P).k_scale, k, id, j & 15, d);
        s = dot * P.scale;
        if (P.cap > 0.f) s = P.cap * tanh_of(s / P.cap);
        s = s * kLog2e - slope * fabsf((float)(pos - j));
      }
      const float mn = __builtin_fmaxf(m, wave_max(s));
      const float base = safe_max(mn);
      const float alpha = fast_exp2(m - base);
      const float p = ok ? fast_exp2(s - base) : 0.f;
      m = mn;
      l = l * alpha + wave_sum(p);
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r] *= alpha;
      for (unsigned long long left = __builtin_amdgcn_ballot_w64(ok); left; left &= left - 1) {
        const int from = __builtin_ctzll(left), page = __shfl(id, from, 64), slot = (j0 + from) & 15;
        const float w = __shfl(p, from, 64);
        const long long v = page * P.vp + slot * P.vs + kvh * P.vh;
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] += w * value(P.v, more(P).v_scale, v, page, slot, 64 * r + lane);
      }
    }
  }
  uint16_t* const out = P.out + ((size_t)t * P.hq + h) * D;
#pragma unroll
  for (int r = 0; r < R; ++r)
    out[64 * r + lane] = round_to<T>(l > 0.f || l != l ? acc[r] / l : 0.f);
}

template <typename T, int D, bool FP8>
__global__ __launch_bounds__(kThreads) void chunk_rows_kernel(Taken<FP8> A) {
  const ChunkParams& P = reinterpret_cast<const ChunkParams&>(A);  // begins both
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y * (kThreads / 64) + wave;
  if (h >= P.hq) return;
  for (unsigned row = blockIdx.x; row < (unsigned)P.tokens; row += gridDim.x)
    attend_row<T, D, FP8>(P, (int)row, h, lane);
}

template <bool FP8>
hipError_t launch_rows(const MoreParams& M, int dim, int dtype, hipStream_t st) {
  const ChunkParams& P = M.t.c;
  const dim3 grid(P.tokens < kMostGroups ? P.tokens : kMostGroups,
                  (P.hq + kThreads / 64 - 1) / (kThreads / 64));
  if (dtype == BC_FLOAT16) {
    if (dim == 64)
      chunk_rows_kernel<_Float16, 64, FP8><<<grid, kThreads, 0, st>>>(taken<FP8>(M));
    else
      chunk_rows_kernel<_Float16, 128, FP8><<<grid, kThreads, 0, st>>>(taken<FP8>(M));
  } else {
    if (dim == 64)
      chunk_rows_kernel<__bf16, 64, FP8><<<grid, kThreads, 0, st>>>(taken<FP8>(M));
    else
      chunk_rows_kernel<__bf16, 128, FP8><<<grid, kThreads, 0, st>>>(taken<FP8>(M));
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Tiles of rows

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// What differs between the types: the matrix instruction, the rounding of two
// weights to nearest even, and what added to a value's magnitude carries into
// the sign bit where the value is infinite or NaN.
template <typename T>
struct Num;
template <>
struct Num<_Float16> {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kCarry = 0x04000400;
  // Weights are kept at 2^7 of their value relative to the largest: the
  // running maximum may lag by 2^kRescaleSlack, which leaves the largest at
  // most 2^15, and the smallest normal FP16 weight at 2^-21.
  static constexpr float kLift = 7.f;
  static __device__ __forceinline__ float add2(uint32_t w, float sum) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, w), v2{(_Float16)1.f, (_Float16)1.f}, sum,
                                  false);
  }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a),
                                                  __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Num<__bf16> {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kCarry = 0x00800080;
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ float add2(uint32_t w, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w),
                                           v2{(__bf16)1.f, (__bf16)1.f}, sum, false);
  }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a),
                                                   __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_convertvector(f32x2{a, b}, typename Num<T>::v2));
}

constexpr int kStep = 64;       // tokens per step of a tile of rows
using bch::kFewRows;
constexpr int kManyRows = 128;  // rows per workgroup of the wide form
constexpr int kLeastSteps = 4;  // fewest steps per part of a split tile of rows
constexpr int kLeastRun = 4;    // fewest 32-token tiles per wave of the narrow form

// The kernel's arguments, read anew: each phase of the tile kernel loads the
// fields that it needs in one round at its start, and none lives through
// another phase.  Read through the argument itself they were loaded in five
// rounds, most of them spilled to lanes of a vector register.
typedef const __attribute__((address_space(4))) TileParams* Args;

__device__ __forceinline__ const TileParams& reread(Args args) {
  unsigned long long at = (unsigned long long)args;
  asm volatile("" : "+s"(at));
  return *(const TileParams*)(Args)at;
}

__device__ __forceinline__ void pin_plan(const TileParams& P) {
  const ChunkParams& C = P.c;
  asm volatile("" ::"s"(C.starts), "s"(C.lengths), "s"(C.prefix), "s"(C.first), "s"(C.tokens),
               "s"(C.batch), "s"(C.group), "s"(C.hkv), "s"(C.hkv_mul), "s"(C.max_pages),
               "s"(C.causal), "s"(C.window), "s"(P.part_acc), "s"(P.target), "s"(P.waves),
               "s"(P.most_parts));
  __builtin_amdgcn_sched_barrier(0);
}

template <bool FP8>
__device__ __forceinline__ void pin_rows(const TileParams& P) {
  const ChunkParams& C = P.c;
  if constexpr (FP8) asm volatile("" ::"s"(more(C).k_scale), "s"(more(C).v_scale), "s"(C.hkv));
  asm volatile("" ::"s"(C.q), "s"(C.k), "s"(C.v), "s"(C.pages), "s"(C.slopes), "s"(C.first),
               "s"(C.qt), "s"(C.qh), "s"(C.kp), "s"(C.ks), "s"(C.kh), "s"(C.vp), "s"(C.vs),
               "s"(C.vh), "s"(C.group), "s"(C.group_mul), "s"(C.max_pages), "s"(C.phys_pages),
               "s"(C.causal), "s"(C.window), "s"(C.scale), "s"(C.cap));
  __builtin_amdgcn_sched_barrier(0);
}

// The rows of one request (new tokens times group), at rows start .. of the
// step, the first of them at place pos0 of the request.
struct Request {
  int b, start, len, pos0, rows;
  int prefix;  // tokens that all rows see
  // With groups: the entry, the tokens that its group's has (a request's own part
  // starts there), and of a group's entry its members, g1 > g0, whose rows these
  // are (pos0 and prefix have no meaning then).
  int entry, floor, g0, g1;
};

// With groups a batch has an entry per request, for its own tokens, and then one
// per group, for what its members share: the rows of all of them, over the first
// one's pages.  Entries of rows that another entry also has leave partials.
__device__ __forceinline__ bool is_group(const Request& r) { return r.g1 > r.g0; }
__device__ __forceinline__ bool joined(const Request& r) { return r.floor > 0 || is_group(r); }

__device__ __forceinline__ int prefix_of(const ChunkParams& P, int b) {
  return P.prefix && P.causal ? max(P.prefix[b], 0) : 0;
}

template <typename F>
__device__ __forceinline__ int wave_join_i(int x, F f) {
  x = f(x, dpp_i<kDppRowMirror>(x));
  x = f(x, dpp_i<kDppRowHalfMirror>(x));
  x = f(x, dpp_i<kDppQuadXor2>(x));
  x = f(x, dpp_i<kDppQuadXor1>(x));
  x = f(x, __shfl_xor(x, 16, 64));
  return __builtin_amdgcn_readfirstlane(f(x, __shfl_xor(x, 32, 64)));
}

__device__ __forceinline__ int wave_min_i(int x) {
  return wave_join_i(x, [](int a, int b) { return min(a, b); });
}

__device__ __forceinline__ int wave_max_i(int x) {
  return wave_join_i(x, [](int a, int b) { return max(a, b); });
}

__device__ __forceinline__ int lanes_sum(int x) {
  return __builtin_amdgcn_readfirstlane(wave_sum_i(x));
}

// Sums up to and including each lane: inside the 16-lane rows, then the rows'
// last lanes to the rows behind them.
__device__ __forceinline__ int lanes_upto(int x) {
  x += dpp_i<0x111>(x);  // row_shr 1, 2, 4, 8
  x += dpp_i<0x112>(x);
  x += dpp_i<0x114>(x);
  x += dpp_i<0x118>(x);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 of a row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31
  return x;
}

// A request per lane: its rows and its work, as tiles of 128 rows by steps of
// 64 tokens, or, with few rows, as tiles of 32 tokens (one at least, so that
// rows which see nothing are written).
struct Asked {
  int start, n, len, full, rows;
  int tiles, steps;        // of the wide form
  int first_tile, narrow;  // of the narrow form
};

struct AskedEntry : Asked {
  int floor, g0, g1;  // see Request
};

__device__ __forceinline__ int wide_steps(const ChunkParams& P, int span) {
  if (P.causal && P.window > 0) span = min(span, min(P.window, 1 << 29) + kManyRows + kStep);
  return max(1, (span + kStep - 1) / kStep);
}

// The work of a request whose start, n, len, full and rows are known, from token
// `floor` on.  With `tiles` the narrow form's tiles are those that the rows'
// documents reach.
__device__ __forceinline__ void ask_work(const ChunkParams& P, Asked& a, int floor, bool tiles) {
  int tiles_of = 0, steps = 0, first_tile = 0, narrow = 0;
  if (a.rows > kFewRows) {
    tiles_of = (a.rows + kManyRows - 1) / kManyRows;
    steps = wide_steps(P, max(a.len - floor, 0));
  } else if (a.rows > 0) {
    int lo = P.window > 0 ? (int)max(0ll, (long long)a.full - a.n - P.window + 1) : 0;
    if (P.first && tiles) {
      int least = 0x7fffffff;
      for (int i = 0; i < a.n; i += 4)  // four loads at a time
#pragma unroll
        for (int x = 0; x < 4; ++x) least = min(least, P.first[a.start + min(i + x, a.n - 1)]);
      lo = max(lo, least);
    }
    first_tile = min(max(lo, floor), max(a.len - 1, 0)) / 32;
    narrow = max(1, (a.len + 31) / 32 - first_tile);
  }
  a.tiles = tiles_of;
  a.steps = steps;
  a.first_tile = first_tile;
  a.narrow = narrow;
}

__device__ __forceinline__ Asked asked_of(const ChunkParams& P, int b, bool tiles) {
  Asked a{};
  if (b < P.batch) {
    a.start = min(max(P.starts[b], 0), P.tokens);
    a.n = max(min(max(P.starts[b + 1], 0), P.tokens) - a.start, 0);
    a.full = max(P.lengths[b], 0);
    a.len = min(a.full, P.max_pages * BC_PAGE_SIZE);
    a.rows = a.n * P.group;
    ask_work(P, a, 0, tiles);
  }
  return a;
}

// How a batch is cut: a tile of rows into parts of at most `share` steps, the
// narrow requests' tiles, one after another, into ranges of `run`, one per
// wave.  A step of the wide form takes its four waves about as long as half a
// tile of the narrow one takes its wave.  No part is shorter than half a
// share, so there are at most 2 * target / Hkv of them, and at most `waves`
// ranges.
struct Cutting {
  int share, run, narrow;
  int groups;  // workgroups of the narrow requests: four (range, KV head) each
};

// `ROUND`: the shares fill what the narrow requests' workgroups leave of a round;
// else both are cut to the same time, if each had a part of the card to itself.
template <bool ROUND>
__device__ __forceinline__ Cutting cut_batch(const TileParams& P, const Asked& head, int lane) {
  const ChunkParams& C = P.c;
  float work = (float)head.tiles * (float)head.steps;
  int narrow = head.narrow;
  for (int b = 64 + lane; b - lane < C.batch; b += 64) {
    const Asked x = asked_of(C, b, true);
    work += (float)x.tiles * (float)x.steps;
    narrow += x.narrow;
  }
  Cutting c;
  work = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wave_sum(work))));
  c.narrow = lanes_sum(narrow);
  const float share = (work + 0.5f * (float)c.narrow) * (float)C.hkv / (float)P.target;
  const float run = ((float)c.narrow + 2.f * work) / (float)P.waves;
  c.share = max(kLeastSteps, (int)__builtin_fminf(share, 1e9f) + 1);
  c.run = max(min((int)__builtin_fminf(run, 1e9f) + 1, c.narrow), (c.narrow + P.waves - 1) / P.waves);
  c.run = max(c.run, kLeastRun);
  c.groups = ((c.narrow + c.run - 1) / c.run * C.hkv + 3) / 4;
  if (ROUND) {
    const float part = work * (float)C.hkv / (float)max(P.target - c.groups, P.target / 4);
    c.share = max(kLeastSteps, (int)__builtin_fminf(part, 1e9f) + 1);
  }
  return c;
}

// What a workgroup does of the wide form, or, without a workspace, of either:
// part `part` of `parts` of row tile `tile` of a request.
struct Item {
  Request r;
  int tile, part, parts;
  int slot;    // of the first part
  int record;  // of a split tile
  long long items;             // where no item has the index: how many there are
  int records, narrow_records; // likewise
  bool found;
};

// Entry b0 + at of the batch, of which lane `at` holds what is asked.
template <bool FORKS, typename A>
__device__ __forceinline__ Request request_at(const ChunkParams& C, const A& a, int b0, int at) {
  Request r{b0 + at, __builtin_amdgcn_readlane(a.start, at), __builtin_amdgcn_readlane(a.len, at),
            __builtin_amdgcn_readlane(a.full - a.n, at), __builtin_amdgcn_readlane(a.rows, at)};
  if constexpr (FORKS) {
    r.floor = __builtin_amdgcn_readlane(a.floor, at);
    r.g0 = __builtin_amdgcn_readlane(a.g0, at);
    r.g1 = __builtin_amdgcn_readlane(a.g1, at);
    r.entry = r.b;
    if (is_group(r)) {  // those come behind the requests, from a full 64 on
      r.entry += C.batch - (C.batch + 63) / 64 * 64;
      r.b = r.g0;
    }
  }
  r.prefix = prefix_of(C, r.b);
  return r;
}

// Item `idx` of the batch, found by every wave for itself from starts and
// lengths.  A request's last tiles, which see most, come first.  `all`: go to
// the end and count.  Where starts decrease, requests overlap and the grid,
// which is sized for the rows of a step, may end before the items: the records
// counted are those whose writer, the first part's workgroup, is among the
// first `launched` items and has place for its parts.  Both bounds rise from
// one record to the next, so these are the first ones.
__device__ __forceinline__ Item plan_item(const TileParams& P, Asked a, int share, long long idx,
                                          int lane, bool all, int launched) {
  const ChunkParams& C = P.c;
  const bool split = P.part_acc != nullptr;
  Item it{};
  long long before = 0;
  int slots = 0, cut = 0, records = 0, narrow = 0;
  for (int b0 = 0; b0 < C.batch; b0 += 64) {
    if (b0 > 0) a = asked_of(C, b0 + lane, split);
    const int parts = split && a.steps > share ? (a.steps + share - 1) / share : 1;
    const int tiles = split ? a.tiles : a.tiles + (a.narrow > 0);
    const int mine = tiles * parts;
    const int upto = lanes_upto(mine);
    const int total = __builtin_amdgcn_readlane(upto, 63);
    const int cut_parts = parts > 1 ? mine : 0, cut_tiles = parts > 1 ? tiles : 0;
    if (!it.found && idx >= before && idx - before < total) {
      const int local = (int)(idx - before);
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > local));
      it.found = true;
      it.r = request_at<false>(C, a, b0, at);
      it.parts = __builtin_amdgcn_readlane(parts, at);
      const int in = local - __builtin_amdgcn_readlane(upto - mine, at);
      const int nth = it.parts == 1 ? in : in / it.parts;
      it.part = in - nth * it.parts;
      it.tile = __builtin_amdgcn_readlane(tiles, at) - 1 - nth;
      if (it.parts > 1) {
        it.slot = slots + lanes_sum(lane < at ? cut_parts : 0) + in - it.part;
        it.record = cut + lanes_sum(lane < at ? cut_tiles : 0) + nth;
        // Cannot be, see Cutting.
        if (it.slot < 0 || it.slot + it.parts > P.most_parts || it.record < 0 ||
            it.record >= P.most_parts / 2)
          it.parts = 1;
      }
      if (!all) return it;
    }
    if (all && split) {
      const int ahead = (int)max(0ll, min((long long)launched - before, 0x3fffffffll)) - (upto - mine);
      const int places = P.most_parts - slots - (lanes_upto(cut_parts) - cut_parts);
      const int in_grid = ahead > 0 ? (ahead - 1) / parts + 1 : 0;
      records += lanes_sum(min(cut_tiles, min(in_grid, max(places, 0) / parts)));
    }
    before += total;
    if (split) {
      slots += lanes_sum(cut_parts);
      cut += lanes_sum(cut_tiles);
      narrow += __builtin_popcountll(__builtin_amdgcn_ballot_w64(a.narrow > 0));
    }
  }
  it.items = before;
  it.records = min(records, P.most_parts / 2);
  it.narrow_records = narrow;
  return it;
}

// A wave's 32 rows: lane lr of either half has row lr.
template <int D>
struct Rows {
  f32x16 acc[D / 32];  // O^T: dimension 32 dt + 8 (j / 4) + 4 g + j % 4
  float m, l;
  float slope;         // in the scores' units
  int pos, lo, hi;
};

template <int D>
struct Offsets {
  int k[D / 16];       // halves into a staged tile of 32 tokens
  int v[2][D / 32];
};

template <int D>
__device__ __forceinline__ Offsets<D> read_offsets(int lane) {
  const int g = lane >> 5, lr = lane & 31, tg = lane >> 4, tj = lane & 15;
  Offsets<D> o;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) o.k[s] = lr * D + ((2 * s + g) ^ swz<D>(lr)) * 8;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      const int row = 4 * (tg >> 1) + (tj >> 2) + 8 * hf;
      const int dim = 32 * dt + 16 * (tg & 1) + 4 * (tj & 3);
      o.v[hf][dt] = row * D + ((dim >> 3) ^ swz<D>(row)) * 8 + (dim & 7);
    }
  return o;
}

__device__ __forceinline__ u32x4 lds16(const uint16_t* p) {
  return *reinterpret_cast<const u32x4*>(p);
}

// V^T's A operand of 16 tokens: the same token order as the score
// accumulators, tokens 4 g .. and 8 + 4 g ...
__device__ __forceinline__ u32x4 read_v(const uint16_t* lo, const uint16_t* hi) {
  typedef __attribute__((address_space(3))) i16x4* Ptr;
  const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)lo);
  const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)hi);
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  return u32x4{x.x, x.y, y.x, y.y};
}

// How scores become exponents.  All forms end as exp2(scale2 * s - base), with
// one maximum and one product per score in the softmax itself:
//  - Plain: s is the product q.k, scale2 = scale log2 e.
//  - Bias: the same, and the products start from -slope / scale * |p - token|,
//    one FMA per score in place of a zero.
//  - Cap: cap tanh(x) = cap - 2 cap / (e^2x + 1), of which the softmax drops the
//    constant, so s = -1 / (e^2x + 1) and scale2 = 2 cap log2 e; two more
//    transcendentals per score.  That is off by about cap 2^-23, so large caps
//    take s = tanh(x) / 2 by tanh_of.  A bias is added to s in these units.
enum class Form { kPlain, kBias, kCap };
constexpr float kFineCap = 256.f;

__device__ __forceinline__ float scale2_of(const ChunkParams& C, Form form) {
  return (form == Form::kCap ? 2.f * C.cap : C.scale) * kLog2e;
}

// What a score of token t0 + 4 g + off starts from in the biased form.  Without
// a prefix the tokens behind the row's place are masked, so that the distance
// needs no magnitude.
template <int D>
__device__ __forceinline__ float bias_at(const Rows<D>& r, float from, int off) {
  return -r.slope * __builtin_fabsf(from - (float)off);
}

template <int D, int NT>
__device__ __forceinline__ void start_scores(const ChunkParams& C, f32x16 (&sc)[NT], const Rows<D>& r,
                                             int t0, int g) {
  const float from = (float)(r.pos - t0 - 4 * g);
  if (C.causal && !C.prefix) {
    const float at = -r.slope * from;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        sc[i][j] = __builtin_fmaf(r.slope, (float)(32 * i + 8 * (j >> 2) + (j & 3)), at);
  } else {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[i][j] = bias_at(r, from, 32 * i + 8 * (j >> 2) + (j & 3));
  }
}

// The tokens of a step that a row must not take: those before its lo, behind
// its hi, or in pages that are not in the pool.
struct Edges {
  bool lo, hi, pages;
  unsigned long long valid;
};

template <int D, Form FORM, int NT>
__device__ __forceinline__ void finish_scores(const ChunkParams& C, f32x16 (&sc)[NT],
                                              const Rows<D>& r, int t0, int g, const Edges& e) {
  if (FORM == Form::kCap) {
    // The first products to be read here may be the last instruction before a
    // branch, over which the compiler counts no wait states: it left one or two
    // between a matrix instruction and the read of its result, which needs
    // twelve.  (The other forms come to their first read through the masks.)
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
    const float in = C.scale / C.cap;
    if (C.cap <= kFineCap) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sc[i][j] = __builtin_amdgcn_rcpf(-1.f - fast_exp2(sc[i][j] * (in * (2.f * kLog2e))));
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[i][j] = 0.5f * tanh_of(sc[i][j] * in);
    }
    if (C.slopes) {
      const float from = (float)(r.pos - t0 - 4 * g);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[i][j] += bias_at(r, from, 32 * i + 8 * (j >> 2) + (j & 3));
    }
  }
  if (e.hi) {
    const int b = r.hi - t0 - 4 * g;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[i][j] = 32 * i + 8 * (j >> 2) + (j & 3) <= b ? sc[i][j] : kNegInf;
  }
  if (e.lo) {
    const int a = r.lo - t0 - 4 * g;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[i][j] = 32 * i + 8 * (j >> 2) + (j & 3) >= a ? sc[i][j] : kNegInf;
  }
  if (e.pages) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t ok = (uint32_t)(e.valid >> (32 * i)) >> (4 * g);
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[i][j] = (ok >> (8 * (j >> 2) + (j & 3))) & 1u ? sc[i][j] : kNegInf;
    }
  }
}

// Online softmax and O^T += V^T P^T over NT staged tiles.  The maximum moves
// only when it would grow by more than kRescaleSlack.  Weights are rounded to
// T, to nearest, for the product (half a step of T each, as the output's own
// rounding); their sum is of the rounded weights, in 32 bits.
template <typename T, int D, int NT>
__device__ __forceinline__ void weigh(f32x16 (&sc)[NT], Rows<D>& r, const uint16_t* vt,
                                      const Offsets<D>& o, float scale2) {
  constexpr int DT = D / 32, NG = 2 * NT;
  typedef Num<T> N;
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) top = __builtin_fmaxf(top, sc[i][j]);
  top *= scale2;
  if (__builtin_amdgcn_ballot_w64(top > r.m + kRescaleSlack)) {
    const float mnew = __builtin_fmaxf(r.m, __builtin_fmaxf(top, shfl_xor_f(top, 32)));
    const float alpha = fast_exp2(r.m - safe_max(mnew));
    r.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 16; ++j) r.acc[dt][j] *= alpha;
    r.m = mnew;
  }
  const float base = safe_max(r.m) - N::kLift;
  u32x4 pb[2], av[2][DT];
  auto weights = [&](int grp) {
    u32x4 w;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float s0 = sc[grp / 2][8 * (grp % 2) + 2 * x], s1 = sc[grp / 2][8 * (grp % 2) + 2 * x + 1];
      const float p0 = fast_exp2(__builtin_fmaf(s0, scale2, -base));
      const float p1 = fast_exp2(__builtin_fmaf(s1, scale2, -base));
      w[x] = pack2<T>(p0, p1);
      r.l = N::add2(w[x], r.l);
    }
    pb[grp % 2] = w;
  };
  auto values = [&](int grp) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      av[grp % 2][dt] = read_v(vt + grp * 16 * D + o.v[0][dt], vt + grp * 16 * D + o.v[1][dt]);
  };
  values(0);
  weights(0);
#pragma unroll
  for (int grp = 0; grp < NG; ++grp) {
    if (grp + 1 < NG) {
      values(grp + 1);
      weights(grp + 1);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) r.acc[dt] = N::mfma(av[grp % 2][dt], pb[grp % 2], r.acc[dt]);
  }
}

// A weight of zero times an infinity or a NaN is a NaN, so a tile that some
// row does not see whole must have neither in V.  16 bytes of such a tile in
// LDS: zeros where the token is none (`real` false), else zeros for the values
// that are not finite; true if there were any.
template <typename T>
__device__ __forceinline__ bool tidy(u32x4* at, bool real) {
  u32x4 w = *at;
  uint32_t any = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) any |= (w[x] & 0x7fff7fffu) + Num<T>::kCarry;
  any &= 0x80008000u;
  if (real && !any) return false;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const uint32_t odd = ((w[x] & 0x7fff7fffu) + Num<T>::kCarry) & 0x80008000u;
    w[x] &= ~((odd >> 15) * 0xffffu);
  }
  *at = real ? w : u32x4{0, 0, 0, 0};
  return real;
}

// The same of 16 bytes on their way into LDS.
template <typename T>
__device__ __forceinline__ bool tidy_value(u32x4& w, bool real) {
  uint32_t all = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const uint32_t odd = ((w[x] & 0x7fff7fffu) + Num<T>::kCarry) & 0x80008000u;
    all |= odd;
    w[x] = real ? w[x] & ~((odd >> 15) * 0xffffu) : 0u;
  }
  return real && all;
}

// What tidy() took out of the tokens t0 .. t0 + count - 1, added to the rows
// that see it.  Rare, so token by token and from the cache.
template <typename T, int D, bool FP8>
__device__ __forceinline__ void add_untidy(const ChunkParams& C, const Request& it, int kvh, Rows<D>& R,
                                           int t0, int count, int g) {
  const int32_t* const table = C.pages + (size_t)it.b * C.max_pages;
#pragma unroll 1
  for (int j = t0; j < min(t0 + count, it.len); ++j) {
    const int p = table[j >> 4];
    if ((unsigned)p >= (unsigned)C.phys_pages) continue;
    const bool seen = j >= R.lo && j <= R.hi;
    const long long at = p * C.vp + (j & 15) * C.vs + kvh * C.vh + 4 * g;
    const uint16_t* const v = C.v + (FP8 ? 0 : at);
    const uint8_t* const codes = reinterpret_cast<const uint8_t*>(C.v) + (FP8 ? at : 0);
    const uint8_t* const scales = FP8 ? more(C).v_scale + scale_at<D>(C, p, kvh, j & 15) : nullptr;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int jq = 0; jq < 4; ++jq) {
        uint2 w;
        if constexpr (FP8) {
          const uint32_t four = *reinterpret_cast<const uint32_t*>(codes + 32 * dt + 8 * jq);
          const float power = power_of(scales[dt]);
          w = make_uint2(values2<T, false>(four, power), values2<T, true>(four, power));
        } else {
          w = *reinterpret_cast<const uint2*>(v + 32 * dt + 8 * jq);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float f = to_float(__builtin_bit_cast(T, (uint16_t)((x < 2 ? w.x : w.y) >> (16 * (x & 1)))));
          R.acc[dt][4 * jq + x] += seen && !(__builtin_fabsf(f) < -kNegInf) ? f : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
}

// The tokens, of 16 per bit of `pages`, that lie in pages of the pool, and
// below the length, `left` tokens away.
template <int PAGES>
__device__ __forceinline__ unsigned long long tokens_of(int left, int pages) {
  unsigned long long ok = left >= 16 * PAGES ? ~0ull >> (64 - 16 * PAGES) : left > 0 ? (1ull << left) - 1 : 0ull;
#pragma unroll
  for (int q = 0; q < PAGES; ++q)
    if (!((pages >> q) & 1)) ok &= ~(0xffffull << (16 * q));
  return ok;
}

// The pages of a wave's next 64, one per lane: their addresses, so that a tile
// reads them out instead of multiplying, and which lie in the pool (others
// are loaded from page 0 and masked).
template <bool FP8>
struct Pages {
  unsigned long long k, v, in_pool;
  int id;
  __device__ __forceinline__ void take(const ChunkParams& C, int kvh, int page_id) {
    const bool in = (unsigned)page_id < (unsigned)C.phys_pages;
    in_pool = __builtin_amdgcn_ballot_w64(in);
    id = in ? page_id : 0;
    const long long page = id;
    if constexpr (FP8) {
      k = (unsigned long long)C.k + kvh * C.kh + page * C.kp;
      v = (unsigned long long)C.v + kvh * C.vh + page * C.vp;
    } else {
      k = (unsigned long long)(C.k + kvh * C.kh + page * C.kp);
      v = (unsigned long long)(C.v + kvh * C.vh + page * C.vp);
    }
  }
  static __device__ __forceinline__ const void* at(unsigned long long x, int lane) {
    const unsigned hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
    return (const void*)((unsigned long long)hi << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, lane));
  }
};

// Sixteen codes of a page, `off` bytes from its wave-uniform address; STREAM: of what
// a call reads once (64 single tokens over 128-4096 tokens 59 us, 67 without).
template <bool STREAM>
__device__ __forceinline__ u32x4 load_codes(const void* page, unsigned off) {
  typedef const __attribute__((address_space(1))) char* Bytes;
  typedef const __attribute__((address_space(1))) u32x4* Codes;
  const Codes at = (Codes)((Bytes)page + off);
  return STREAM ? __builtin_nontemporal_load(at) : *at;
}

// Sixteen codes as values, the first eight and the others.
template <typename T>
__device__ __forceinline__ void values16(const u32x4& w, float power, u32x4& lo, u32x4& hi) {
  lo = u32x4{values2<T, false>(w[0], power), values2<T, true>(w[0], power), values2<T, false>(w[1], power),
             values2<T, true>(w[1], power)};
  hi = u32x4{values2<T, false>(w[2], power), values2<T, true>(w[2], power), values2<T, false>(w[3], power),
             values2<T, true>(w[3], power)};
}

// Their 16-byte chunks 2 c and 2 c + 1 of row `row` of a tile into LDS.  A write takes
// two turns, since eight lanes have either the even or the odd chunks; an order that
// gives each bank to one lane costs a select per word and is no faster (1096 us for
// 2048 new tokens of 32768, with it 1132; 64 single tokens 59.5 and 59.8).
template <int D>
__device__ __forceinline__ void put_values(const u32x4& lo, const u32x4& hi, uint16_t* tile, int row, int c) {
  *reinterpret_cast<u32x4*>(tile + row * D + ((2 * c) ^ swz<D>(row)) * 8) = lo;
  *reinterpret_cast<u32x4*>(tile + row * D + ((2 * c + 1) ^ swz<D>(row)) * 8) = hi;
}

// Of 64 rising numbers, one per lane, how many are at most `x`.
__device__ __forceinline__ int count_upto(int number, int x) {
  int n = 0;
#pragma unroll
  for (int step = 32; step; step >>= 1) n += __shfl(number, n + step - 1, 64) <= x ? step : 0;
  return n + (__shfl(number, n, 64) <= x ? 1 : 0);
}

// The member of a group that row t, a lane's own, belongs to, the row's place in
// it, and its length.  All lanes of the wave take part.
struct Place {
  int b, pos, len;
};

__device__ __forceinline__ Place place_of(const ChunkParams& P, const Request& group, int t) {
  const int lane = threadIdx.x & 63;
  Place at{group.g1 - 1, 0, 0};
  bool found = false;
  for (int i = group.g0; i < group.g1; i += 64) {
    const int b = min(i + lane, group.g1 - 1);
    const int end = P.starts[b + 1], full = max(P.lengths[b], 0);
    const int n = count_upto(end, t), from = min(n, 63);
    const int pos = __shfl(full, from, 64) - (min(__shfl(end, from, 64), P.tokens) - t);
    const int len = min(__shfl(full, from, 64), P.max_pages * BC_PAGE_SIZE);
    if (!found && n < 64) at = Place{min(i + n, group.g1 - 1), pos, len};
    found = found || n < 64;
    if (!__builtin_amdgcn_ballot_w64(!found)) break;
  }
  return at;
}

// This lane's row of the wave's 32: its token, counted from the request's first new
// one, and its head.
struct RowAt {
  bool real;
  int i, h;
};

__device__ __forceinline__ RowAt row_at(const ChunkParams& C, const Request& it, int r, int kvh) {
  const bool real = r < it.rows;
  const int i = real ? by_group(C, r) : 0, h = kvh * C.group + (real ? r - i * C.group : 0);
  return {real, i, h};
}

// Its Q.
template <int D>
__device__ __forceinline__ void load_q(const ChunkParams& C, const Request& it, const RowAt& row, int g,
                                       u32x4 (&qB)[D / 16]) {
  const int t = it.start + row.i;
  const uint16_t* const q = C.q + t * C.qt + row.h * C.qh + 8 * g;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qB[s] = *reinterpret_cast<const u32x4*>(q + 16 * s);
}

// Its place and what it sees.
template <int D, Form FORM, bool FORKS>
__device__ __forceinline__ void start_rows(const ChunkParams& C, const Request& it, const RowAt& row,
                                           Rows<D>& R) {
  const int t = it.start + row.i;
  R.pos = it.pos0 + row.i;
  int2 seen;
  if (FORKS && is_group(it)) {
    const Place at = place_of(C, it, t);
    R.pos = at.pos;
    seen = row_range(C, at.b, t, at.pos, min(at.len, it.len));
  } else {
    seen = row_range(C, it.b, t, R.pos, it.len);
    if constexpr (FORKS) seen.x = max(seen.x, it.floor);
  }
  R.lo = row.real ? seen.x : 0;
  R.hi = row.real ? seen.y : -1;
  R.slope = 0.f;
  if (FORM != Form::kPlain && C.slopes) {
    const float slope = C.slopes[row.h];
    R.slope = FORM == Form::kCap ? slope / (2.f * C.cap) : slope / C.scale;
  }
  R.m = kNegInf;
  R.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) R.acc[dt][j] = 0.f;
}

// All three.
template <typename T, int D, Form FORM, bool FORKS>
__device__ __forceinline__ void load_rows(const ChunkParams& C, const Request& it, int r, int kvh,
                                          int g, Rows<D>& R, u32x4 (&qB)[D / 16]) {
  const RowAt row = row_at(C, it, r, kvh);
  load_q<D>(C, it, row, g, qB);
  start_rows<D, FORM, FORKS>(C, it, row, R);
}

// Bounds on what rows see: any of them the tokens any_lo .. any_hi at most, all
// of them all_lo .. all_hi.
struct Seen {
  int any_lo, any_hi, all_lo, all_hi;
};

// Of rows r0 .. r1 - 1 of a request, from their places alone (no `first`).
template <bool FORKS>
__device__ __forceinline__ Seen rows_seen(const ChunkParams& C, const Request& rq, int r0, int r1) {
  if (r0 >= r1) return {0x7fffffff, -1, 0, 0x7fffffff};
  const int pa = rq.pos0 + by_group(C, r0), pb = rq.pos0 + by_group(C, r1 - 1), end = rq.len - 1;
  Seen s{0, end, 0, end};
  if (C.causal) {
    s.any_hi = min(end, max(pb, rq.prefix - 1));
    s.all_hi = min(end, max(pa, rq.prefix - 1));
  }
  if (C.window > 0) {
    s.any_lo = max(0, max(pa, 0) - C.window + 1);
    s.all_lo = max(0, max(pb, 0) - C.window + 1);
  }
  if (pa < 0) s.all_hi = -1;  // rows before the request see nothing
  if constexpr (FORKS) {
    s.any_lo = max(s.any_lo, rq.floor);
    s.all_lo = max(s.all_lo, rq.floor);
  }
  return s;
}

// Of the wave's rows as they are.
template <int D>
__device__ __forceinline__ Seen wave_seen(const Rows<D>& R, bool real) {
  const bool some = real && R.lo <= R.hi;
  return {wave_min_i(some ? R.lo : 0x7fffffff), wave_max_i(some ? R.hi : -1),
          wave_max_i(real ? (some ? R.lo : 0x7fffffff) : 0), wave_min_i(real ? R.hi : 0x7fffffff)};
}

// Waits until at most N of the wave's vector loads are on their way.
template <int N>
__device__ __forceinline__ void wait_to() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Ends the wait for Q where it stands.
template <int N>
__device__ __forceinline__ void wait_rows(u32x4 (&qB)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(qB[s]));
}

__device__ __forceinline__ float one_over(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }

template <typename T, int D>
__device__ __forceinline__ uint16_t* out_row(const ChunkParams& C, const Request& rq, int r, int kvh) {
  const int n = by_group(C, r), h = kvh * C.group + r - n * C.group;
  return C.out + ((size_t)(rq.start + n) * C.hq + h) * D;
}

// Where a partial row of a KV head lies, in rows.
__device__ __forceinline__ size_t partial_row(const TileParams& P, int row, int kvh) {
  return (size_t)row * P.c.hkv + kvh;
}

// What the join needs of a split tile of rows: rows row0 .. row0 + rows - 1 of
// the request whose new tokens start at `start`; part p's are the partial
// rows first + p * stride ...
__device__ __forceinline__ void put_record(const TileParams& P, int i, int start, int row0, int rows,
                                           int parts, int first, int stride) {
  P.records[1 + 2 * i] = make_int4(start, row0, rows, parts);
  P.records[2 + 2 * i] = make_int4(first, stride, 0, 0);
}

// With groups: the record of tile `tile` of an entry whose new tokens start at
// `start`.  No two entries have one in common, since the rows of the
// ones before end there.
__device__ __forceinline__ int record_of(const TileParams& P, int entry, int start, int tile) {
  const int from = entry < P.c.batch ? entry : more(P.c).own_records + entry - P.c.batch;
  return from + start * P.c.group / kManyRows + tile;
}

// The partial row of an entry's first row, where a tile is in one piece.
__device__ __forceinline__ int single_row(const TileParams& P, const Request& rq) {
  const int rows = P.c.tokens * P.c.group;
  return more(P.c).single_rows + (is_group(rq) ? rows : 0) + rq.start * P.c.group;
}

// Part p of the tile's rows are the partial rows first + p * stride ...; parts 0:
// there are none.
__device__ __forceinline__ void put_fork_record(const TileParams& P, const Request& rq, int tile, int parts,
                                                int first, int stride) {
  P.records[record_of(P, rq.entry, rq.start, tile)] = make_int4(parts, first, stride, 0);
}

// The wide form: 128 rows per workgroup, 32 per wave, each 64-token step's K
// and V shared through two LDS buffers, which loads straight into LDS fill one
// step ahead; one barrier a step, two workgroups per CU (three at D = 64).
//  - 128 rows: the step's 32 KB from L2 serve 4.2 MFLOP.  32 rows per wave: the
//    output takes 64 registers, and eight waves fit a CU's register file.
//  - Bound at D = 128 by the matrix units and the clock that they leave (2048
//    new tokens over 32768, 32/8 heads: 988 to 1050 us with the clock, 1010 to
//    1080 TFLOP/s; a library product of 8192^3 1246), at D = 64 by the vector
//    units: the same softmax for half the products (32 heads, 512 new tokens
//    over 2048, sixteen of them: 180 us, 670 TFLOP/s).
//  - A full round of workgroups takes 8.6 us, launch included, and 2.1 per step
//    (2048 new tokens over 2048 to 32768, none masked: 75.8 to 1082 us).
//  - FP8: codes come into registers a step ahead and are converted into the buffer
//    of the next one between the products, by two values an instruction with their
//    power in it.  2048 of 32768 1083 to 1130 us: matrix units 43 %, vector units
//    45 %, LDS 44 % of the cycles at 2.1 GHz, none of them full.
template <typename T, int D, Form FORM, bool FP8, bool FORKS>
__device__ __forceinline__ void wide_body(const TileParams& A, Args args, const Item& it, int kvh,
                                          uint16_t* s_kv, Seen* s_seen, int* s_bad) {
  const ChunkParams& C = A.c;
  const Request& rq = it.r;
  constexpr int KS = D / 16, CPR = D / 8;
  constexpr int NX = kStep * CPR / 256;  // chunks per thread and step, of K and of V each
  constexpr int HALF = kStep * D;        // halves of a step's K, then as many of V
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, lr = lane & 31;
  const int tile0 = it.tile * kManyRows, row0 = tile0 + wave * 32;
  const int32_t* const table = C.pages + (size_t)rq.b * C.max_pages;
  auto load_ids = [&](int t) { return table[min(t * 4 + lane, C.max_pages - 1)]; };
  Rows<D> R;
  u32x4 qB[KS];
  Seen mine, wg;
  int t0, tend, ids = 0, ids_next = 0;
  // This part's steps of those that the workgroup's rows see, and its first
  // page ids, ahead of Q's loads where they do not depend on the rows.
  auto range = [&] {
    const int first = wg.any_lo / kStep;
    const int steps = wg.any_hi >= wg.any_lo ? wg.any_hi / kStep - first + 1 : 0;
    t0 = first + (int)((long long)steps * it.part / it.parts);
    tend = first + (int)((long long)steps * (it.part + 1) / it.parts);
    if (t0 < tend) {
      ids = load_ids(t0);
      ids_next = load_ids(t0 + 16);
    }
  };
  if (tid < 4) s_bad[tid] = 0;
  // What a group's rows see depends on their requests, but without a window or
  // documents it is read from its start to its end: its first step goes out ahead of
  // the look at them.
  const bool group = FORKS && is_group(rq), ahead = group && !C.first && C.window == 0;
  auto rows = [&](auto early) {
    if (!C.first && !group) {
      mine = rows_seen<FORKS>(C, rq, row0, min(row0 + 32, rq.rows));
      wg = rows_seen<FORKS>(C, rq, tile0, min(tile0 + kManyRows, rq.rows));
      range();
      load_rows<T, D, FORM, FORKS>(C, rq, row0 + lr, kvh, g, R, qB);
    } else {
      if (ahead) {
        wg.any_lo = 0;
        wg.any_hi = rq.len - 1;
        range();
        if (t0 < tend) early();
      }
      load_rows<T, D, FORM, FORKS>(C, rq, row0 + lr, kvh, g, R, qB);
      mine = wave_seen(R, row0 + lr < rq.rows);
      if (lane == 0) s_seen[wave] = mine;
      __syncthreads();
      wg = s_seen[0];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        wg.any_lo = min(wg.any_lo, s_seen[w].any_lo);
        wg.any_hi = max(wg.any_hi, s_seen[w].any_hi);
        wg.all_lo = max(wg.all_lo, s_seen[w].all_lo);
        wg.all_hi = min(wg.all_hi, s_seen[w].all_hi);
      }
      wg.any_lo = __builtin_amdgcn_readfirstlane(wg.any_lo);
      wg.any_hi = __builtin_amdgcn_readfirstlane(wg.any_hi);
      wg.all_lo = __builtin_amdgcn_readfirstlane(wg.all_lo);
      wg.all_hi = __builtin_amdgcn_readfirstlane(wg.all_hi);
      if (!ahead) range();
    }
  };
  if constexpr (!FORKS) rows([] {});

  const int lrow = tid / CPR, lcol = 8 * (tid % CPR ^ swz<D>(lrow));
  const unsigned koff = (unsigned)(((lrow % BC_PAGE_SIZE) * C.ks + lcol) * 2);
  const unsigned voff = (unsigned)(((lrow % BC_PAGE_SIZE) * C.vs + lcol) * 2);
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)s_kv + wave * 1024);
  Pages<FP8> pg;
  // An 8-bit cache's step goes through registers: codes and their powers are
  // loaded where loads into LDS would be issued, and converted into LDS behind the
  // step's product.
  constexpr int CPR8 = D / 16, NX8 = kStep * CPR8 / 256;  // of 16 codes
  const int crow = wave * (64 / CPR8) + lane / CPR8, ccol = lane % CPR8;
  const unsigned kcode = (unsigned)((crow % BC_PAGE_SIZE) * C.ks + ccol * 16);
  const unsigned vcode = (unsigned)((crow % BC_PAGE_SIZE) * C.vs + ccol * 16);
  u32x4 kc[NX8], vc[NX8];
  uint32_t kx[NX8], vx[NX8];
  auto fetch = [&](int x, int at) {
    const int from = 4 * at + (CPR8 == 8 ? 2 * x + (wave >> 1) : wave);
    kc[x] = load_codes<false>(Pages<FP8>::at(pg.k, from), kcode);
    vc[x] = load_codes<false>(Pages<FP8>::at(pg.v, from), vcode);
    const int page = __builtin_amdgcn_readlane(pg.id, from);
    const size_t scales = scale_at<D>(C, page, kvh, 0);
    const unsigned off = (crow % BC_PAGE_SIZE) * (D / kFp8Block) + ccol / 2;
    kx[x] = more(C).k_scale[scales + off];
    vx[x] = more(C).v_scale[scales + off];
  };
  // ... and what inspect() does; `whole`: nothing.
  auto put = [&](int buf, bool whole, unsigned long long ok) {
    uint16_t* const k = s_kv + buf * (2 * HALF);
    bool bad = false;
#pragma unroll
    for (int x = 0; x < NX8; ++x) {
      const int row = crow + 256 / CPR8 * x;
      u32x4 lo, hi;
      values16<T>(kc[x], power_of(kx[x]), lo, hi);
      put_values<D>(lo, hi, k, row, ccol);
      values16<T>(vc[x], power_of(vx[x]), lo, hi);
      if (!whole) {
        bad |= tidy_value<T>(lo, (ok >> row) & 1u);
        bad |= tidy_value<T>(hi, (ok >> row) & 1u);
      }
      put_values<D>(lo, hi, k + HALF, row, ccol);
    }
    return bad;
  };
  auto issue_chunk = [&](int x, int at, int buf) {
    const int from = 4 * at + (CPR == 16 ? x : 2 * x + (wave >> 1));
    const unsigned dst = lds0 + buf * (4 * HALF) + x * 4096;
    load2_to_lds(Pages<FP8>::at(pg.k, from), Pages<FP8>::at(pg.v, from), koff, voff, dst, dst + 2 * HALF);
  };
  auto first_step = [&] {  // its loads
    pg.take(C, kvh, ids);
#pragma unroll
    for (int x = 0; x < (FP8 ? NX8 : NX); ++x)
      if constexpr (FP8)
        fetch(x, 0);
      else
        issue_chunk(x, 0, 0);
  };
  if constexpr (FORKS) rows(first_step);
  // Steps whole_lo .. whole_hi - 1 are seen whole by every row, given their pages.
  const int whole_lo = wg.all_lo / kStep + (wg.all_lo % kStep != 0);
  const int whole_hi = (min(wg.all_hi, rq.len - 1) + 1) / kStep;
  // Each thread tidies the chunks that its own loads, already waited for,
  // have filled.
  auto inspect = [&](unsigned long long ok, uint16_t* v) {
    bool bad = false;
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      u32x4* const at = reinterpret_cast<u32x4*>(v + (tid + 256 * x) * 8);
      bad |= tidy<T>(at, (ok >> (lrow + 256 / CPR * x)) & 1u);
    }
    return bad;
  };

  const Offsets<D> o = read_offsets<D>(lane);
  const float scale2 = scale2_of(C, FORM);
  bool bad = false;
  int pages = 15;  // of the step at hand, a bit each: in the pool
  if (t0 < tend) {
    if (!ahead) first_step();
    pages = (int)pg.in_pool & 15;
    const bool whole = pages == 15 && t0 >= whole_lo && t0 < whole_hi;
    if constexpr (FP8) {
      bad = put(0, whole, tokens_of<4>(rq.len - t0 * kStep, pages));
    } else {
      wait_loads();
      if (!whole) bad = inspect(tokens_of<4>(rq.len - t0 * kStep, pages), s_kv + HALF);
    }
    bad = __builtin_amdgcn_readfirstlane(__syncthreads_or(bad));
  }
  // The wait for Q belongs here, on every path into the loop: at its first use
  // the compiler's wait, inside the loop, also covers the loads that each step
  // has just issued.
  wait_rows(qB);
  // Products start from the bias where registers allow that.  Over an 8-bit cache, and
  // with groups, at D = 128 some would be spilled, in every step: there it is added
  // behind them, one more instruction a score (8 bits, 2048 new tokens of 16384 612 us,
  // 834 with spills, of 16 bits 535; 4 x 1024 of 4096 312, 429, 280; 64 single tokens
  // over a shared 16384 64, 69).
  constexpr bool kStarts = FORM == Form::kBias && !((FP8 || FORKS) && D == 128);
  // One step, its K and V in buffer `buf`; the next one's loads go out between
  // the score products.
  auto step = [&](auto which, int t) {
    constexpr int buf = decltype(which)::value;
    const uint16_t* const kt = s_kv + buf * (2 * HALF);
    const bool next = t + 1 < tend;
    const int at = (t + 1 - t0) % 16;
    if (at == 0 && next) {
      pg.take(C, kvh, ids_next);
      ids_next = load_ids(t + 17);
    }
    const int pages_n = (int)(pg.in_pool >> (4 * at)) & 15;
    const bool whole_n = !next || (pages_n == 15 && t + 1 >= whole_lo && t + 1 < whole_hi);
    f32x16 sc[2];
    u32x4 kf[2][KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) kf[i][s] = lds16(kt + i * 32 * D + o.k[s]);
    const f32x16 zero = {};
    if (kStarts) start_scores<D, 2>(C, sc, R, t * kStep, g);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[i] = Num<T>::mfma(kf[i][s], qB[s], !kStarts && s == 0 ? zero : sc[i]);
      if (!FP8 && s % 2 == 1 && s / 2 < NX) {
        if (next) issue_chunk(s / 2, at, buf ^ 1);
      }
    }
    if constexpr (FP8) {
      if (next) {
#pragma unroll
        for (int x = 0; x < NX8; ++x) fetch(x, at);
      }
    }
    Edges e{t * kStep < mine.all_lo, t * kStep + kStep - 1 > mine.all_hi, pages != 15, 0};
    if (e.pages) e.valid = tokens_of<4>(rq.len - t * kStep, pages);
    if (FORM == Form::kBias && !kStarts) {
      f32x16 bias[2];
      start_scores<D, 2>(C, bias, R, t * kStep, g);
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[i] += bias[i];
    }
    finish_scores<D, FORM, 2>(C, sc, R, t * kStep, g, e);
    // The softmax and its product ahead of other waves' score products, so that
    // the two of a SIMD do not fall into step: 4096 of 4096 tokens (D = 128) 167
    // -> 156 us, 2048 of 32768 1070 -> 1034; at D = 64 and with a cap it takes 2
    // to 4 % more.
    constexpr bool kAhead = D == 128 && FORM != Form::kCap;
    if (kAhead) __builtin_amdgcn_s_setprio(2);
    weigh<T, D, 2>(sc, R, kt + HALF, o, scale2);
    if (kAhead) __builtin_amdgcn_s_setprio(0);
    if (bad) add_untidy<T, D, FP8>(C, rq, kvh, R, t * kStep, kStep, g);
    if constexpr (!FP8) wait_loads();
    // Step s of the part sets flag s % 4 before the barrier that ends the step
    // before it; the flag is read behind that barrier and cleared behind the
    // next, two barriers before it is set again.
    const int s = t - t0;
    if constexpr (FP8) {
      if (next && put(buf ^ 1, whole_n, tokens_of<4>(rq.len - (t + 1) * kStep, pages_n)))
        s_bad[(s + 1) & 3] = 1;
    } else if (!whole_n && inspect(tokens_of<4>(rq.len - (t + 1) * kStep, pages_n),
                                   s_kv + (buf ^ 1) * (2 * HALF) + HALF)) {
      s_bad[(s + 1) & 3] = 1;
    }
    __syncthreads();
    if (bad && tid == 0) s_bad[s & 3] = 0;
    bad = !whole_n && __builtin_amdgcn_readfirstlane(s_bad[(s + 1) & 3]);
    pages = pages_n;
  };
  for (int t = t0; t < tend; t += 2) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + 1 < tend) step(std::integral_constant<int, 1>{}, t + 1);
  }

  const TileParams& P = reread(args);
  R.l += shfl_xor_f(R.l, 32);
  const int r = row0 + lr;
  if (it.parts > 1 || (FORKS && joined(rq))) {
    const int first = FORKS && it.parts == 1 ? single_row(P, rq) + tile0
                                             : P.narrow_rows + (it.slot + it.part) * P.part_rows;
    const size_t at = partial_row(P, first + wave * 32 + lr, kvh);
    if (r < rq.rows) {
      if (g == 0) *reinterpret_cast<float2*>(P.part_ml + 2 * at) = make_float2(R.m, R.l);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int jq = 0; jq < 4; ++jq)
          *reinterpret_cast<float4*>(P.part_acc + at * D + 32 * dt + 8 * jq + 4 * g) =
              make_float4(R.acc[dt][4 * jq], R.acc[dt][4 * jq + 1], R.acc[dt][4 * jq + 2],
                          R.acc[dt][4 * jq + 3]);
    }
    return;
  }
  // Rows leave through LDS, each wave's in its own part of the staged tiles
  // (all read by now), so that a store covers whole rows.
  const float inv = one_over(R.l);
  uint16_t* const out = s_kv + wave * 32 * D;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int jq = 0; jq < 4; ++jq)
      *reinterpret_cast<uint2*>(out + lr * D + ((4 * dt + jq) ^ (lr % CPR)) * 8 + 4 * g) =
          make_uint2(pack2<T>(R.acc[dt][4 * jq] * inv, R.acc[dt][4 * jq + 1] * inv),
                     pack2<T>(R.acc[dt][4 * jq + 2] * inv, R.acc[dt][4 * jq + 3] * inv));
  wave_lds_sync();
  constexpr int RPS = 64 / CPR;  // rows per store
#pragma unroll
  for (int i = 0; i < 32; i += RPS) {
    const int row = i + lane / CPR, c = lane % CPR;
    const u32x4 w = lds16(out + row * D + (c ^ (row % CPR)) * 8);
    const int rr = row0 + row;
    if (rr < rq.rows) *reinterpret_cast<u32x4*>(out_row<T, D>(P.c, rq, rr, kvh) + 8 * c) = w;
  }
}

// A tile's two pages, N loads of 1 KB each, one after another in LDS, of what a
// call reads once: the lines are marked for early replacement.  64 single tokens
// over 128-4096 tokens (32/8 heads, D = 128) 122 -> 108 us.  The bases' five wait
// states (see load2_to_lds) stand before the first.
template <int N>
__device__ __forceinline__ void stream_to_lds(const void* base0, const void* base1,
                                              const unsigned (&off)[N], unsigned dst) {
  static_assert(N == 2 || N == 4, "loads per page");
#define BC_LOAD(OFF, BASE) "global_load_lds_dwordx4 %" #OFF ", %" #BASE " nt\n\t"
#define BC_NEXT "s_add_u32 m0, m0, 1024\n\ts_nop 0\n\t"
  if constexpr (N == 2)
    asm volatile("s_mov_b32 m0, %4\n\ts_nop 3\n\t"
                 BC_LOAD(0, 2) BC_NEXT BC_LOAD(1, 2) BC_NEXT BC_LOAD(0, 3) BC_NEXT BC_LOAD(1, 3)
                 :
                 : "v"(off[0]), "v"(off[1]), "s"(base0), "s"(base1), "s"(dst)
                 : "memory", "scc");
  else
    asm volatile("s_mov_b32 m0, %6\n\ts_nop 3\n\t"
                 BC_LOAD(0, 4) BC_NEXT BC_LOAD(1, 4) BC_NEXT BC_LOAD(2, 4) BC_NEXT BC_LOAD(3, 4) BC_NEXT
                 BC_LOAD(0, 5) BC_NEXT BC_LOAD(1, 5) BC_NEXT BC_LOAD(2, 5) BC_NEXT BC_LOAD(3, 5)
                 :
                 : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base0), "s"(base1), "s"(dst)
                 : "memory", "scc");
#undef BC_LOAD
#undef BC_NEXT
}

// A wave's stream of 32-token tiles through its own part of LDS: K of the next
// tile goes out behind the scores, V behind the product, and no barrier.
template <typename T, int D, Form FORM>
struct Stream {
  static constexpr int KS = D / 16, CPR = D / 8;
  static constexpr int RPL = 64 / CPR;         // token rows per load
  static constexpr int NL = 32 / RPL;          // loads per tile, of K and of V each
  static constexpr int NV = D == 128 ? 4 : 2;  // lane offsets: the swizzle repeats every 16 rows
  static constexpr int TILE = 32 * D;
  static_assert(NL / NV == 2 && NV * RPL == BC_PAGE_SIZE, "a tile is two pages");

  const ChunkParams& C;
  int kvh, lane;
  uint16_t* kt;
  unsigned lds0, koff[NV], voff[NV];
  Offsets<D> o;
  Pages<false> pg;

  __device__ __forceinline__ Stream(const ChunkParams& c, int head, uint16_t* area)
      : C(c), kvh(head), lane(threadIdx.x & 63), kt(area), o(read_offsets<D>(threadIdx.x & 63)) {
    lds0 = __builtin_amdgcn_readfirstlane(
        (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)area);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = i * RPL + lane / CPR, col = 8 * (lane % CPR ^ swz<D>(row));
      koff[i] = (unsigned)((row * C.ks + col) * 2);
      voff[i] = (unsigned)((row * C.vs + col) * 2);
    }
  }
  // Lane i: page i % 2 of tile t + apart * (i / 2).
  __device__ __forceinline__ int ids(int b, int t, int apart) const {
    const int i = 2 * (t + apart * (lane >> 1)) + (lane & 1);
    return C.pages[(size_t)b * C.max_pages + min(i, C.max_pages - 1)];
  }
  __device__ __forceinline__ void issue(unsigned long long x, int at, const unsigned (&off)[NV],
                                        unsigned dst) const {
    stream_to_lds<NV>(Pages<false>::at(x, 2 * at), Pages<false>::at(x, 2 * at + 1), off, dst);
  }
  __device__ __forceinline__ void issue_k(int at) const { issue(pg.k, at, koff, lds0); }
  __device__ __forceinline__ void issue_v(int at) const { issue(pg.v, at, voff, lds0 + 2 * TILE); }
  __device__ __forceinline__ int in_pool(int at) const { return (int)(pg.in_pool >> (2 * at)) & 3; }

  // The staged tile's scores; K has been read when this returns.
  __device__ __forceinline__ void scores(f32x16 (&sc)[1], const u32x4 (&qB)[KS], const Rows<D>& R,
                                         int t) const {
    wait_to<NL>();  // K is there, V may be not
    const f32x16 zero = {};
    if (FORM == Form::kBias) start_scores<D, 1>(C, sc, R, t * 32, lane >> 5);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      sc[0] = Num<T>::mfma(lds16(kt + o.k[s]), qB[s], FORM != Form::kBias && s == 0 ? zero : sc[0]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // Their softmax and product with V, behind which `next` K loads may be on
  // their way; V has been read when this returns.
  __device__ __forceinline__ void product(f32x16 (&sc)[1], const Request& rq, Rows<D>& R, const Seen& mine,
                                          int t, int pages, bool next) const {
    const int g = lane >> 5, left = rq.len - t * 32;
    uint16_t* const vt = kt + TILE;
    const Edges e{t * 32 < mine.all_lo, t * 32 + 31 > mine.all_hi, pages != 3, tokens_of<2>(left, pages)};
    finish_scores<D, FORM, 1>(C, sc, R, t * 32, g, e);
    if (next) wait_to<NL>();  // V is there
    else wait_loads();
    bool bad = false;
    if (e.lo || e.hi || e.pages || left < 32) {
#pragma unroll
      for (int c = 0; c < NL; ++c)
        bad |= tidy<T>(reinterpret_cast<u32x4*>(vt + c * 512 + lane * 8), (e.valid >> (c * RPL + lane / CPR)) & 1u);
      bad = __builtin_amdgcn_ballot_w64(bad) != 0;
      wave_lds_sync();
    }
    weigh<T, D, 1>(sc, R, vt, o, scale2_of(C, FORM));
    if (bad) add_untidy<T, D, false>(C, rq, kvh, R, t * 32, 32, g);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
};

// The same over an 8-bit cache.  Codes come into registers and are converted into
// LDS ahead of their use, where the rest is as for 16 bits; the next tile's go out
// as soon as that has freed their registers.  A lane's load has 16 codes
// of a row; the powers of a tile, 32 rows of K and 32 of V, come a row per lane in
// one load, from where the lanes take their row's.
// 64 single tokens over 128-4096 tokens (302 MB): 57 us, 5.3 TB/s, of which HBM would
// take 46: half the bytes per tile of the 16-bit form at the same work in LDS, whose
// cycles are 46 % (products 16 %, vector units 37 %).
template <typename T, int D, Form FORM>
struct Stream8 {
  static constexpr int KS = D / 16, CPR = D / 16;
  static constexpr int RPL = 64 / CPR;  // token rows per load
  static constexpr int NL = 32 / RPL;   // loads per tile, of K and of V each
  static constexpr int NP = NL / 2;     // loads per page
  static constexpr int TILE = 32 * D;
  static_assert(NP * RPL == BC_PAGE_SIZE, "a tile is two pages");
  typedef typename std::conditional<D == 128, uint32_t, uint16_t>::type Powers;

  const ChunkParams& C;
  int kvh, lane;
  uint16_t* kt;
  unsigned koff[NP], voff[NP];
  Offsets<D> o;
  Pages<true> pg;
  u32x4 k[NL], v[NL];
  uint32_t powers, powers_next;  // of the tile at hand, and of the one on its way

  __device__ __forceinline__ Stream8(const ChunkParams& c, int head, uint16_t* area)
      : C(c), kvh(head), lane(threadIdx.x & 63), kt(area), o(read_offsets<D>(threadIdx.x & 63)) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = i * RPL + lane / CPR, col = lane % CPR * 16;
      koff[i] = (unsigned)(row * C.ks + col);
      voff[i] = (unsigned)(row * C.vs + col);
    }
  }
  __device__ __forceinline__ int ids(int b, int t, int apart) const {
    const int i = 2 * (t + apart * (lane >> 1)) + (lane & 1);
    return C.pages[(size_t)b * C.max_pages + min(i, C.max_pages - 1)];
  }
  __device__ __forceinline__ void issue_k(int at) {
    const int page = __shfl(pg.id, 2 * at + ((lane >> 4) & 1), 64);
    const uint8_t* const scales = lane < 32 ? more(C).k_scale : more(C).v_scale;
    powers_next = *reinterpret_cast<const Powers*>(scales + scale_at<D>(C, page, kvh, lane & 15));
#pragma unroll
    for (int i = 0; i < NL; ++i) k[i] = load_codes<true>(Pages<true>::at(pg.k, 2 * at + i / NP), koff[i % NP]);
  }
  __device__ __forceinline__ void issue_v(int at) {
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = load_codes<true>(Pages<true>::at(pg.v, 2 * at + i / NP), voff[i % NP]);
  }
  __device__ __forceinline__ int in_pool(int at) const { return (int)(pg.in_pool >> (2 * at)) & 3; }

  __device__ __forceinline__ float power(int row) const {  // of this lane's codes of row `row` (V's from 32)
    return power_of(((uint32_t)__shfl((int)powers, row, 64) >> (8 * (lane % CPR / 2))) & 255u);
  }

  // As in Stream, but for the next tile's loads, which these issue (`next`, at `at`).
  __device__ __forceinline__ void scores(f32x16 (&sc)[1], const u32x4 (&qB)[KS], const Rows<D>& R, int t,
                                         bool next, int at) {
    powers = powers_next;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = i * RPL + lane / CPR;
      u32x4 lo, hi;
      values16<T>(k[i], power(row), lo, hi);
      put_values<D>(lo, hi, kt, row, lane % CPR);
    }
    if (next) issue_k(at);
    wave_lds_sync();
    const f32x16 zero = {};
    if (FORM == Form::kBias) start_scores<D, 1>(C, sc, R, t * 32, lane >> 5);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      sc[0] = Num<T>::mfma(lds16(kt + o.k[s]), qB[s], FORM != Form::kBias && s == 0 ? zero : sc[0]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  __device__ __forceinline__ void product(f32x16 (&sc)[1], const Request& rq, Rows<D>& R, const Seen& mine,
                                          int t, int pages, bool next, int at) {
    const int g = lane >> 5, left = rq.len - t * 32;
    uint16_t* const vt = kt + TILE;
    const Edges e{t * 32 < mine.all_lo, t * 32 + 31 > mine.all_hi, pages != 3, tokens_of<2>(left, pages)};
    finish_scores<D, FORM, 1>(C, sc, R, t * 32, g, e);
    const bool edge = e.lo || e.hi || e.pages || left < 32;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = i * RPL + lane / CPR;
      u32x4 lo, hi;
      values16<T>(v[i], power(32 + row), lo, hi);
      if (edge) {
        bad |= tidy_value<T>(lo, (e.valid >> row) & 1u);
        bad |= tidy_value<T>(hi, (e.valid >> row) & 1u);
      }
      put_values<D>(lo, hi, vt, row, lane % CPR);
    }
    if (next) issue_v(at);
    bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    wave_lds_sync();
    weigh<T, D, 1>(sc, R, vt, o, scale2_of(C, FORM));
    if (bad) add_untidy<T, D, true>(C, rq, kvh, R, t * 32, 32, g);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
};

template <typename T, int D, Form FORM, bool FP8>
using StreamOf = typename std::conditional<FP8, Stream8<T, D, FORM>, Stream<T, D, FORM>>::type;

// The narrow form over a batch: the tiles of all requests with few rows, one
// after another, in ranges of equal length, a range per wave.  HBM-bound: 64
// single tokens over 128-4096 tokens (32/8 heads, D = 128, 585 MB) 96 us, 6.5
// TB/s in this kernel; with a part of a request per workgroup, the longest
// parts last, it took 127.  The waves of a workgroup take the KV heads of one
// range, whose lines lie side by side; four waves per CU 96 us, eight 99.
// A request that a range holds whole leaves as output rows, of others each
// range leaves a partial.  Range r's partial of a request whose predecessors
// have n rows starts at partial row 32 r + n: a range's next request is
// further by the rows of the last one, a request's next range by 32.
// `ask(b0)` is what is asked of the requests (with groups: entries) b0 .. b0 + 63,
// `a` of the first, and `batch` how many there are.
template <typename T, int D, Form FORM, bool FP8, bool FORKS, typename A, typename F>
__device__ __forceinline__ void flat_body(const TileParams& P, A a, int batch, F ask, const Cutting& cut,
                                          uint16_t* s_kv) {
  const ChunkParams& C = P.c;
  const int lane = threadIdx.x & 63, g = lane >> 5, lr = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned task = 4 * blockIdx.x + wave;
  const int range = task / (unsigned)C.hkv, kvh = task - (unsigned)range * C.hkv;
  if ((long long)range * cut.run >= cut.narrow) return;
  const int lo = range * cut.run, hi = min(lo + cut.run, cut.narrow);
  // The requests that the range meets, one after another.
  struct Part {
    Request rq;
    int x0, tiles, first_tile, nth, row;
  };
  int b0 = 0, before = 0, rows_before = 0, nth = 0;
  int upto, rows, rows_upto;
  unsigned long long some, left;
  auto look = [&] {  // at the 64 requests from b0 on
    upto = lanes_upto(a.narrow);
    rows = a.narrow > 0 ? a.rows : 0;
    rows_upto = lanes_upto(rows);
    some = __builtin_amdgcn_ballot_w64(a.narrow > 0);
    left = some & __builtin_amdgcn_ballot_w64(before + upto > lo && before + upto - a.narrow < hi);
  };
  look();
  auto next_part = [&](Part& p) {
    while (!left) {
      before += __builtin_amdgcn_readlane(upto, 63);
      rows_before += __builtin_amdgcn_readlane(rows_upto, 63);
      nth += __builtin_popcountll(some);
      b0 += 64;
      if (b0 >= batch || before >= hi) return false;
      a = ask(b0);
      look();
    }
    const int at = __builtin_ctzll(left);
    left &= left - 1;
    p.rq = request_at<FORKS>(C, a, b0, at);
    p.tiles = __builtin_amdgcn_readlane(a.narrow, at);
    p.x0 = before + __builtin_amdgcn_readlane(upto, at) - p.tiles;
    p.first_tile = __builtin_amdgcn_readlane(a.first_tile, at);
    p.nth = nth + __builtin_popcountll(some & ((1ull << at) - 1));
    p.row = rows_before + __builtin_amdgcn_readlane(rows_upto - rows, at);
    return true;
  };
  auto first_of = [&](const Part& p) { return p.first_tile + max(lo, p.x0) - p.x0; };

  Part p;
  if (!next_part(p)) return;
  StreamOf<T, D, FORM, FP8> st(C, kvh, s_kv + wave * (64 * D));
  int t = first_of(p), at = 0;
  st.pg.take(C, kvh, st.ids(p.rq.b, t, 1));
  int ids_next = st.ids(p.rq.b, t + 32, 1);
  int pages = st.in_pool(0);
  st.issue_k(0);
  st.issue_v(0);
  // With groups a request's own part is short for a wave: Q comes a request ahead.
  constexpr bool kAhead = FORKS && FORM != Form::kCap;
  u32x4 q_next[D / 16];
  if constexpr (kAhead) load_q<D>(C, p.rq, row_at(C, p.rq, lr, kvh), g, q_next);
  for (;;) {  // over the requests
    Rows<D> R;
    u32x4 qB[D / 16];
    if constexpr (kAhead) {
      start_rows<D, FORM, FORKS>(C, p.rq, row_at(C, p.rq, lr, kvh), R);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) qB[s] = q_next[s];
    } else {
      load_rows<T, D, FORM, FORKS>(C, p.rq, lr, kvh, g, R, qB);
    }
    const Seen mine = C.first || (FORKS && is_group(p.rq)) ? wave_seen(R, lr < p.rq.rows)
                                                           : rows_seen<FORKS>(C, p.rq, 0, p.rq.rows);
    const int tend = p.first_tile + min(hi, p.x0 + p.tiles) - p.x0;
    // The next request's first pages, so that its first tile follows this
    // one's last as any tile follows another.
    Part n;
    const bool more = next_part(n);
    const int ids_more = more ? st.ids(n.rq.b, first_of(n), 1) : 0;
    wait_rows(qB);
    if constexpr (kAhead) {
      if (more) load_q<D>(C, n.rq, row_at(C, n.rq, lr, kvh), g, q_next);
    }
    for (;; ++t) {
      f32x16 sc[1];
      const bool same = t + 1 < tend, next = same || more;
      int pages_n = 3;
      auto go_on = [&] {  // to the next tile's pages
        if (!next) return;
        at = same ? (at + 1) % 32 : 0;
        if (at == 0) {
          st.pg.take(C, kvh, same ? ids_next : ids_more);
          ids_next = same ? st.ids(p.rq.b, t + 33, 1) : st.ids(n.rq.b, first_of(n) + 32, 1);
        }
        pages_n = st.in_pool(at);
      };
      if constexpr (FP8) {
        go_on();
        st.scores(sc, qB, R, t, next, at);
        st.product(sc, p.rq, R, mine, t, pages, next, at);
      } else {
        st.scores(sc, qB, R, t);
        go_on();
        if (next) st.issue_k(at);
        st.product(sc, p.rq, R, mine, t, pages, next);
        if (next) st.issue_v(at);
      }
      pages = pages_n;
      if (!same) break;
    }
    R.l += shfl_xor_f(R.l, 32);
    const int from = p.x0 / cut.run, parts = (p.x0 + p.tiles - 1) / cut.run - from + 1;
    const bool single = FORKS && parts == 1 && joined(p.rq);
    const int first = single ? single_row(P, p.rq) : p.row + 32 * from;
    // Partials past their place cannot be unless starts decrease.
    const bool fits = single || first + 32 * (parts - 1) + p.rq.rows <= P.narrow_rows;
    if (p.x0 >= lo && kvh == 0 && lane == 0) {
      if constexpr (FORKS)
        put_fork_record(P, p.rq, 0, fits ? parts : 0, first, 32);
      else
        put_record(P, P.most_parts / 2 + p.nth, p.rq.start, 0, p.rq.rows, fits ? parts : 0, first, 32);
    }
    if (parts == 1 && !single) {
      const float inv = one_over(R.l);
      if (lr < p.rq.rows) {
        uint16_t* const out = out_row<T, D>(C, p.rq, lr, kvh) + 4 * g;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int jq = 0; jq < 4; ++jq)
            *reinterpret_cast<uint2*>(out + 32 * dt + 8 * jq) =
                make_uint2(pack2<T>(R.acc[dt][4 * jq] * inv, R.acc[dt][4 * jq + 1] * inv),
                           pack2<T>(R.acc[dt][4 * jq + 2] * inv, R.acc[dt][4 * jq + 3] * inv));
      }
    } else {
      const int row = first + 32 * (range - from) + lr;
      if (lr < p.rq.rows && fits) {
        const size_t to_row = partial_row(P, row, kvh);
        if (g == 0) *reinterpret_cast<float2*>(P.part_ml + 2 * to_row) = make_float2(R.m, R.l);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int jq = 0; jq < 4; ++jq)
            *reinterpret_cast<float4*>(P.part_acc + to_row * D + 32 * dt + 8 * jq + 4 * g) =
                make_float4(R.acc[dt][4 * jq], R.acc[dt][4 * jq + 1], R.acc[dt][4 * jq + 2],
                            R.acc[dt][4 * jq + 3]);
      }
    }
    if (!more) return;
    p = n;
    t = first_of(p);
  }
}

// The narrow form without a workspace: a workgroup per request and KV head,
// its waves every fourth tile each; the four states meet at the end.
template <typename T, int D, Form FORM, bool FP8>
__device__ __forceinline__ void narrow_body(const ChunkParams& C, const Request& rq, int kvh,
                                            uint16_t* s_kv, float2* s_ml) {
  constexpr int TILE = 32 * D;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, lr = lane & 31;
  Rows<D> R;
  u32x4 qB[D / 16];
  load_rows<T, D, FORM, false>(C, rq, lr, kvh, g, R, qB);
  const Seen mine = C.first ? wave_seen(R, lr < rq.rows) : rows_seen<false>(C, rq, 0, rq.rows);
  StreamOf<T, D, FORM, FP8> st(C, kvh, s_kv + wave * (2 * TILE));
  int t = mine.any_hi < mine.any_lo ? 1 : mine.any_lo / 32 + wave;
  const int tend = mine.any_hi < mine.any_lo ? 0 : mine.any_hi / 32 + 1;
  if (t < tend) {
    st.pg.take(C, kvh, st.ids(rq.b, t, 4));
    int ids_next = st.ids(rq.b, t + 128, 4), at = 0, pages = st.in_pool(0);
    st.issue_k(0);
    st.issue_v(0);
    wait_rows(qB);
    for (; t < tend; t += 4) {
      f32x16 sc[1];
      const bool next = t + 4 < tend;
      int pages_n = 3;
      auto go_on = [&] {
        if (!next) return;
        at = (at + 1) % 32;
        if (at == 0) {
          st.pg.take(C, kvh, ids_next);
          ids_next = st.ids(rq.b, t + 132, 4);
        }
        pages_n = st.in_pool(at);
      };
      if constexpr (FP8) {
        go_on();
        st.scores(sc, qB, R, t, next, at);
        st.product(sc, rq, R, mine, t, pages, next, at);
      } else {
        st.scores(sc, qB, R, t);
        go_on();
        if (next) st.issue_k(at);
        st.product(sc, rq, R, mine, t, pages, next);
        if (next) st.issue_v(at);
      }
      pages = pages_n;
    }
  }

  // The four states through LDS: four-float chunk c of row r at c ^ (r % (D / 4)).
  R.l += shfl_xor_f(R.l, 32);
  float* const acc = reinterpret_cast<float*>(st.kt);
  wave_lds_sync();
  if (lr < rq.rows) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int jq = 0; jq < 4; ++jq)
        *reinterpret_cast<float4*>(acc + lr * D + (((8 * dt + 2 * jq + g) ^ (lr % (D / 4))) << 2)) =
            make_float4(R.acc[dt][4 * jq], R.acc[dt][4 * jq + 1], R.acc[dt][4 * jq + 2],
                        R.acc[dt][4 * jq + 3]);
    if (g == 0) s_ml[wave * 32 + lr] = make_float2(R.m, R.l);
  }
  __syncthreads();
  for (int x = tid; x < rq.rows * (D / 4); x += 256) {
    const int r = x / (D / 4), c = x % (D / 4);
    float m = kNegInf, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = __builtin_fmaxf(m, s_ml[w * 32 + r].x);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 ml = s_ml[w * 32 + r];
      const float a = fast_exp2(ml.x - safe_max(m));
      const float4 v = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(s_kv + w * (2 * TILE)) + r * D + ((c ^ (r % (D / 4))) << 2));
      l += ml.y * a;
      sum.x += v.x * a;
      sum.y += v.y * a;
      sum.z += v.z * a;
      sum.w += v.w * a;
    }
    const float inv = one_over(l);
    *reinterpret_cast<uint2*>(out_row<T, D>(C, rq, r, kvh) + 4 * c) =
        make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
  }
}

// Zeros for the rows of no request, by the workgroups that have no item.
template <int D>
__device__ __forceinline__ void clear_rows(const ChunkParams& C, long long at, long long of) {
  const int head = min(max(C.starts[0], 0), C.tokens);
  const int tail = min(max(C.starts[C.batch], 0), C.tokens);
  const long long row = (long long)C.hq * (D / 8), gap = (long long)(tail - head) * row;
  const long long total = (long long)C.tokens * row - gap;
  u32x4* const out = reinterpret_cast<u32x4*>(C.out);
  for (long long x = at * 256 + threadIdx.x; x < total; x += of * 256)
    out[x < head * row ? x : x + gap] = u32x4{0, 0, 0, 0};
}

// Workgroups per CU: three at D = 64 (see wide_body), but two for the biased and capped
// forms of an 8-bit cache, which spill with the registers of three: 64 single tokens
// over 2048, bias 39 us and cap 41 (three: 42, 46), 24 mixed requests with a cap 95
// (103), against 4 x 1024 new tokens of 4096 199 and 247 (188, 234).  At D = 128 the
// 8-bit forms have 256 registers and keep more in memory: the capped one 30, four of
// them loaded and one stored in every tile of the narrow body, the biased one three,
// the plain one two.  Of the 16-bit forms the capped one at D = 64 keeps one.
template <typename T, int D, Form FORM, bool FP8>
__global__ __launch_bounds__(256, D == 64 && !(FP8 && FORM != Form::kPlain) ? 3 : 2) void chunk_tile_kernel(
    Taken<FP8>) {
  __shared__ __attribute__((aligned(256))) uint16_t s_kv[2 * 2 * kStep * D];
  __shared__ float2 s_ml[4 * 32];
  __shared__ Seen s_seen[4];
  __shared__ int s_bad[4];
  const int lane = threadIdx.x & 63;
  const Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  const TileParams& P = reread(args);
  pin_plan(P);
  const Asked head = asked_of(P.c, lane, P.part_acc != nullptr);
  Cutting cut{};
  if (P.part_acc) cut = cut_batch<FP8>(P, head, lane);
  const bool counts = blockIdx.x == 0 && P.part_acc;
  // The narrow requests first: theirs is memory's time, the others' the
  // matrix units', so they run beside each other.
  const bool flat = (int)blockIdx.x < cut.groups;
  // KV heads in the low bits: with eight of them, each XCD serves one.
  const int in = blockIdx.x - cut.groups, at = divide(in, P.c.hkv, P.c.hkv_mul);
  const int kvh = in - at * P.c.hkv;
  Item it{};
  if (!flat || counts) {
    const int launched = counts ? (int)(gridDim.x - cut.groups + P.c.hkv - 1) / P.c.hkv : 0;
    it = plan_item(P, head, cut.share, flat ? -1ll : (long long)at, lane, counts, launched);
  }
  if (counts && threadIdx.x == 0) P.records[0] = make_int4(it.records, it.narrow_records, 0, 0);
  if (flat) {
    const TileParams& A = reread(args);
    pin_rows<FP8>(A);
    auto ask = [&](int b0) { return asked_of(A.c, b0 + lane, true); };
    flat_body<T, D, FORM, FP8, false>(A, head, A.c.batch, ask, cut, s_kv);
    return;
  }
  if (!it.found) {
    const long long items = it.items * P.c.hkv + cut.groups;
    clear_rows<D>(P.c, blockIdx.x - items, gridDim.x - items);
    return;
  }
  if (it.parts > 1 && it.part == 0 && kvh == 0 && threadIdx.x == 0)
    put_record(P, it.record, it.r.start, it.tile * kManyRows,
               min(it.r.rows - it.tile * kManyRows, kManyRows), it.parts,
               P.narrow_rows + it.slot * P.part_rows, P.part_rows);
  const TileParams& A = reread(args);
  pin_rows<FP8>(A);
  if (it.r.rows <= kFewRows)
    narrow_body<T, D, FORM, FP8>(A.c, it.r, kvh, s_kv, s_ml);
  else
    wide_body<T, D, FORM, FP8, false>(A, args, it, kvh, s_kv, s_seen, s_bad);
}

// One part's state joined to another's.
__device__ __forceinline__ void join(float& m, float& l, float4& acc, float m2, float l2, float4 v) {
  const float top = __builtin_fmaxf(m, m2), base = safe_max(top);
  const float a = fast_exp2(m - base), b = fast_exp2(m2 - base);
  m = top;
  l = l * a + l2 * b;
  acc.x = acc.x * a + v.x * b;
  acc.y = acc.y * a + v.y * b;
  acc.z = acc.z * a + v.z * b;
  acc.w = acc.w * a + v.w * b;
}

constexpr int kFewParts = 16;  // parts that one wave joins by itself

// Joins the partials, latency-bound (4 to 5 us): `apart` workgroups share the rows of a record and KV
// head.  Few parts: a wave per row, each group of D / 4 lanes taking the parts
// in turn; many: the whole workgroup per row.
template <typename T, int D>
__global__ __launch_bounds__(256) void chunk_join_kernel(TileParams P, int apart) {
  constexpr int LPR = D / 4, G = 256 / LPR, GW = 64 / LPR;  // lanes per row, groups, groups per wave
  __shared__ float4 s_acc[G][LPR];
  __shared__ float2 s_ml[G];
  const int tid = threadIdx.x, grp = tid / LPR, c = tid % LPR;
  const int4 counts = P.records[0];
  const int total = (counts.x + counts.y) * P.c.hkv * apart;
  for (int x = blockIdx.x; x < total; x += gridDim.x) {
    const int in = x / apart, sub = x - in * apart, i = in / P.c.hkv, kvh = in - i * P.c.hkv;
    const int at = i < counts.x ? i : P.most_parts / 2 + i - counts.x;
    const int4 rec = P.records[1 + 2 * at], part = P.records[2 + 2 * at];
    const int parts = rec.w;
    if (parts < 2) continue;
    const Request rq{0, rec.x, 0, 0, 0, 0};
    auto gather = [&](int r, int from, int step, float& m, float& l, float4& acc) {
#pragma unroll 4
      for (int p = from; p < parts; p += step) {
        const size_t row = partial_row(P, part.x + p * part.y + r, kvh);
        const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + 2 * row);
        join(m, l, acc, ml.x, ml.y, *reinterpret_cast<const float4*>(P.part_acc + row * D + 4 * c));
      }
    };
    if (parts <= kFewParts) {
      for (int r = 4 * sub + (tid >> 6); r < rec.z; r += 4 * apart) {
        float m = kNegInf, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        gather(r, grp % GW, GW, m, l, acc);
#pragma unroll
        for (int s = LPR; s < 64; s <<= 1)
          join(m, l, acc, shfl_xor_f(m, s), shfl_xor_f(l, s),
               make_float4(shfl_xor_f(acc.x, s), shfl_xor_f(acc.y, s), shfl_xor_f(acc.z, s),
                           shfl_xor_f(acc.w, s)));
        const float inv = one_over(l);
        if (grp % GW == 0)
          *reinterpret_cast<uint2*>(out_row<T, D>(P.c, rq, rec.y + r, kvh) + 4 * c) =
              make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
      }
      continue;
    }
    for (int r = sub; r < rec.z; r += apart) {
      float m = kNegInf, l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      gather(r, grp, G, m, l, acc);
      s_acc[grp][c] = acc;
      if (c == 0) s_ml[grp] = make_float2(m, l);
      __syncthreads();
      if (tid < D) {
        float top = kNegInf, sum = 0.f, out = 0.f;
#pragma unroll
        for (int w = 0; w < G; ++w) top = __builtin_fmaxf(top, s_ml[w].x);
#pragma unroll
        for (int w = 0; w < G; ++w) {
          const float a = fast_exp2(s_ml[w].x - safe_max(top));
          sum += s_ml[w].y * a;
          out += reinterpret_cast<const float*>(s_acc[w])[tid] * a;
        }
        out_row<T, D>(P.c, rq, rec.y + r, kvh)[tid] = round_to<T>(out * one_over(sum));
      }
      __syncthreads();
    }
  }
}

// How a call with a workspace cuts its work; bytes 0: it does not.
struct Cut {
  int target, waves, most_parts, part_rows, narrow_rows;
  size_t acc_bytes, ml_bytes, bytes;
};

inline Cut cut_of(const bc_shape& s, int tokens, bool fp8) {
  Cut c{};
  const long long steps = ((long long)s.max_pages * BC_PAGE_SIZE + kStep - 1) / kStep;
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  // Short tables are not cut: joining costs a launch (one token over 512: 8.2
  // us, cut 12.5; 64 over 16-512 18.9, 25.8), unless tiles of rows are few (128
  // new tokens of 1024: 22.1 cut, 27.4).
  const bool few = rows <= (long long)kFewRows * s.batch;
  if (steps <= (few ? 16 : 8) || rows < 1 || rows > 1 << 30 ||
      (long long)s.batch * (s.max_pages + 1ll) > 1 << 28 ||
      (long long)s.batch * s.query_heads > 1 << 26)
    return c;
  c.target = 2 * bch::device_cus();
  // One request's rows that fill the card as whole tiles need no join (5 us).
  if (s.batch == 1 && rows / kManyRows * s.kv_heads >= c.target) return Cut{};
  // Four ranges per CU, eight at dim 64, where a tile is half the bytes (64
  // single tokens over 128-4096: 52.5 us, 54.4 with four; at dim 128 96 us with
  // four, 99 with eight).
  const int per = s.dim == 64 || fp8 ? 4 : 2;
  c.waves = per * c.target / s.kv_heads > 1 ? per * c.target / s.kv_heads : 1;
  c.narrow_rows = 32 * c.waves + (int)(rows < 32ll * s.batch ? rows : 32ll * s.batch);
  if (rows > kFewRows) {
    c.most_parts = 2 * c.target / s.kv_heads;
    c.part_rows = rows < kManyRows ? (int)rows : kManyRows;
  }
  const long long all = c.narrow_rows + (long long)c.most_parts * c.part_rows;
  if (all > 0x7fffffff) return Cut{};
  const size_t slots = (size_t)all * s.kv_heads;
  c.acc_bytes = slots * s.dim * sizeof(float);
  c.ml_bytes = (slots * 2 * sizeof(float) + 15) / 16 * 16;
  c.bytes = c.acc_bytes + c.ml_bytes + (1 + 2 * ((size_t)c.most_parts / 2 + s.batch)) * sizeof(int4);
  return c;
}

template <typename T, int D, bool FP8>
hipError_t launch_tiles(MoreParams M, const Cut& cut, void* ws, unsigned grid, hipStream_t st) {
  TileParams& P = M.t;
  const ChunkParams& C = P.c;
  P.target = cut.target;
  if (ws) {
    char* const at = static_cast<char*>(ws);
    P.part_acc = reinterpret_cast<float*>(at);
    P.part_ml = reinterpret_cast<float*>(at + cut.acc_bytes);
    P.records = reinterpret_cast<int4*>(at + cut.acc_bytes + cut.ml_bytes);
    P.waves = cut.waves;
    P.most_parts = cut.most_parts;
    P.part_rows = cut.part_rows;
    P.narrow_rows = cut.narrow_rows;
  }
  if (C.cap > 0.f)
    chunk_tile_kernel<T, D, Form::kCap, FP8><<<dim3(grid), 256, 0, st>>>(taken<FP8>(M));
  else if (C.slopes)
    chunk_tile_kernel<T, D, Form::kBias, FP8><<<dim3(grid), 256, 0, st>>>(taken<FP8>(M));
  else
    chunk_tile_kernel<T, D, Form::kPlain, FP8><<<dim3(grid), 256, 0, st>>>(taken<FP8>(M));
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || !ws) return err;
  // Enough workgroups for the rows of a record and KV head, on average, but not
  // more than a round of them: 1024 in place of 2048 save 2 us.
  const long long pairs = (long long)C.batch * C.hkv, rows = (long long)C.tokens * C.group / C.batch;
  long long apart = 2ll * cut.target / pairs;
  apart = apart < rows ? apart : rows;
  apart = apart < 2 ? 2 : apart > 32 ? 32 : apart;
  const long long most = ((long long)cut.most_parts / 2 + C.batch) * C.hkv * apart;
  const long long grid_join = most < 2 * cut.target ? most : 2 * cut.target;
  chunk_join_kernel<T, D><<<dim3((unsigned)grid_join), 256, 0, st>>>(P, (int)apart);
  return hipGetLastError();
}

template <bool FP8>
hipError_t launch_tiles(const MoreParams& M, int dim, int dtype, const Cut& cut, void* ws, long long grid,
                        hipStream_t st) {
  if (dtype == BC_FLOAT16)
    return dim == 64 ? launch_tiles<_Float16, 64, FP8>(M, cut, ws, (unsigned)grid, st)
                     : launch_tiles<_Float16, 128, FP8>(M, cut, ws, (unsigned)grid, st);
  return dim == 64 ? launch_tiles<__bf16, 64, FP8>(M, cut, ws, (unsigned)grid, st)
                   : launch_tiles<__bf16, 128, FP8>(M, cut, ws, (unsigned)grid, st);
}

// Workgroups of the tile kernel with a workspace, at most, of a batch whose entries
// of more than 32 rows have `rows` rows in all.  Cut by shares, n tiles have less
// than target / Hkv + n parts.  A workgroup without work still walks the batch to
// see that, some 2 us, so none is launched beyond these.
inline long long split_grid(const bc_shape& s, const Cut& cut, long long rows, long long entries) {
  const long long wide = rows / (kFewRows + 1) < entries ? rows / (kFewRows + 1) : entries;
  const long long items = wide > 0 ? rows / kManyRows + wide + cut.target / s.kv_heads + 1 : 0;
  return items * s.kv_heads + ((long long)cut.waves * s.kv_heads + 3) / 4 + 1;
}

// Workgroups of the tile kernel, at most.
inline long long tile_grid(const bc_shape& s, int tokens, const Cut& cut, bool use) {
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  const long long tiles = (tokens < s.batch ? tokens : s.batch) + rows / kManyRows +
                          (use ? cut.most_parts : 0);
  return tiles * s.kv_heads + (use ? ((long long)cut.waves * s.kv_heads + 3) / 4 : 0) + 1;
}

// ---------------------------------------------------------------------------
// Arguments

inline bool chunk_shape_ok(const bc_shape& s, int tokens) {
  return s.batch >= 1 && s.query_heads >= 1 && s.kv_heads >= 1 &&
         s.query_heads % s.kv_heads == 0 && s.query_heads <= BC_MAX_CHUNK_HEADS &&
         (s.dim == 64 || s.dim == 128) && s.max_pages >= 1 && s.max_pages <= BC_MAX_TABLE_PAGES && s.physical_pages >= 1 &&
         tokens >= 0;
}

// The bits that any stride has, or a negative number where one is negative.
inline long long stride_bits(const bc_chunk_inputs& in) {
  const long long all[] = {in.q_strides.token, in.q_strides.head, in.k_strides.page,
                           in.k_strides.slot,  in.k_strides.head, in.v_strides.page,
                           in.v_strides.slot,  in.v_strides.head};
  long long bits = 0;
  for (long long x : all) bits |= x;
  return bits;
}

inline bool chunk_inputs_ok(const bc_chunk_inputs& in) {
  return in.window >= 0 && in.scale >= BC_LEAST_SCALE && in.scale <= BC_MOST_SCALE &&
         (in.cap == 0.f || (in.cap >= BC_LEAST_SCALE && in.cap <= BC_MOST_SCALE)) &&
         (in.dtype == BC_FLOAT16 || in.dtype == BC_BFLOAT16) && in.k && in.v && in.pages &&
         in.lengths && in.starts && stride_bits(in) >= 0;
}

inline ChunkParams chunk_params(const bc_shape& s, const bc_chunk_inputs& in) {
  const int group = s.query_heads / s.kv_heads;
  const bool exact = (long long)in.tokens * group * group < 1ll << 32;
  const unsigned group_mul = group > 1 && exact ? (unsigned)(((1ull << 32) + group - 1) / group) : 0;
  const bool few_heads = s.kv_heads > 1 && s.kv_heads <= 64;  // grids below 2^24, see `tiled`
  const unsigned hkv_mul = few_heads ? (unsigned)(((1ull << 32) + s.kv_heads - 1) / s.kv_heads) : 0;
  return ChunkParams{in.q,
                     in.k,
                     in.v,
                     in.pages,
                     in.lengths,
                     in.starts,
                     in.slopes,
                     in.prefix,
                     in.first,
                     in.output,
                     in.q_strides.token,
                     in.q_strides.head,
                     in.k_strides.page,
                     in.k_strides.slot,
                     in.k_strides.head,
                     in.v_strides.page,
                     in.v_strides.slot,
                     in.v_strides.head,
                     in.tokens,
                     s.batch,
                     s.query_heads,
                     s.kv_heads,
                     group,
                     s.max_pages,
                     s.physical_pages,
                     in.causal != 0,
                     in.window,
                     group_mul,
                     hkv_mul,
                     in.scale,
                     in.cap};
}

}  // namespace
