// Chunks of new tokens over the paged cache, for gfx950: the block tables and
// slot maps of a step from its requests' lengths (bc_build_tables), the new
// tokens' K and V rows into the pool (bc_append_kv), and the attention of the
// new tokens over their requests' pages (bc_chunk_attention).
//
// No reference counterpart: the reference attends one token per request
// (src/paged_gqa.cu) or a tree of draft tokens outside the cache
// (src/tree_attention.cu), and fills pages on the host
// (python/branchcraft_torch/transaction.py:64-81).
#include <type_traits>

#include "bc_device.h"
#include "bc_host.h"

using namespace bcd;

namespace {

constexpr int kThreads = 256;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---------------------------------------------------------------------------
// Block tables and slot maps

struct TableParams {
  const int32_t* ids;      // page ids of all requests, one after another
  const int32_t* lengths;  // [batch] tokens of a request, its new ones included
  const int32_t* counts;   // [batch] new tokens
  int32_t* pages;          // [batch, max_pages]
  int32_t* starts;         // [batch + 1]
  int32_t* slots;          // [tokens]
  int32_t* positions;      // [tokens]
  int held, batch, max_pages, tokens;
};

constexpr int kTableSpan = 2048;  // table entries, and rows of the slot map, per workgroup

__device__ __forceinline__ long long wave_sum_ll(long long x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s, 64);
  return x;
}

// grid = (batch + 1, slices).  Workgroup (b, s) sums the pages and new tokens
// of the requests before b, so that no workgroup waits for another, and
// writes slice s of b's table row and of its rows of the slot map; workgroup
// row `batch` writes what lies behind the last request.
__global__ __launch_bounds__(kThreads) void build_tables_kernel(TableParams P) {
  const int b = blockIdx.x, tid = threadIdx.x;
  __shared__ long long s_sum[2][kThreads / 64];
  long long before = 0, at = 0;
  for (int i = tid; i < b; i += kThreads) {
    before += ((long long)max(P.lengths[i], 0) + BC_PAGE_SIZE - 1) / BC_PAGE_SIZE;
    at += max(P.counts[i], 0);
  }
  before = wave_sum_ll(before);
  at = wave_sum_ll(at);
  if ((tid & 63) == 0) {
    s_sum[0][tid >> 6] = before;
    s_sum[1][tid >> 6] = at;
  }
  __syncthreads();
  before = at = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before += s_sum[0][w];
    at += s_sum[1][w];
  }
  const int start = (int)min(at, (long long)P.tokens);
  if (blockIdx.y == 0 && tid == 0) P.starts[b] = start;
  const int begin = blockIdx.y * kTableSpan;
  if (b == P.batch) {  // rows behind the last request
    for (int i = begin + tid; i < min(begin + kTableSpan, P.tokens - start); i += kThreads) {
      P.slots[start + i] = -1;
      P.positions[start + i] = -1;
    }
    return;
  }
  const int len = max(P.lengths[b], 0), n = min(max(P.counts[b], 0), P.tokens - start);
  const int old = len - max(P.counts[b], 0);  // may be negative: such rows have no token
  // Pages that the list holds for this request, within its row of the table.
  const long long rest = P.held - before;
  const int used = (int)max(0ll, min(min((len + BC_PAGE_SIZE - 1ll) / BC_PAGE_SIZE,
                                         (long long)P.max_pages), rest));
  int32_t* const row = P.pages + (size_t)b * P.max_pages;
  for (int i = begin + tid; i < min(begin + kTableSpan, P.max_pages); i += kThreads)
    row[i] = i < used ? P.ids[before + i] : -1;
  for (int i = begin + tid; i < min(begin + kTableSpan, n); i += kThreads) {
    const int pos = old + i, c = pos >> 4;
    const int id = pos >= 0 && c < used ? P.ids[before + c] : -1;
    P.positions[start + i] = pos >= 0 ? pos : -1;
    P.slots[start + i] = id >= 0 && id < (1 << 27) ? id * BC_PAGE_SIZE + (pos & 15) : -1;
  }
}

// ---------------------------------------------------------------------------
// New tokens' rows into the pool

struct AppendParams {
  const void* k;
  const void* v;
  void* cache_k;
  void* cache_v;
  const int32_t* slots;
  // In elements of the copy: rows' token and head strides, pools' page, slot
  // and head strides, of K and of V.
  long long ts[2], hs[2], cp[2], cs[2], ch[2];
  int tokens, phys_pages, row_vec, head_vec;
};

// Workgroup i copies rows_per_block rows, K then V, in elements of type E.
template <typename E>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendParams P, int rows_per_block) {
  const int t0 = blockIdx.x * rows_per_block;
  const int n = min(rows_per_block, P.tokens - t0) * P.row_vec;
  for (int x = threadIdx.x; x < n; x += kThreads) {
    const int i = x / P.row_vec, c = x - i * P.row_vec;
    const int h = c / P.head_vec, e = c - h * P.head_vec;
    const int slot = P.slots[t0 + i];
    if (slot < 0 || (slot >> 4) >= P.phys_pages) continue;
    const long long t = t0 + i, page = slot >> 4, in = slot & 15;
    static_cast<E*>(P.cache_k)[page * P.cp[0] + in * P.cs[0] + h * P.ch[0] + e] =
        static_cast<const E*>(P.k)[t * P.ts[0] + h * P.hs[0] + e];
    static_cast<E*>(P.cache_v)[page * P.cp[1] + in * P.cs[1] + h * P.ch[1] + e] =
        static_cast<const E*>(P.v)[t * P.ts[1] + h * P.hs[1] + e];
  }
}

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
  float scale, cap;
};

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

// tanh in terms of one exponential: 1 - 2 / (e^2x + 1), whose absolute error
// is a few 2^-24; exact at both infinities.
__device__ __forceinline__ float fast_tanh(float x) {
  return 1.f - 2.f * __builtin_amdgcn_rcpf(fast_exp2(x * (2.f * kLog2e)) + 1.f);
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

__device__ __forceinline__ int clamp_len(const ChunkParams& P, int b) {
  return max(0, (int)min((long long)P.lengths[b], (long long)P.max_pages * BC_PAGE_SIZE));
}

// The tokens lo .. hi that row t at position pos of request b sees.
__device__ __forceinline__ int2 row_range(const ChunkParams& P, int b, int t, int pos, int len) {
  int lo = 0, hi = len - 1;
  if (P.causal) hi = min(hi, P.prefix ? max(pos, max(P.prefix[b], 0) - 1) : pos);
  if (P.window > 0) lo = max(lo, pos - P.window + 1);
  if (P.first) lo = max(lo, P.first[t]);
  return pos < 0 ? make_int2(1, 0) : make_int2(lo, hi);
}

// The plain form of the operator, for tensors whose addresses or strides rule
// out 16-byte loads.  One wave per (row, query head): lane j scores token j
// of 64, the online softmax's maximum and sum stay in the wave, and each lane
// keeps D / 64 dimensions of the output.  Tokens that the row does not see
// are never multiplied, whatever their K and V hold.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void chunk_rows_kernel(ChunkParams P) {
  constexpr int R = D / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x, h = blockIdx.y * (kThreads / 64) + wave;
  if (h >= P.hq) return;
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
    for (int j0 = seen.x & ~63; j0 <= seen.y; j0 += 64) {
      const int j = j0 + lane;
      const int id = j >= seen.x && j <= seen.y ? row[j >> 4] : -1;
      const bool ok = (unsigned)id < (unsigned)P.phys_pages;
      float s = kNegInf;
      if (ok) {
        const uint16_t* const k = P.k + id * P.kp + (j & 15) * P.ks + kvh * P.kh;
        float dot = 0.f;
        for (int d = 0; d < D; ++d) dot += load_elem<T>(q + d) * load_elem<T>(k + d);
        s = dot * P.scale;
        if (P.cap > 0.f) s = P.cap * fast_tanh(s / P.cap);
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
        const int from = __builtin_ctzll(left);
        const float w = __shfl(p, from, 64);
        const uint16_t* const v =
            P.v + __shfl(id, from, 64) * P.vp + ((j0 + from) & 15) * P.vs + kvh * P.vh;
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] += w * load_elem<T>(v + 64 * r + lane);
      }
    }
  }
  uint16_t* const out = P.out + ((size_t)t * P.hq + h) * D;
#pragma unroll
  for (int r = 0; r < R; ++r)
    out[64 * r + lane] = round_to<T>(l > 0.f || l != l ? acc[r] / l : 0.f);
}

template <typename T, int D>
void launch_rows(const ChunkParams& P, hipStream_t st) {
  const dim3 grid(P.tokens, (P.hq + kThreads / 64 - 1) / (kThreads / 64));
  chunk_rows_kernel<T, D><<<grid, kThreads, 0, st>>>(P);
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
constexpr int kFewRows = 32;    // rows of a request that take the narrow form
constexpr int kManyRows = 128;  // rows per workgroup of the wide form
constexpr int kLeastSteps = 4;  // fewest steps per part of a split tile

struct TileParams {
  ChunkParams c;
  float* part_acc;  // [parts][Hkv][part_rows][D]; null: nothing is split
  float* part_ml;   // [parts][Hkv][part_rows][2]: maximum and sum
  int* records;     // count, then four ints per split tile
  int part_rows;    // rows of a partial
  int target;       // workgroups that a batch's work is cut for
  int most_parts;   // partials per KV head that the workspace holds
};

// What a workgroup does: part `part` of `parts` of row tile `tile` of request
// b, whose rows (new tokens times group) are `rows`, at tokens start .. of the
// step, the first of them at place pos0 of the request.
struct Item {
  int b, start, n, len, pos0, rows, tile, part, parts, slot;
  int record;          // of a split tile
  long long items;     // where no item has the index: how many there are
  int records;         // likewise
  bool found;
};

__device__ __forceinline__ int wave_min_i(int x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x = min(x, __shfl_xor(x, s, 64));
  return x;
}

__device__ __forceinline__ int wave_max_i(int x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x = max(x, __shfl_xor(x, s, 64));
  return x;
}

__device__ __forceinline__ int lanes_sum(int x) {
  return __builtin_amdgcn_readfirstlane(wave_sum_i(x));
}

// One request's share of the plan, a request per lane.
struct Asked {
  int start, n, len, full, rows, tiles, steps;
};

__device__ __forceinline__ Asked asked_of(const ChunkParams& P, int b) {
  Asked a{};
  if (b < P.batch) {
    a.start = min(max(P.starts[b], 0), P.tokens);
    a.n = max(min(max(P.starts[b + 1], 0), P.tokens) - a.start, 0);
    a.full = max(P.lengths[b], 0);
    a.len = (int)min((long long)a.full, (long long)P.max_pages * BC_PAGE_SIZE);
    a.rows = a.n * P.group;
    a.tiles = a.rows <= kFewRows ? (a.rows > 0) : (a.rows + kManyRows - 1) / kManyRows;
    int span = a.len;
    if (P.causal && P.window > 0) span = min(span, min(P.window, 1 << 29) + kManyRows + kStep);
    a.steps = max(1, (span + kStep - 1) / kStep);
  }
  return a;
}

// Item `idx` of the batch, found by every wave for itself from starts and
// lengths.  A tile of rows whose steps are more than the batch's work over
// `target` workgroups is cut into equal parts; as no part is shorter than
// that share, half of it at least, the split tiles have at most 2 * target /
// Hkv parts per KV head.  A request's last tiles, which see most, come first.
// `all`: go to the end and count.
__device__ __forceinline__ Item plan_item(const TileParams& P, long long idx, int lane, bool all) {
  const ChunkParams& C = P.c;
  Asked a = asked_of(C, lane);
  int share = 0x7fffffff;
  if (P.part_acc) {
    long long work = (long long)a.tiles * a.steps;
    for (int b = 64 + lane; b - lane < C.batch; b += 64) {
      const Asked x = asked_of(C, b);
      work += (long long)x.tiles * x.steps;
    }
    work = wave_sum_ll(work);
    const double cut = (double)work * C.hkv / P.target;
    share = max(kLeastSteps, cut < 1e9 ? (int)cut + 1 : 1000000000);
  }
  Item it{};
  long long before = 0;
  int slots = 0, records = 0;
  for (int b0 = 0; b0 < C.batch; b0 += 64) {
    if (b0 > 0) a = asked_of(C, b0 + lane);
    const int parts = a.steps > share ? (a.steps + share - 1) / share : 1;
    const int mine = a.tiles * parts;
    int upto = mine;  // inclusive sum over the lanes
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int x = __shfl_up(upto, s, 64);
      upto += lane >= s ? x : 0;
    }
    const int total = __builtin_amdgcn_readlane(upto, 63);
    const int cut_parts = parts > 1 ? mine : 0, cut_tiles = parts > 1 ? a.tiles : 0;
    if (!it.found && idx - before < total) {
      const int local = (int)(idx - before);
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > local));
      it.found = true;
      it.b = b0 + at;
      it.start = __builtin_amdgcn_readlane(a.start, at);
      it.n = __builtin_amdgcn_readlane(a.n, at);
      it.len = __builtin_amdgcn_readlane(a.len, at);
      it.pos0 = __builtin_amdgcn_readlane(a.full, at) - it.n;
      it.rows = __builtin_amdgcn_readlane(a.rows, at);
      it.parts = __builtin_amdgcn_readlane(parts, at);
      const int in = local - __builtin_amdgcn_readlane(upto - mine, at);
      const int nth = in / it.parts;
      it.part = in - nth * it.parts;
      it.tile = __builtin_amdgcn_readlane(a.tiles, at) - 1 - nth;
      if (it.parts > 1) {
        it.slot = slots + lanes_sum(lane < at ? cut_parts : 0) + in;
        it.record = records + lanes_sum(lane < at ? cut_tiles : 0) + nth;
        if (it.slot - it.part + it.parts > P.most_parts) it.parts = 1;  // cannot be: see above
      }
      if (!all) return it;
    }
    before += total;
    if (P.part_acc) {
      slots += lanes_sum(cut_parts);
      records += lanes_sum(cut_tiles);
    }
  }
  it.items = before;
  it.records = records;
  return it;
}

// A wave's 32 rows: lane lr of either half has row lr.
template <int D>
struct Rows {
  f32x16 acc[D / 32];  // O^T: dimension 32 dt + 8 (j / 4) + 4 g + j % 4
  float m, l;
  float slope;         // times log2 e
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

// Scores of NT staged tiles, from token t0 on, to the softmax's exponents:
// raw products in the plain form (their scale is applied with the maximum),
// log2 units otherwise.  `edge`: mask to the row's lo .. hi and to `valid`.
template <typename T, int D, bool PLAIN, int NT>
__device__ __forceinline__ void finish_scores(const ChunkParams& C, f32x16 (&sc)[NT],
                                              const Rows<D>& r, int t0, int g, bool edge,
                                              unsigned long long valid) {
  if (!PLAIN) {
    const float from = (float)(r.pos - t0 - 4 * g);
    if (C.cap > 0.f) {
      // cap * tanh(x) in log2 units, x = scale * s / cap.
      const float in = C.scale / C.cap * (2.f * kLog2e), top = C.cap * kLog2e;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sc[i][j] = __builtin_fmaf(
              -2.f * top, __builtin_amdgcn_rcpf(fast_exp2(sc[i][j] * in) + 1.f), top);
    } else {
      const float by = C.scale * kLog2e;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[i][j] *= by;
    }
    if (C.slopes) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sc[i][j] = __builtin_fmaf(
              -r.slope, __builtin_fabsf(from - (float)(32 * i + 8 * (j >> 2) + (j & 3))),
              sc[i][j]);
    }
  }
  if (edge) {
    const int a = r.lo - t0 - 4 * g, b = r.hi - t0 - 4 * g;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t ok = (uint32_t)(valid >> (32 * i)) >> (4 * g);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int off = 8 * (j >> 2) + (j & 3);
        const bool in = 32 * i + off >= a && 32 * i + off <= b && ((ok >> off) & 1u);
        sc[i][j] = in ? sc[i][j] : kNegInf;
      }
    }
  }
}

// Online softmax and O^T += V^T P^T over NT staged tiles.  The maximum moves
// only when it would grow by more than kRescaleSlack.  Weights are rounded to
// T, to nearest, for the product (half a step of T each, as the output's own
// rounding); their sum is of the rounded weights, in 32 bits.
template <typename T, int D, bool PLAIN, int NT>
__device__ __forceinline__ void weigh(f32x16 (&sc)[NT], Rows<D>& r, const uint16_t* vt,
                                      const Offsets<D>& o, float scale_log2) {
  constexpr int DT = D / 32, NG = 2 * NT;
  typedef Num<T> N;
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) top = __builtin_fmaxf(top, sc[i][j]);
  if (PLAIN) top *= scale_log2;
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
      const float p0 = fast_exp2(PLAIN ? __builtin_fmaf(s0, scale_log2, -base) : s0 - base);
      const float p1 = fast_exp2(PLAIN ? __builtin_fmaf(s1, scale_log2, -base) : s1 - base);
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

// What tidy() took out of the tokens t0 .. t0 + count - 1, added to the rows
// that see it.  Rare, so token by token and from the cache.
template <typename T, int D>
__device__ __forceinline__ void add_untidy(const ChunkParams& C, const Item& it, int kvh, Rows<D>& R,
                                           int t0, int count, int g) {
  const int32_t* const table = C.pages + (size_t)it.b * C.max_pages;
#pragma unroll 1
  for (int j = t0; j < min(t0 + count, it.len); ++j) {
    const int p = table[j >> 4];
    if ((unsigned)p >= (unsigned)C.phys_pages) continue;
    const bool seen = j >= R.lo && j <= R.hi;
    const uint16_t* const v = C.v + p * C.vp + (j & 15) * C.vs + kvh * C.vh + 4 * g;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int jq = 0; jq < 4; ++jq) {
        const uint2 w = *reinterpret_cast<const uint2*>(v + 32 * dt + 8 * jq);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float f = to_float(__builtin_bit_cast(T, (uint16_t)((x < 2 ? w.x : w.y) >> (16 * (x & 1)))));
          R.acc[dt][4 * jq + x] += seen && !(__builtin_fabsf(f) < -kNegInf) ? f : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
}

// Page ids that lie in the pool, and the tokens they and the length allow.
template <int PAGES>
__device__ __forceinline__ unsigned long long valid_tokens(const ChunkParams& C, const int (&id)[PAGES],
                                                           int left) {
  unsigned long long ok = left >= 64 ? ~0ull : left > 0 ? (1ull << left) - 1 : 0ull;
#pragma unroll
  for (int q = 0; q < PAGES; ++q)
    if ((unsigned)id[q] >= (unsigned)C.phys_pages) ok &= ~(0xffffull << (16 * q));
  return ok;
}

// This lane's row of the wave's 32: its place, what it sees, and its Q.
template <typename T, int D, bool PLAIN>
__device__ __forceinline__ void load_rows(const ChunkParams& C, const Item& it, int r, int kvh,
                                          int g, Rows<D>& R, u32x4 (&qB)[D / 16]) {
  const bool real = r < it.rows;
  const int i = real ? r / C.group : 0, h = kvh * C.group + (real ? r - i * C.group : 0);
  const int t = it.start + i;
  const uint16_t* const q = C.q + t * C.qt + h * C.qh + 8 * g;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qB[s] = *reinterpret_cast<const u32x4*>(q + 16 * s);
  R.pos = it.pos0 + i;
  const int2 seen = row_range(C, it.b, t, R.pos, it.len);
  R.lo = real ? seen.x : 1;
  R.hi = real ? seen.y : 0;
  R.slope = !PLAIN && C.slopes ? C.slopes[h] * kLog2e : 0.f;
  R.m = kNegInf;
  R.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) R.acc[dt][j] = 0.f;
}

// The tokens that a wave's real rows see: all of them (whole) or some (any).
struct Seen {
  int any_lo, any_hi, all_lo, all_hi;
};

template <int D>
__device__ __forceinline__ Seen wave_seen(const Rows<D>& R, bool real) {
  const bool some = real && R.lo <= R.hi;
  const int any_lo = wave_min_i(some ? R.lo : 0x7fffffff), any_hi = wave_max_i(some ? R.hi : -1);
  const int all_lo = wave_max_i(real ? (some ? R.lo : 0x7fffffff) : 0);
  const int all_hi = wave_min_i(real ? R.hi : 0x7fffffff);
  return {__builtin_amdgcn_readfirstlane(any_lo), __builtin_amdgcn_readfirstlane(any_hi),
          __builtin_amdgcn_readfirstlane(all_lo), __builtin_amdgcn_readfirstlane(all_hi)};
}

__device__ __forceinline__ float one_over(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }

// The wide form: 128 rows per workgroup, 32 per wave, each step's K and V
// shared through LDS.
template <typename T, int D, bool PLAIN>
__device__ __forceinline__ void wide_body(const TileParams& P, const Item& it, int kvh,
                                          uint16_t* s_kv, Seen* s_seen) {
  const ChunkParams& C = P.c;
  constexpr int KS = D / 16, CPR = D / 8;
  constexpr int NX = kStep * CPR / 256;  // chunks per thread and step, of K and of V each
  constexpr int HALF = kStep * D;        // halves of a step's K, then as many of V
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, lr = lane & 31;
  const int row0 = it.tile * kManyRows + wave * 32;
  Rows<D> R;
  u32x4 qB[KS];
  load_rows<T, D, PLAIN>(C, it, row0 + lr, kvh, g, R, qB);
  const Seen mine = wave_seen(R, row0 + lr < it.rows);
  if (lane == 0) s_seen[wave] = mine;
  __syncthreads();
  Seen wg = s_seen[0];
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
  const int first = wg.any_lo / kStep;
  const int steps = wg.any_hi >= wg.any_lo ? wg.any_hi / kStep - first + 1 : 0;
  const int t0 = first + (int)((long long)steps * it.part / it.parts);
  const int tend = first + (int)((long long)steps * (it.part + 1) / it.parts);

  const int lrow = tid / CPR, lcol = 8 * (tid % CPR ^ swz<D>(lrow));
  const unsigned koff = (unsigned)(((lrow % BC_PAGE_SIZE) * C.ks + lcol) * 2);
  const unsigned voff = (unsigned)(((lrow % BC_PAGE_SIZE) * C.vs + lcol) * 2);
  const uint16_t* const kb = C.k + kvh * C.kh;
  const uint16_t* const vb = C.v + kvh * C.vh;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)s_kv + wave * 1024);
  // The pages of 16 steps, one per lane: their addresses, so that a step reads
  // them out instead of multiplying, and which lie in the pool (others are
  // loaded from page 0 and masked).
  const int32_t* const table = C.pages + (size_t)it.b * C.max_pages;
  auto load_ids = [&](int t) { return table[min(t * 4 + lane, C.max_pages - 1)]; };
  unsigned long long k_at = 0, v_at = 0, pool = 0;
  auto take_ids = [&](int ids) {
    const bool in = (unsigned)ids < (unsigned)C.phys_pages;
    pool = __builtin_amdgcn_ballot_w64(in);
    const long long id = in ? ids : 0;
    k_at = (unsigned long long)(kb + id * C.kp);
    v_at = (unsigned long long)(vb + id * C.vp);
  };
  auto lane_of = [&](unsigned long long x, int from) {
    return (const void*)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), from) << 32 |
                         (unsigned)__builtin_amdgcn_readlane((int)x, from));
  };
  auto issue_chunk = [&](int x, int at, int buf) {
    const int from = 4 * at + (CPR == 16 ? x : 2 * x + (wave >> 1));
    const unsigned dst = lds0 + buf * (4 * HALF) + x * 4096;
    load_to_lds(lane_of(k_at, from), koff, dst);
    load_to_lds(lane_of(v_at, from), voff, dst + 2 * HALF);
  };
  // The tokens of step t that are any: in pages of the pool, below the length.
  auto tokens_of = [&](int t, int pages) {
    const int left = it.len - t * kStep;
    unsigned long long ok = left >= 64 ? ~0ull : left > 0 ? (1ull << left) - 1 : 0ull;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (!((pages >> q) & 1)) ok &= ~(0xffffull << (16 * q));
    return ok;
  };
  // Steps whole_lo .. whole_hi - 1 are seen whole by every row, given their pages.
  const int whole_lo = wg.all_lo / kStep + (wg.all_lo % kStep != 0);
  const int whole_hi = min(wg.all_hi == 0x7fffffff ? 0 : wg.all_hi + 1, it.len) / kStep;
  // Each thread tidies the chunks that its own loads, already waited for,
  // have filled.
  auto inspect = [&](unsigned long long ok, uint16_t* v) {
    bool bad = false;
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      u32x4* const at = reinterpret_cast<u32x4*>(v + (tid + 256 * x) * 8);
      bad |= tidy<T>(at, (ok >> (lrow + 256 / CPR * x)) & 1u);
    }
    return __builtin_amdgcn_readfirstlane(__syncthreads_or(bad)) != 0;
  };

  const Offsets<D> o = read_offsets<D>(lane);
  const float scale_log2 = C.scale * kLog2e;
  bool is_whole = true, bad = false;
  int pages = 15;  // of the step at hand, a bit each: in the pool
  int ids_next = 0;
  if (t0 < tend) {
    take_ids(load_ids(t0));
    ids_next = load_ids(t0 + 16);
#pragma unroll
    for (int x = 0; x < NX; ++x) issue_chunk(x, 0, 0);
    pages = (int)pool & 15;
    is_whole = pages == 15 && t0 >= whole_lo && t0 < whole_hi;
    // The wait for Q belongs here, not inside the loop over steps.
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qB[s]));
    wait_loads();
    if (!is_whole)
      bad = inspect(tokens_of(t0, pages), s_kv + HALF);
    else
      __syncthreads();
  }
  // One step, its K and V in buffer `buf`; the next one's loads go out between
  // the score products.
  auto step = [&](auto which, int t) {
    constexpr int buf = decltype(which)::value;
    const uint16_t* const kt = s_kv + buf * (2 * HALF);
    const bool next = t + 1 < tend;
    const int at = (t + 1 - t0) % 16;
    if (at == 0 && next) {
      take_ids(ids_next);
      ids_next = load_ids(t + 17);
    }
    const int pages_n = (int)(pool >> (4 * at)) & 15;
    const bool whole_n = !next || (pages_n == 15 && t + 1 >= whole_lo && t + 1 < whole_hi);
    f32x16 sc[2];
    u32x4 kf[2][KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) kf[i][s] = lds16(kt + i * 32 * D + o.k[s]);
    const f32x16 zero = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[i] = Num<T>::mfma(kf[i][s], qB[s], s == 0 ? zero : sc[i]);
      if (s % 2 == 1 && s / 2 < NX) {
        if (next) issue_chunk(s / 2, at, buf ^ 1);
      }
    }
    const bool edge = !is_whole && (pages != 15 || it.len - t * kStep < kStep ||
                                    t * kStep < mine.all_lo || t * kStep + kStep - 1 > mine.all_hi);
    finish_scores<T, D, PLAIN, 2>(C, sc, R, t * kStep, g, edge, edge ? tokens_of(t, pages) : 0);
    weigh<T, D, PLAIN, 2>(sc, R, kt + HALF, o, scale_log2);
    if (bad) add_untidy<T, D>(C, it, kvh, R, t * kStep, kStep, g);
    wait_loads();
    bad = false;
    if (!whole_n)
      bad = inspect(tokens_of(t + 1, pages_n), s_kv + (buf ^ 1) * (2 * HALF) + HALF);
    else
      __syncthreads();
    is_whole = whole_n;
    pages = pages_n;
  };
  for (int t = t0; t < tend; t += 2) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + 1 < tend) step(std::integral_constant<int, 1>{}, t + 1);
  }

  R.l += shfl_xor_f(R.l, 32);
  const int r = row0 + lr;
  if (it.parts > 1) {
    const size_t at = ((size_t)it.slot * C.hkv + kvh) * P.part_rows + wave * 32 + lr;
    if (r < it.rows) {
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
    if (rr < it.rows) {
      const int n = rr / C.group, h = kvh * C.group + rr - n * C.group;
      *reinterpret_cast<u32x4*>(C.out + ((size_t)(it.start + n) * C.hq + h) * D + 8 * c) = w;
    }
  }
}

// The narrow form: the few rows of a request, at most 32, in every wave of
// the workgroup; each wave streams every fourth tile of 32 tokens through its
// own part of LDS, K of the next tile behind the scores, V behind the
// product, without a barrier, and the four states meet at the end.
template <typename T, int D, bool PLAIN>
__device__ __forceinline__ void narrow_body(const TileParams& P, const Item& it, int kvh,
                                            uint16_t* s_kv, float2* s_ml) {
  const ChunkParams& C = P.c;
  constexpr int KS = D / 16, CPR = D / 8;
  constexpr int RPL = 64 / CPR;   // token rows per load
  constexpr int NL = 32 / RPL;    // loads per tile, of K and of V each
  constexpr int NV = D == 128 ? 4 : 2;  // lane offsets: the swizzle repeats every 16 rows
  constexpr int TILE = 32 * D;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, lr = lane & 31;
  Rows<D> R;
  u32x4 qB[KS];
  load_rows<T, D, PLAIN>(C, it, lr, kvh, g, R, qB);
  const Seen mine = wave_seen(R, lr < it.rows);
  const int lo = mine.any_lo, hi = mine.any_hi;
  const int first = lo / kStep;
  const int steps = hi >= lo ? hi / kStep - first + 1 : 0;
  const int t0 = 2 * (first + (int)((long long)steps * it.part / it.parts)) + wave;
  const int tend = min(2 * (first + (int)((long long)steps * (it.part + 1) / it.parts)), hi / 32 + 1);

  unsigned koff[NV], voff[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int row = c * RPL + lane / CPR, col = 8 * (lane % CPR ^ swz<D>(row));
    koff[c] = (unsigned)((row * C.ks + col) * 2);
    voff[c] = (unsigned)((row * C.vs + col) * 2);
  }
  const uint16_t* const kb = C.k + kvh * C.kh;
  const uint16_t* const vb = C.v + kvh * C.vh;
  uint16_t* const kt = s_kv + wave * (2 * TILE);
  uint16_t* const vt = kt + TILE;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)kt);
  const int32_t* const table = C.pages + (size_t)it.b * C.max_pages;
  // Lane i: page i % 2 of this wave's tile i / 2 from tile t on.
  auto load_ids = [&](int t) {
    return table[min(2 * (t + 4 * (lane >> 1)) + (lane & 1), C.max_pages - 1)];
  };
  auto in_pool = [&](int p) { return (unsigned)p < (unsigned)C.phys_pages ? p : 0; };
  auto issue_k = [&](const int (&id)[2]) {
#pragma unroll
    for (int c = 0; c < NL; ++c)
      load_to_lds(kb + in_pool(id[c / NV]) * C.kp, koff[c % NV], lds0 + c * 1024);
  };
  auto issue_v = [&](const int (&id)[2]) {
#pragma unroll
    for (int c = 0; c < NL; ++c)
      load_to_lds(vb + in_pool(id[c / NV]) * C.vp, voff[c % NV], lds0 + 2 * TILE + c * 1024);
  };
  static_assert(NL / NV == 2 && NV * RPL == BC_PAGE_SIZE, "a tile is two pages");
  const Offsets<D> o = read_offsets<D>(lane);
  const float scale_log2 = C.scale * kLog2e;
  if (t0 < tend) {
    int ids = load_ids(t0), ids_next = load_ids(t0 + 128);
    int id[2] = {__builtin_amdgcn_readlane(ids, 0), __builtin_amdgcn_readlane(ids, 1)};
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qB[s]));
    issue_k(id);
    issue_v(id);
    int i = 0;
    for (int t = t0; t < tend; t += 4) {
      const bool next = t + 4 < tend;
      const unsigned long long ok = valid_tokens(C, id, it.len - t * 32) & 0xffffffffull;
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");  // K is there, V may be not
      f32x16 sc[1];
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[0][j] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) sc[0] = Num<T>::mfma(lds16(kt + o.k[s]), qB[s], sc[0]);
      int id_n[2] = {id[0], id[1]};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
      if (next) {
        i = (i + 1) % 32;
        if (i == 0) {
          ids = ids_next;
          ids_next = load_ids(t + 4 + 128);
        }
        id_n[0] = __builtin_amdgcn_readlane(ids, 2 * i);
        id_n[1] = __builtin_amdgcn_readlane(ids, 2 * i + 1);
        issue_k(id_n);
      }
      const bool edge = ok != 0xffffffffull || t * 32 < mine.all_lo || t * 32 + 31 > mine.all_hi;
      finish_scores<T, D, PLAIN, 1>(C, sc, R, t * 32, g, edge, ok);
      if (next)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");  // V is there
      else
        wait_loads();
      bool bad = false;
      if (edge) {
#pragma unroll
        for (int c = 0; c < NL; ++c) {
          u32x4* const at = reinterpret_cast<u32x4*>(vt + c * 512 + lane * 8);
          bad |= tidy<T>(at, (ok >> (c * RPL + lane / CPR)) & 1u);
        }
        bad = __builtin_amdgcn_ballot_w64(bad) != 0;
        wave_lds_sync();
      }
      weigh<T, D, PLAIN, 1>(sc, R, vt, o, scale_log2);
      if (bad) add_untidy<T, D>(C, it, kvh, R, t * 32, 32, g);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V has been read
      if (next) issue_v(id_n);
      id[0] = id_n[0];
      id[1] = id_n[1];
    }
  }

  // The four states through LDS: four-float chunk c of row r at c ^ (r % (D / 4)).
  R.l += shfl_xor_f(R.l, 32);
  float* const acc = reinterpret_cast<float*>(kt);
  wave_lds_sync();
  if (lr < it.rows) {
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
  for (int x = tid; x < it.rows * (D / 4); x += 256) {
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
    if (it.parts > 1) {
      const size_t at = ((size_t)it.slot * C.hkv + kvh) * P.part_rows + r;
      if (c == 0) *reinterpret_cast<float2*>(P.part_ml + 2 * at) = make_float2(m, l);
      *reinterpret_cast<float4*>(P.part_acc + at * D + 4 * c) = sum;
    } else {
      const float inv = one_over(l);
      const int n = r / C.group, h = kvh * C.group + r - n * C.group;
      *reinterpret_cast<uint2*>(C.out + ((size_t)(it.start + n) * C.hq + h) * D + 4 * c) =
          make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
    }
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

template <typename T, int D, bool PLAIN>
__global__ __launch_bounds__(256, 2) void chunk_tile_kernel(TileParams P) {
  __shared__ __attribute__((aligned(256))) uint16_t s_kv[2 * 2 * kStep * D];
  __shared__ float2 s_ml[4 * 32];
  __shared__ Seen s_seen[4];
  const int lane = threadIdx.x & 63;
  const long long idx = blockIdx.x / (unsigned)P.c.hkv;
  const int kvh = blockIdx.x - (unsigned)idx * P.c.hkv;
  const bool counts = blockIdx.x == 0 && P.part_acc;
  const Item it = plan_item(P, idx, lane, counts);
  if (counts && threadIdx.x == 0) P.records[0] = it.records;
  if (!it.found) {
    const long long items = it.items * P.c.hkv;
    clear_rows<D>(P.c, blockIdx.x - items, gridDim.x - items);
    return;
  }
  if (it.parts > 1 && it.part == 0 && kvh == 0 && threadIdx.x == 0) {
    int* const rec = P.records + 4 + 4 * it.record;
    rec[0] = it.start;
    rec[1] = it.tile * kManyRows;  // a narrow request has one tile, 0
    rec[2] = it.rows;
    rec[3] = it.slot << 12 | it.parts;
  }
  if (it.rows <= kFewRows)
    narrow_body<T, D, PLAIN>(P, it, kvh, s_kv, s_ml);
  else
    wide_body<T, D, PLAIN>(P, it, kvh, s_kv, s_seen);
}

// Joins the parts of the split tiles: grid (split tile, KV head, rows apart),
// a workgroup takes every gridDim.z'th row of the tile, its waves the parts
// of a row in turn.
template <typename T, int D>
__global__ __launch_bounds__(256) void chunk_merge_kernel(TileParams P) {
  constexpr int R = D / 64;
  __shared__ float s_acc[4][D];
  __shared__ float2 s_ml[4];
  if ((int)blockIdx.x >= P.records[0]) return;
  const int* const rec = P.records + 4 + 4 * blockIdx.x;
  const int start = rec[0], row0 = rec[1], rows = min(rec[2] - row0, kManyRows);
  const int slot = rec[3] >> 12, parts = rec[3] & 4095, kvh = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int r = blockIdx.z; r < rows; r += gridDim.z) {
    float m = kNegInf, l = 0.f, acc[R] = {};
#pragma unroll 4
    for (int p = wave; p < parts; p += 4) {
      const size_t at = ((size_t)(slot + p) * P.c.hkv + kvh) * P.part_rows + r;
      const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + 2 * at);
      float v[R];
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = P.part_acc[at * D + R * lane + i];
      const float mn = __builtin_fmaxf(m, ml.x), base = safe_max(mn);
      const float a = fast_exp2(m - base), b = fast_exp2(ml.x - base);
      l = l * a + ml.y * b;
#pragma unroll
      for (int i = 0; i < R; ++i) acc[i] = acc[i] * a + v[i] * b;
      m = mn;
    }
    if (lane == 0) s_ml[wave] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < R; ++i) s_acc[wave][R * lane + i] = acc[i];
    __syncthreads();
    if (threadIdx.x < D) {
      float top = kNegInf, sum = 0.f, out = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = __builtin_fmaxf(top, s_ml[w].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float a = fast_exp2(s_ml[w].x - safe_max(top));
        sum += s_ml[w].y * a;
        out += s_acc[w][threadIdx.x] * a;
      }
      const int n = (row0 + r) / P.c.group, h = kvh * P.c.group + row0 + r - n * P.c.group;
      P.c.out[((size_t)(start + n) * P.c.hq + h) * D + threadIdx.x] = round_to<T>(out * one_over(sum));
    }
    __syncthreads();
  }
}

// How a call with a workspace cuts its tiles; most_parts 0: it does not.
struct Cut {
  int target, most_parts, part_rows;
  size_t acc_bytes, ml_bytes, bytes;
};

Cut cut_of(const bc_shape& s, int tokens) {
  Cut c{};
  const long long steps = ((long long)s.max_pages * BC_PAGE_SIZE + kStep - 1) / kStep;
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  c.target = 2 * bch::device_cus();
  const int most = 2 * c.target / s.kv_heads;
  if (steps <= kLeastSteps || most < 2 || rows < 1) return c;
  c.most_parts = most;
  c.part_rows = rows < kManyRows ? (int)rows : kManyRows;
  const size_t slots = (size_t)most * s.kv_heads * c.part_rows;
  c.acc_bytes = slots * s.dim * sizeof(float);
  c.ml_bytes = (slots * 2 * sizeof(float) + 15) / 16 * 16;
  c.bytes = c.acc_bytes + c.ml_bytes + (4 + 4 * (size_t)(most / 2)) * sizeof(int);
  return c;
}

template <typename T, int D>
hipError_t launch_tiles(const ChunkParams& C, const Cut& cut, void* ws, unsigned grid,
                        hipStream_t st) {
  TileParams P{};
  P.c = C;
  P.target = cut.target;
  if (ws) {
    char* const at = static_cast<char*>(ws);
    P.part_acc = reinterpret_cast<float*>(at);
    P.part_ml = reinterpret_cast<float*>(at + cut.acc_bytes);
    P.records = reinterpret_cast<int*>(at + cut.acc_bytes + cut.ml_bytes);
    P.part_rows = cut.part_rows;
    P.most_parts = cut.most_parts;
  }
  if (C.cap > 0.f || C.slopes)
    chunk_tile_kernel<T, D, false><<<dim3(grid), 256, 0, st>>>(P);
  else
    chunk_tile_kernel<T, D, true><<<dim3(grid), 256, 0, st>>>(P);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || !ws) return err;
  const dim3 tiles(cut.most_parts / 2, C.hkv, cut.part_rows < 8 ? cut.part_rows : 8);
  chunk_merge_kernel<T, D><<<tiles, 256, 0, st>>>(P);
  return hipGetLastError();
}

}  // namespace

extern "C" int bc_build_tables(const int32_t* page_ids, int held, const int32_t* lengths,
                               const int32_t* counts, int batch, int max_pages, int tokens,
                               int32_t* pages, int32_t* starts, int32_t* slots,
                               int32_t* positions, bc_stream_t stream) {
  if (held < 0 || (held > 0 && !page_ids) || !lengths || !counts || batch < 1 || max_pages < 1 ||
      tokens < 0 || !pages || !starts || (tokens > 0 && (!slots || !positions)))
    return BC_ERROR_INVALID_VALUE;
  const TableParams P{page_ids, lengths, counts,    pages,     starts, slots, positions,
                      held,     batch,   max_pages, tokens};
  const int longest = tokens > max_pages ? tokens : max_pages;
  const dim3 grid(batch + 1, (longest - 1) / kTableSpan + 1);
  if (grid.y > 65535) return BC_ERROR_INVALID_VALUE;
  build_tables_kernel<<<grid, kThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
  return hipGetLastError();
}

extern "C" int bc_append_kv(bc_shape s, const bc_half* k, const bc_half* v, bc_row_strides ks,
                            bc_row_strides vs, bc_half* cache_k, bc_half* cache_v,
                            bc_pool_strides cks, bc_pool_strides cvs, const int32_t* slots,
                            int tokens, bc_stream_t stream) {
  if (!k || !v || !cache_k || !cache_v || !slots || tokens < 0 || s.physical_pages < 1 ||
      s.kv_heads < 1 || (s.dim != 64 && s.dim != 128))
    return BC_ERROR_INVALID_VALUE;
  const long long all[] = {ks.token, ks.head, vs.token, vs.head, cks.page,
                           cks.slot, cks.head, cvs.page, cvs.slot, cvs.head};
  long long bits = 0;
  for (long long x : all) {
    if (x < 0) return BC_ERROR_INVALID_VALUE;
    bits |= x;
  }
  if (tokens == 0) return BC_SUCCESS;
  const bool vec = aligned16(k) && aligned16(v) && aligned16(cache_k) && aligned16(cache_v) &&
                   bits % 8 == 0;
  const int e = vec ? 8 : 1;
  const AppendParams P{k,
                       v,
                       cache_k,
                       cache_v,
                       slots,
                       {ks.token / e, vs.token / e},
                       {ks.head / e, vs.head / e},
                       {cks.page / e, cvs.page / e},
                       {cks.slot / e, cvs.slot / e},
                       {cks.head / e, cvs.head / e},
                       tokens,
                       s.physical_pages,
                       s.kv_heads * s.dim / e,
                       s.dim / e};
  const int rows = P.row_vec >= kThreads ? 1 : kThreads / P.row_vec;
  const dim3 grid((tokens - 1) / rows + 1);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (vec)
    append_kernel<uint4><<<grid, kThreads, 0, st>>>(P, rows);
  else
    append_kernel<uint16_t><<<grid, kThreads, 0, st>>>(P, rows);
  return hipGetLastError();
}

namespace {

bool chunk_shape_ok(const bc_shape& s, int tokens) {
  return s.batch >= 1 && s.query_heads >= 1 && s.kv_heads >= 1 &&
         s.query_heads % s.kv_heads == 0 && s.query_heads <= BC_MAX_CHUNK_HEADS &&
         (s.dim == 64 || s.dim == 128) && s.max_pages >= 1 && s.physical_pages >= 1 && tokens >= 0;
}

}  // namespace

extern "C" size_t bc_chunk_attention_workspace_size(bc_shape s, int tokens) {
  return chunk_shape_ok(s, tokens) ? cut_of(s, tokens).bytes : 0;
}

extern "C" int bc_chunk_attention(bc_shape s, bc_chunk_inputs in, void* workspace,
                                  size_t workspace_bytes, bc_stream_t stream) {
  if (!chunk_shape_ok(s, in.tokens) || in.window < 0 || !(in.scale > 0.f) ||
      !(in.scale < __builtin_huge_valf()) || !(in.cap >= 0.f) ||
      !(in.cap < __builtin_huge_valf()) ||
      (in.dtype != BC_FLOAT16 && in.dtype != BC_BFLOAT16))
    return BC_ERROR_INVALID_VALUE;
  if (!in.k || !in.v || !in.pages || !in.lengths || !in.starts) return BC_ERROR_INVALID_VALUE;
  const long long all[] = {in.q_strides.token, in.q_strides.head, in.k_strides.page,
                           in.k_strides.slot,  in.k_strides.head, in.v_strides.page,
                           in.v_strides.slot,  in.v_strides.head};
  long long bits = 0;
  for (long long x : all) {
    if (x < 0) return BC_ERROR_INVALID_VALUE;
    bits |= x;
  }
  if (in.tokens == 0) return BC_SUCCESS;
  if (!in.q || !in.output) return BC_ERROR_INVALID_VALUE;
  const ChunkParams P{in.q,
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
                      s.query_heads / s.kv_heads,
                      s.max_pages,
                      s.physical_pages,
                      in.causal != 0,
                      in.window,
                      in.scale,
                      in.cap};
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // Tiles of rows take 16-byte loads, 32-bit offsets inside a page and 31 bits
  // of rows and workgroups; anything else goes row by row.
  const long long rows = (long long)in.tokens * P.group;
  const Cut cut = cut_of(s, in.tokens);
  const bool use = cut.bytes > 0 && workspace && aligned16(workspace) && workspace_bytes >= cut.bytes;
  const long long tiles = (in.tokens < s.batch ? in.tokens : s.batch) + rows / kManyRows +
                          (use ? cut.most_parts : 0);
  const long long grid = tiles * s.kv_heads + 1;
  const long long far = 1 << 26;
  const bool tiled = aligned16(in.q) && aligned16(in.k) && aligned16(in.v) && aligned16(in.output) &&
                     bits % 8 == 0 && in.k_strides.slot < far && in.v_strides.slot < far &&
                     rows <= 1 << 30 && grid <= 0x7fffffff;
  void* const ws = use ? workspace : nullptr;
  if (tiled) {
    if (in.dtype == BC_FLOAT16)
      return s.dim == 64 ? launch_tiles<_Float16, 64>(P, cut, ws, (unsigned)grid, st)
                         : launch_tiles<_Float16, 128>(P, cut, ws, (unsigned)grid, st);
    return s.dim == 64 ? launch_tiles<__bf16, 64>(P, cut, ws, (unsigned)grid, st)
                       : launch_tiles<__bf16, 128>(P, cut, ws, (unsigned)grid, st);
  }
  if (in.dtype == BC_FLOAT16)
    s.dim == 64 ? launch_rows<_Float16, 64>(P, st) : launch_rows<_Float16, 128>(P, st);
  else
    s.dim == 64 ? launch_rows<__bf16, 64>(P, st) : launch_rows<__bf16, 128>(P, st);
  return hipGetLastError();
}
