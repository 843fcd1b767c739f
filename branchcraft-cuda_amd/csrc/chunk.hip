// Chunks of new tokens over the paged cache, for gfx950: the block tables and
// slot maps of a step from its requests' lengths (bc_build_tables), the new
// tokens' K and V rows into the pool (bc_append_kv), and the attention of the
// new tokens over their requests' pages (bc_chunk_attention).
//
// No reference counterpart: the reference attends one token per request
// (src/paged_gqa.cu) or a tree of draft tokens outside the cache
// (src/tree_attention.cu), and fills pages on the host
// (python/branchcraft_torch/transaction.py:64-81).
#include "bc_device.h"

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
  if (P.causal) hi = min(hi, P.prefix ? max(pos, P.prefix[b] - 1) : pos);
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
    const int pos = P.lengths[b] - (min(P.starts[b + 1], P.tokens) - t);
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

extern "C" size_t bc_chunk_attention_workspace_size(bc_shape s, int tokens) { return 0; }

extern "C" int bc_chunk_attention(bc_shape s, bc_chunk_inputs in, void* workspace,
                                  size_t workspace_bytes, bc_stream_t stream) {
  if (s.batch < 1 || s.query_heads < 1 || s.kv_heads < 1 || s.query_heads % s.kv_heads != 0 ||
      (s.dim != 64 && s.dim != 128) || s.max_pages < 1 || s.physical_pages < 1 ||
      in.tokens < 0 || in.window < 0 || !(in.scale > 0.f) || !(in.scale < __builtin_huge_valf()) ||
      !(in.cap >= 0.f) || !(in.cap < __builtin_huge_valf()) ||
      (in.dtype != BC_FLOAT16 && in.dtype != BC_BFLOAT16) || s.query_heads > BC_MAX_CHUNK_HEADS)
    return BC_ERROR_INVALID_VALUE;
  if (!in.k || !in.v || !in.pages || !in.lengths || !in.starts) return BC_ERROR_INVALID_VALUE;
  const long long all[] = {in.q_strides.token, in.q_strides.head, in.k_strides.page,
                           in.k_strides.slot,  in.k_strides.head, in.v_strides.page,
                           in.v_strides.slot,  in.v_strides.head};
  for (long long x : all)
    if (x < 0) return BC_ERROR_INVALID_VALUE;
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
  if (in.dtype == BC_FLOAT16)
    s.dim == 64 ? launch_rows<_Float16, 64>(P, st) : launch_rows<_Float16, 128>(P, st);
  else
    s.dim == 64 ? launch_rows<__bf16, 64>(P, st) : launch_rows<__bf16, 128>(P, st);
  return hipGetLastError();
}
