// Chunks of new tokens over the paged cache, for gfx950: the block tables and
// slot maps of a step from its requests' lengths (bc_build_tables), the new
// tokens' K and V rows into the pool (bc_append_kv), and the attention of the
// new tokens over their requests' pages (bc_chunk_attention).
//
// No reference counterpart: the reference attends one token per request
// (src/paged_gqa.cu) or a tree of draft tokens outside the cache
// (src/tree_attention.cu), and fills pages on the host
// (python/branchcraft_torch/transaction.py:64-81).
#include "bc_tiles.h"

namespace {

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

constexpr int kTableSpan = kThreads;  // table entries, and rows of the slot map, at a time

__device__ __forceinline__ long long wave_sum_ll(long long x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s, 64);
  return x;
}

// grid = (batch + 1, slices).  Workgroup (b, s) sums the pages and new tokens
// of the requests before b, so that no workgroup waits for another, and
// writes every slices'th span of b's table row and of its rows of the slot
// map; workgroup row `batch` writes what lies behind the last request.
// Latency-bound, four rounds of loads and stores: 64 single tokens over tables
// of 256 pages 3.3 us, 64 new prompts of 128-4096 tokens (1.2 MB) 4.2 (8.0 with
// as many slices as the longest possible request has).  A call costs its host 7.
__global__ __launch_bounds__(kThreads) void build_tables_kernel(TableParams P) {
  const int b = blockIdx.x, tid = threadIdx.x, step = gridDim.y * kTableSpan;
  const bool tail = b == P.batch;
  const int len = tail ? 0 : max(P.lengths[b], 0), count = tail ? 0 : max(P.counts[b], 0);
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
  const int begin = blockIdx.y * kTableSpan + tid;
  if (begin == 0) P.starts[b] = start;
  if (tail) {  // rows behind the last request
    for (int i = begin; i < P.tokens - start; i += step) {
      P.slots[start + i] = -1;
      P.positions[start + i] = -1;
    }
    return;
  }
  const int n = min(count, P.tokens - start);
  const int old = len - count;  // may be negative: such rows have no token
  // Pages that the list holds for this request, within its row of the table.
  const int used = (int)max(0ll, min(min((len + BC_PAGE_SIZE - 1ll) / BC_PAGE_SIZE,
                                         (long long)P.max_pages), P.held - before));
  int32_t* const row = P.pages + (size_t)b * P.max_pages;
  for (int i = begin; i < P.max_pages; i += step) row[i] = i < used ? P.ids[before + i] : -1;
  for (int i = begin; i < n; i += step) {
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
// Memory-bound: 8192 rows of 8 heads x 128 out of a fused projection (67 MB moved)
// 12.1 us, 5.5 TB/s; torch's copy moves as much, contiguous, in 10.1 (6.6 TB/s,
// some of it out of the last-level cache), half a GB and more at 5.2-5.4; 64
// rows 2.6 us.
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
  static_assert(BC_MAX_TABLE_REQUESTS + 1 <= kMostGroups, "a workgroup row per request and one");
  if (max_pages > BC_MAX_TABLE_PAGES || tokens >= 1 << 27 || batch > BC_MAX_TABLE_REQUESTS)
    return BC_ERROR_INVALID_VALUE;
  const int longest = tokens > max_pages ? tokens : max_pages;
  // At most about four workgroups per CU.
  const int spans = (longest - 1) / kTableSpan + 1, rounds = 4 * bch::device_cus() / (batch + 1);
  const dim3 grid(batch + 1, spans < rounds ? spans : rounds < 1 ? 1 : rounds);
  build_tables_kernel<<<grid, kThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
  return hipGetLastError();
}

extern "C" int bc_append_kv(bc_shape s, const bc_half* k, const bc_half* v, bc_row_strides ks,
                            bc_row_strides vs, bc_half* cache_k, bc_half* cache_v,
                            bc_pool_strides cks, bc_pool_strides cvs, const int32_t* slots,
                            int tokens, bc_stream_t stream) {
  if (!k || !v || !cache_k || !cache_v || !slots || tokens < 0 || s.physical_pages < 1 ||
      s.kv_heads < 1 || s.kv_heads > BC_MAX_CHUNK_HEADS || (s.dim != 64 && s.dim != 128))
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
  AppendParams P{k,
                 v,
                 cache_k,
                 cache_v,
                 slots,
                 {ks.token / e, vs.token / e},
                 {ks.head / e, vs.head / e},
                 {cks.page / e, cvs.page / e},
                 {cks.slot / e, cvs.slot / e},
                 {cks.head / e, cvs.head / e},
                 0,
                 s.physical_pages,
                 s.kv_heads * s.dim / e,
                 s.dim / e};
  const int rows = P.row_vec >= kThreads ? 1 : kThreads / P.row_vec;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // One launch, or several for rows past kMostGroups workgroups (a loop in the
  // kernel costs every call 1 %).
  const long long most = (long long)kMostGroups * rows;
  for (long long t0 = 0; t0 < tokens; t0 += most) {
    P.k = k + t0 * ks.token;
    P.v = v + t0 * vs.token;
    P.slots = slots + t0;
    P.tokens = (int)(tokens - t0 < most ? tokens - t0 : most);
    const dim3 grid((P.tokens - 1) / rows + 1);
    if (vec)
      append_kernel<uint4><<<grid, kThreads, 0, st>>>(P, rows);
    else
      append_kernel<uint16_t><<<grid, kThreads, 0, st>>>(P, rows);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return BC_SUCCESS;
}

extern "C" size_t bc_chunk_attention_workspace_size(bc_shape s, int tokens) {
  return chunk_shape_ok(s, tokens) ? cut_of(s, tokens, false).bytes : 0;
}

extern "C" int bc_chunk_attention(bc_shape s, bc_chunk_inputs in, void* workspace,
                                  size_t workspace_bytes, bc_stream_t stream) {
  if (!chunk_shape_ok(s, in.tokens) || !chunk_inputs_ok(in)) return BC_ERROR_INVALID_VALUE;
  if (in.tokens == 0) return BC_SUCCESS;
  if (!in.q || !in.output) return BC_ERROR_INVALID_VALUE;
  MoreParams M{};
  M.t.c = chunk_params(s, in);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // Tiles of rows take 16-byte loads, 32-bit offsets inside a page and 31 bits
  // of rows and workgroups; anything else goes row by row.
  const long long rows = (long long)in.tokens * M.t.c.group;
  const Cut cut = cut_of(s, in.tokens, false);
  const bool use = cut.bytes > 0 && workspace && aligned16(workspace) && workspace_bytes >= cut.bytes;
  const long long grid = tile_grid(s, in.tokens, cut, use);
  const long long far = 1 << 26;
  const bool tiled = aligned16(in.q) && aligned16(in.k) && aligned16(in.v) && aligned16(in.output) &&
                     stride_bits(in) % 8 == 0 && in.k_strides.slot < far && in.v_strides.slot < far &&
                     rows <= 1 << 30 && grid <= kMostGroups;
  void* const ws = use ? workspace : nullptr;
  if (tiled) return launch_tiles<false>(M, s.dim, in.dtype, cut, ws, grid, st);
  return launch_rows<false>(M, s.dim, in.dtype, st);
}
