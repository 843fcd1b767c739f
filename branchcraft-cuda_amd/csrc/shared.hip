// Attention of requests that begin with the same pages, for gfx950: forks of one
// prompt (bc_shared_chunk_attention).  The tokens that a group of requests share
// are an entry of their own in the plan of the chunk attention, with the rows of
// all members, and its partials are joined with those of each member's own tokens.
//
// No reference counterpart: the reference reads every request's pages by
// themselves (src/paged_gqa.cu).
#include "bc_tiles.h"

namespace {

struct ForkCut : Cut {
  int single_rows, total_rows, own_records;
};

// How a call cuts its work; bytes 0: every request reads its own pages.
ForkCut fork_cut(const bc_shape& s, int tokens, int groups) {
  ForkCut c{};
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  if (groups < 1 || s.batch < 2 || rows < 1 || rows > 1 << 28 ||
      (s.batch + (long long)groups) * (s.max_pages + 1ll) > 1 << 28 ||
      (long long)s.batch * s.query_heads > 1 << 26)
    return c;
  c.target = 2 * bch::device_cus();
  const int per = s.dim == 64 ? 4 : 2;
  c.waves = per * c.target / s.kv_heads > 1 ? per * c.target / s.kv_heads : 1;
  const long long own = rows < 32ll * s.batch ? rows : 32ll * s.batch;
  const long long of_groups = rows < 32ll * groups ? rows : 32ll * groups;
  const long long narrow = 32ll * c.waves + own + of_groups;
  c.most_parts = 2 * c.target / s.kv_heads;
  c.part_rows = kManyRows;
  const long long single = narrow + (long long)c.most_parts * c.part_rows, all = single + 2 * rows;
  const long long per_side = rows / kManyRows + 1;
  if (all * s.kv_heads > 0x7fffffff) return ForkCut{};
  c.narrow_rows = (int)narrow;
  c.single_rows = (int)single;
  c.total_rows = (int)all;
  c.own_records = (int)(per_side + s.batch);
  const size_t slots = (size_t)all * s.kv_heads;
  c.acc_bytes = slots * s.dim * sizeof(float);
  c.ml_bytes = (slots * 2 * sizeof(float) + 15) / 16 * 16;
  c.bytes = c.acc_bytes + c.ml_bytes + (c.own_records + per_side + groups) * sizeof(int4);
  return c;
}

template <typename T, int D>
hipError_t launch_forks(const ChunkParams& C, const ForkCut& cut, void* ws, unsigned grid, hipStream_t st) {
  char* const at = static_cast<char*>(ws);
  TileParams P{};
  P.c = C;
  P.target = cut.target;
  P.part_acc = reinterpret_cast<float*>(at);
  P.part_ml = reinterpret_cast<float*>(at + cut.acc_bytes);
  P.records = reinterpret_cast<int4*>(at + cut.acc_bytes + cut.ml_bytes);
  P.waves = cut.waves;
  P.most_parts = cut.most_parts;
  P.part_rows = cut.part_rows;
  P.narrow_rows = cut.narrow_rows;
  P.single_rows = cut.single_rows;
  P.total_rows = cut.total_rows;
  P.own_records = cut.own_records;
  if (C.cap > 0.f)
    chunk_tile_kernel<T, D, Form::kCap, false, true><<<dim3(grid), 256, 0, st>>>(P);
  else if (C.slopes)
    chunk_tile_kernel<T, D, Form::kBias, false, true><<<dim3(grid), 256, 0, st>>>(P);
  else
    chunk_tile_kernel<T, D, Form::kPlain, false, true><<<dim3(grid), 256, 0, st>>>(P);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  // A round of waves, eight workgroups per CU, with the rows of a token and KV head
  // apart where there is room.
  const long long pairs = (long long)C.tokens * C.hkv, most = 4ll * cut.target;
  long long apart = 4 * most / pairs;
  apart = apart < 1 ? 1 : apart < C.group ? apart : C.group;
  const long long join = (pairs * apart + 3) / 4;
  fork_join_kernel<T, D><<<dim3((unsigned)(join < most ? join : most)), 256, 0, st>>>(P, (int)apart);
  return hipGetLastError();
}

}  // namespace

extern "C" size_t bc_shared_chunk_attention_workspace_size(bc_shape s, int tokens, int group_count) {
  return chunk_shape_ok(s, tokens) && group_count >= 0 && group_count <= s.batch
             ? fork_cut(s, tokens, group_count).bytes
             : 0;
}

extern "C" int bc_shared_chunk_attention(bc_shape s, bc_chunk_inputs in, const int32_t* groups,
                                         const int32_t* shared, int group_count, void* workspace,
                                         size_t workspace_bytes, bc_stream_t stream) {
  if (!chunk_shape_ok(s, in.tokens) || !chunk_inputs_ok(in) || !groups || group_count < 0 ||
      (group_count > 0 && !shared) || group_count > s.batch)
    return BC_ERROR_INVALID_VALUE;
  const ForkCut cut = fork_cut(s, in.tokens, group_count);
  const bool use = cut.bytes > 0 && workspace && aligned16(workspace) && workspace_bytes >= cut.bytes;
  // As in bc_chunk_attention.  Rows count twice, as a request's and as a group's;
  // under a window, or with documents, a group of few rows is of the wide form.
  const long long rows = (long long)in.tokens * (s.query_heads / s.kv_heads);
  const long long few = in.window > 0 || in.first ? (long long)(kFewRows + 1) * group_count : 0;
  const long long grid = split_grid(s, cut, 2 * rows + few, (long long)s.batch + group_count);
  const long long far = 1 << 26;
  if (!use || !aligned16(in.q) || !aligned16(in.k) || !aligned16(in.v) || !aligned16(in.output) ||
      stride_bits(in) % 8 != 0 || in.k_strides.slot >= far || in.v_strides.slot >= far || grid > kMostGroups)
    return bc_chunk_attention(s, in, nullptr, 0, stream);
  if (!in.q || !in.output) return BC_ERROR_INVALID_VALUE;
  ChunkParams P = chunk_params(s, in);
  P.groups = groups;
  P.shared = shared;
  P.group_count = group_count;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (in.dtype == BC_FLOAT16)
    return s.dim == 64 ? launch_forks<_Float16, 64>(P, cut, workspace, (unsigned)grid, st)
                       : launch_forks<_Float16, 128>(P, cut, workspace, (unsigned)grid, st);
  return s.dim == 64 ? launch_forks<__bf16, 64>(P, cut, workspace, (unsigned)grid, st)
                     : launch_forks<__bf16, 128>(P, cut, workspace, (unsigned)grid, st);
}
