// Attention of requests that begin with the same pages, for gfx950: forks of one
// prompt (bc_shared_chunk_attention).
//
// The softmax over a row's tokens joins the states (maximum, sum, weighted sum of V)
// of two sets of them: those that its group shares, and its request's own.  A batch
// has an entry for each: one per request, for its own tokens, and one per group, the
// rows of all members over the first one's pages, so that these are read once per
// tile of rows and not once per request.  The entries are cut into parts as the
// requests of the chunk attention are, every part leaves its state, and the join
// takes a row's parts of both.
//
// No reference counterpart: the reference reads every request's pages by
// themselves (src/paged_gqa.cu).
#include "bc_tiles.h"

namespace {

// ---------------------------------------------------------------------------
// The plan

// Group g: its members and the tokens they share, none of fewer than two members.
struct Group {
  int g0, g1, shared;
};

__device__ __forceinline__ Group group_at(const ChunkParams& P, int g) {
  const int from = more(P).groups[g], to = more(P).groups[g + 1], tokens = more(P).shared[g];  // in one round
  Group x;
  x.g0 = min(max(from, 0), P.batch);
  x.g1 = min(max(to, 0), P.batch);
  x.shared = x.g1 - x.g0 > 1 ? min(max(tokens, 0), P.max_pages * BC_PAGE_SIZE) : 0;
  return x;
}

// The groups i .. i + 63, a lane each; behind the last, groups of no request.
__device__ __forceinline__ Group groups_from(const ChunkParams& P, int i) {
  const int lane = threadIdx.x & 63;
  const Group x = group_at(P, min(i + lane, more(P).group_count - 1));
  return i + lane < more(P).group_count ? x : Group{0x7fffffff, 0, 0};
}

// Of the 64 groups that the lanes hold, that of request b, a lane's own; -1, and 0
// tokens, where it has none.  All lanes of the wave take part.
__device__ __forceinline__ int group_in(const Group& x, int b, int& shared) {
  const int n = count_upto(x.g0, b) - 1, from = max(n, 0);
  const int end = __shfl(x.g1, from, 64), tokens = __shfl(x.shared, from, 64);
  shared = n >= 0 && b < end ? tokens : 0;
  return n;
}

// The group of request b, a lane's own, with b rising over the lanes: of the first 64
// (`head`), or of those from the last that begins at or before the first lane's
// request on, found in 64 steps at a time.  Looked through from the first on they
// were 32 rounds of loads for 2048 groups, of every block of requests.
__device__ __forceinline__ int group_of(const ChunkParams& P, const Group& head, int b, int& shared) {
  int at = group_in(head, b, shared);
  const int count = more(P).group_count;
  if (count <= 64) return at;
  const int lane = threadIdx.x & 63, first = __builtin_amdgcn_readfirstlane(b);
  int from = 0;
  for (int n = count; n > 64;) {
    const int step = (n + 63) / 64, i = lane * step;
    const bool upto = i < n && more(P).groups[from + min(i, n - 1)] <= first;
    const int skipped = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(upto)) - 1, 0) * step;
    from += skipped;
    n = min(step, n - skipped);
  }
  for (int i = from; i < count; i += 64) {
    const Group x = groups_from(P, i);
    int tokens;
    const int n = group_in(x, b, tokens);
    if (n >= 0) {
      at = i + n;
      shared = tokens;
    }
    if (__builtin_amdgcn_readlane(x.g0, 63) > __builtin_amdgcn_readlane(b, 63)) break;
  }
  return at;
}

// The entries of a batch in blocks of 64, one per lane: the requests' blocks, then
// the groups'.  The first two of the requests and the first of the groups stay, and
// all that these do not depend on each other for is loaded in one round.
struct Entries {
  int lane, own_blocks, blocks;
  Group head;  // a lane's of the first 64 groups
  AskedEntry own0, own1, groups0;

  __device__ __forceinline__ explicit Entries(const ChunkParams& C) : lane(threadIdx.x & 63), own1{} {
    own_blocks = (C.batch + 63) / 64;
    blocks = own_blocks + (more(C).group_count + 63) / 64;
    const int3 x0 = load(C, lane), x1 = load(C, 64 + lane);
    head = groups_from(C, 0);
    own0 = request(C, x0, lane);
    if (own_blocks > 1) own1 = request(C, x1, 64 + lane);
    groups0 = group(C, head, lane);
  }
  __device__ __forceinline__ AskedEntry at(const ChunkParams& C, int block) const {
    if (block == own_blocks) return groups0;
    if (block == 0) return own0;
    if (block == 1 && own_blocks > 1) return own1;
    if (block < own_blocks) return request(C, load(C, 64 * block + lane), 64 * block + lane);
    const int g = 64 * (block - own_blocks);
    return group(C, groups_from(C, g), g + lane);
  }

 private:
  static __device__ __forceinline__ int3 load(const ChunkParams& C, int b) {
    const int i = min(b, C.batch - 1);
    return make_int3(C.starts[i], C.starts[i + 1], C.lengths[i]);
  }
  __device__ __forceinline__ AskedEntry request(const ChunkParams& C, int3 x, int b) const {
    AskedEntry a{};
    int floor;
    group_of(C, head, b, floor);
    if (b < C.batch) {
      a.floor = floor;
      a.start = min(max(x.x, 0), C.tokens);
      a.n = max(min(max(x.y, 0), C.tokens) - a.start, 0);
      a.full = max(x.z, 0);
      a.len = min(a.full, C.max_pages * BC_PAGE_SIZE);
      a.rows = a.n * C.group;
      ask_work(C, a, floor, true);
    }
    return a;
  }
  __device__ __forceinline__ AskedEntry group(const ChunkParams& C, const Group& m, int g) const {
    AskedEntry a{};
    // Where the lanes hold all requests, the ends of its rows are theirs.
    int from = __shfl(own0.start, m.g0, 64), to = __shfl(own0.start + own0.n, m.g1 - 1, 64);
    const bool is = g < more(C).group_count && m.shared > 0;
    if (is && own_blocks > 1) {
      from = min(max(C.starts[m.g0], 0), C.tokens);
      to = min(max(C.starts[m.g1], 0), C.tokens);
    }
    if (is) {
      a.g0 = m.g0;
      a.g1 = m.g1;
      a.start = from;
      a.n = max(to - from, 0);
      a.len = m.shared;
      a.rows = a.n * C.group;
      // What the members' rows see of it under a window, or of documents, takes a
      // look at each of them: the wide form does.
      const bool wide = a.rows > kFewRows || (a.rows > 0 && (C.window > 0 || C.first));
      a.tiles = wide ? (a.rows + kManyRows - 1) / (kManyRows) : 0;
      a.steps = wide ? wide_steps(C, a.len) : 0;
      a.narrow = !wide && a.rows > 0 ? (a.len + 31) / 32 : 0;
    }
    return a;
  }
};

// How the batch is cut, see Cutting: a tile of the narrow form takes each of its
// waves about kTileTime times as long as a step of the wide one takes its
// workgroup.  What the narrow entries leave of a round of workgroups is filled with
// shares.
constexpr float kTileTime = 1.2f;
constexpr int kLeastTiles = 2;  // fewest per wave

__device__ __forceinline__ Cutting cut_entries(const TileParams& P, const Entries& all) {
  const ChunkParams& C = P.c;
  float work = 0.f;
  int narrow = 0, tiles = 0;
  for (int block = 0; block < all.blocks; ++block) {
    const AskedEntry x = all.at(C, block);
    work += (float)x.tiles * (float)x.steps;
    narrow += x.narrow;
    tiles += x.tiles;
  }
  Cutting c;
  work = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wave_sum(work))));
  c.narrow = lanes_sum(narrow);
  const float run = ((float)c.narrow + 4.f / kTileTime * work) / (float)P.waves;
  c.run = max(min((int)__builtin_fminf(run, 1e9f) + 1, c.narrow), (c.narrow + P.waves - 1) / P.waves);
  c.run = max(c.run, kLeastTiles);
  c.groups = ((c.narrow + c.run - 1) / c.run * C.hkv + 3) / 4;
  // n tiles have less than work / share + n parts: one more than a round holds
  // would take the time of a second round.
  const int left = max(P.target - c.groups, P.target / 4) / C.hkv - lanes_sum(tiles);
  const float share = work / (float)max(left, P.target / (2 * C.hkv) + 1);
  c.share = max(kLeastSteps, (int)__builtin_fminf(share, 1e9f) + 1);
  return c;
}

// Item `idx` of the wide entries' tiles and their parts, see plan_item.
__device__ __forceinline__ Item plan_entry(const TileParams& P, const Entries& all, int share, long long idx) {
  const ChunkParams& C = P.c;
  const int lane = threadIdx.x & 63;
  Item it{};
  long long before = 0;
  int slots = 0;
  for (int block = 0; block < all.blocks; ++block) {
    const AskedEntry a = all.at(C, block);
    const int parts = a.steps > share ? (a.steps + share - 1) / share : 1;
    const int mine = a.tiles * parts, cut_parts = parts > 1 ? mine : 0;
    const int upto = lanes_upto(mine);
    const int total = __builtin_amdgcn_readlane(upto, 63);
    if (idx >= before && idx - before < total) {
      const int local = (int)(idx - before);
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > local));
      it.found = true;
      it.r = request_at<true>(C, a, 64 * block, at);
      it.parts = __builtin_amdgcn_readlane(parts, at);
      const int in = local - __builtin_amdgcn_readlane(upto - mine, at);
      const int nth = it.parts == 1 ? in : in / it.parts;
      it.part = in - nth * it.parts;
      it.tile = __builtin_amdgcn_readlane(a.tiles, at) - 1 - nth;
      if (it.parts > 1) {
        it.slot = slots + lanes_sum(lane < at ? cut_parts : 0) + in - it.part;
        if (it.slot < 0 || it.slot + it.parts > P.most_parts) it.parts = 1;  // cannot be, see Cutting
      }
      return it;
    }
    before += total;
    slots += lanes_sum(cut_parts);
  }
  it.items = before;
  return it;
}

// ---------------------------------------------------------------------------
// The kernels

// 64 single tokens over a shared 32768 and 16 to 1024 of their own (32/8 heads, D =
// 128, 263 MB): 71 us, 3.7 TB/s, and the join 9; HBM would take 41.  The group's two
// tiles of rows per KV head run over the same pages, once from L2, beside the
// requests' own parts; matrix units 28 %, vector units 34 % of the cycles.  The biased
// and capped forms at D = 64 keep five registers in memory, outside their loops.
template <typename T, int D, Form FORM>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void fork_tile_kernel(MoreParams) {
  __shared__ __attribute__((aligned(256))) uint16_t s_kv[2 * 2 * kStep * D];
  __shared__ Seen s_seen[4];
  __shared__ int s_bad[4];
  const Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  const TileParams& P = reread(args);
  asm volatile("" ::"s"(more(P.c).groups), "s"(more(P.c).shared), "s"(more(P.c).group_count));
  pin_plan(P);
  const Entries all(P.c);
  const Cutting cut = cut_entries(P, all);
  // The narrow entries first, as in chunk_tile_kernel.
  if ((int)blockIdx.x < cut.groups) {
    const TileParams& A = reread(args);
    pin_rows<false>(A);
    // Anew, so that the other blocks' registers do not live through the tiles.
    auto ask = [&](int b0) { return Entries(A.c).at(A.c, b0 / 64); };
    flat_body<T, D, FORM, false, true>(A, all.own0, 64 * all.blocks, ask, cut, s_kv);
    return;
  }
  const int in = blockIdx.x - cut.groups, at = divide(in, P.c.hkv, P.c.hkv_mul);
  const int kvh = in - at * P.c.hkv;
  const Item it = plan_entry(P, all, cut.share, at);
  if (!it.found) {
    const long long items = it.items * P.c.hkv + cut.groups;
    clear_rows<D>(P.c, blockIdx.x - items, gridDim.x - items);
    return;
  }
  if (it.part == 0 && kvh == 0 && threadIdx.x == 0)
    put_fork_record(P, it.r, it.tile, it.parts,
                    it.parts > 1 ? P.narrow_rows + it.slot * P.part_rows
                                 : single_row(P, it.r) + it.tile * kManyRows,
                    P.part_rows);
  const TileParams& A = reread(args);
  pin_rows<false>(A);
  wide_body<T, D, FORM, false, true>(A, args, it, kvh, s_kv, s_seen, s_bad);
}

// The join with groups: `apart` waves share the rows of a new token and KV head; of
// a wave, each group of D / 4 lanes takes the parts of the request's own tokens and
// then of its group's in turn.  Rows that their entry has written as output are
// left.
template <typename T, int D>
__global__ __launch_bounds__(256) void fork_join_kernel(MoreParams M, int apart) {
  constexpr int LPR = D / 4, GW = 64 / LPR;
  const TileParams& P = M.t;
  const ChunkParams& C = P.c;
  const int lane = threadIdx.x & 63, grp = lane / LPR, c = lane % LPR;
  const long long total = (long long)C.tokens * C.hkv * apart, step = 4ll * gridDim.x;
  for (long long x = 4ll * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); x < total; x += step) {
    const long long pair = x / apart;
    const int sub = (int)(x - pair * apart), t = (int)(pair / C.hkv), kvh = (int)(pair - (long long)t * C.hkv);
    // The request of token t, the first of its rows, and its group, of loads in one
    // round for up to 64 of either.
    const Group head = groups_from(C, 0);
    int b = 0, own0 = 0, block = 0, from = 0;
    for (int i = 0; i < C.batch; i += 64) {
      from = C.starts[min(i + lane, C.batch - 1)];
      const int to = C.starts[min(i + lane, C.batch - 1) + 1];
      const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i + lane < C.batch && to <= t));
      b += n;
      block = i;
      if (n < 64) {
        own0 = __builtin_amdgcn_readlane(from, n);
        break;
      }
    }
    if (b >= C.batch || own0 > t) continue;
    int shared;
    const int g = __builtin_amdgcn_readfirstlane(group_of(C, head, b, shared));
    shared = __builtin_amdgcn_readfirstlane(shared);
    auto start_of = [&](int from) { return min(max(from, 0), C.tokens); };
    own0 = start_of(own0);
    int all0 = 0;
    if (shared > 0) {  // from what the lanes have, where they have it
      const int g0 = M.group_count <= 64 ? __builtin_amdgcn_readlane(head.g0, g & 63) : group_at(C, g).g0;
      all0 = start_of(g0 >= block ? __builtin_amdgcn_readlane(from, (g0 - block) & 63) : C.starts[g0]);
    }
    // The records of up to 32 rows in one round: a lane each, of the request's entry
    // and, in the upper half of the wave, of the group's.
    for (int r0 = sub; r0 < C.group; r0 += 32 * apart) {
      const bool of_group = lane >= 32;
      const int mine = r0 + (lane & 31) * apart, start = of_group ? all0 : own0;
      int parts = 0, first = 0, stride = 0;
      if (mine < C.group && t >= start && (!of_group || shared > 0)) {
        const int row = (t - start) * C.group + mine, tile = row / kManyRows;
        const int4 rec = P.records[record_of(P, of_group ? C.batch + g : b, start, tile)];
        // Where starts decrease, a record may be another's or no one's.
        const long long last = rec.y + (long long)max(rec.x - 1, 0) * rec.z + row - tile * kManyRows;
        const bool sane = rec.x > 0 && rec.x <= 2 * (P.waves + P.most_parts) && rec.y >= 0 && rec.z > 0 &&
                          last < M.total_rows;
        parts = sane ? rec.x : 0;
        first = rec.y + row - tile * kManyRows;
        stride = rec.z;
      }
      for (int i = 0; i < 32 && r0 + i * apart < C.group; ++i) {
        const int r = r0 + i * apart;
        const int own_parts = __builtin_amdgcn_readlane(parts, i), all_parts = __builtin_amdgcn_readlane(parts, 32 + i);
        const int own_first = __builtin_amdgcn_readlane(first, i), all_first = __builtin_amdgcn_readlane(first, 32 + i);
        const int own_stride = __builtin_amdgcn_readlane(stride, i), all_stride = __builtin_amdgcn_readlane(stride, 32 + i);
        if (shared <= 0 && own_parts < 2) continue;
        float m = kNegInf, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int p = grp; p < own_parts + all_parts; p += GW) {
          const int at = p < own_parts ? own_first + p * own_stride : all_first + (p - own_parts) * all_stride;
          const size_t row = partial_row(P, at, kvh);
          const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + 2 * row);
          join(m, l, acc, ml.x, ml.y, *reinterpret_cast<const float4*>(P.part_acc + row * D + 4 * c));
        }
#pragma unroll
        for (int s = LPR; s < 64; s <<= 1)
          join(m, l, acc, shfl_xor_f(m, s), shfl_xor_f(l, s),
               make_float4(shfl_xor_f(acc.x, s), shfl_xor_f(acc.y, s), shfl_xor_f(acc.z, s),
                           shfl_xor_f(acc.w, s)));
        const float inv = one_over(l);
        if (grp == 0)
          *reinterpret_cast<uint2*>(C.out + ((size_t)t * C.hq + kvh * C.group + r) * D + 4 * c) =
              make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The call

struct ForkCut : Cut {
  int single_rows, total_rows, own_records;
};

// How a call cuts its work; bytes 0: every request reads its own pages.
ForkCut fork_cut(const bc_shape& s, int tokens, int groups) {
  ForkCut c{};
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  if (groups < 1 || rows < 1 || !bch::sharing_pays(s, tokens, 0) || rows > 1 << 28 ||
      (s.batch + (long long)groups) * (s.max_pages + 1ll) > 1 << 28 ||
      (long long)s.batch * s.query_heads > 1 << 26)
    return c;
  const int per_cu = s.dim == 64 ? 3 : 2;
  c.target = per_cu * bch::device_cus();  // workgroups in a round
  c.waves = 4 * c.target / s.kv_heads > 1 ? 4 * c.target / s.kv_heads : 1;
  const long long own = rows < 32ll * s.batch ? rows : 32ll * s.batch;
  const long long of_groups = rows < 32ll * groups ? rows : 32ll * groups;
  const long long narrow = 32ll * c.waves + own + of_groups;
  c.most_parts = 2 * c.target / s.kv_heads;
  c.part_rows = kManyRows;
  const long long single = narrow + (long long)c.most_parts * c.part_rows, all = single + 2 * rows;
  const long long per_side = rows / c.part_rows + 1;
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
hipError_t launch_forks(MoreParams M, const ForkCut& cut, void* ws, unsigned grid, hipStream_t st) {
  char* const at = static_cast<char*>(ws);
  TileParams& P = M.t;
  const ChunkParams& C = P.c;
  P.target = cut.target;
  P.part_acc = reinterpret_cast<float*>(at);
  P.part_ml = reinterpret_cast<float*>(at + cut.acc_bytes);
  P.records = reinterpret_cast<int4*>(at + cut.acc_bytes + cut.ml_bytes);
  P.waves = cut.waves;
  P.most_parts = cut.most_parts;
  P.part_rows = cut.part_rows;
  P.narrow_rows = cut.narrow_rows;
  M.single_rows = cut.single_rows;
  M.total_rows = cut.total_rows;
  M.own_records = cut.own_records;
  if (C.cap > 0.f)
    fork_tile_kernel<T, D, Form::kCap><<<dim3(grid), 256, 0, st>>>(M);
  else if (C.slopes)
    fork_tile_kernel<T, D, Form::kBias><<<dim3(grid), 256, 0, st>>>(M);
  else
    fork_tile_kernel<T, D, Form::kPlain><<<dim3(grid), 256, 0, st>>>(M);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  // A round of waves, eight workgroups per CU, with the rows of a token and KV head
  // apart where there is room.
  const long long pairs = (long long)C.tokens * C.hkv, most = 8ll * bch::device_cus();
  long long apart = 4 * most / pairs;
  apart = apart < 1 ? 1 : apart < C.group ? apart : C.group;
  const long long join = (pairs * apart + 3) / 4;
  fork_join_kernel<T, D><<<dim3((unsigned)(join < most ? join : most)), 256, 0, st>>>(M, (int)apart);
  return hipGetLastError();
}

}  // namespace

extern "C" size_t bc_shared_chunk_attention_workspace_size(bc_shape s, int tokens, int group_count) {
  if (!chunk_shape_ok(s, tokens) || group_count < 0 || group_count > s.batch) return 0;
  const size_t apart = bc_chunk_attention_workspace_size(s, tokens), once = fork_cut(s, tokens, group_count).bytes;
  return apart > once ? apart : once;
}

extern "C" int bc_shared_chunk_attention(bc_shape s, bc_chunk_inputs in, const int32_t* groups,
                                         const int32_t* shared, int group_count, void* workspace,
                                         size_t workspace_bytes, bc_stream_t stream) {
  if (!chunk_shape_ok(s, in.tokens) || !chunk_inputs_ok(in) || !groups || group_count < 0 ||
      (group_count > 0 && !shared) || group_count > s.batch)
    return BC_ERROR_INVALID_VALUE;
  const ForkCut cut = fork_cut(s, in.tokens, group_count);
  const bool use = cut.bytes > 0 && bch::sharing_pays(s, in.tokens, in.window) && workspace && aligned16(workspace) &&
                   workspace_bytes >= cut.bytes;
  // As in bc_chunk_attention.  Rows count twice, as a request's and as a group's;
  // under a window, or with documents, a group of few rows is of the wide form.
  const long long rows = (long long)in.tokens * (s.query_heads / s.kv_heads);
  const long long few = in.window > 0 || in.first ? (long long)(kFewRows + 1) * group_count : 0;
  const long long grid = use ? split_grid(s, cut, 2 * rows + few, (long long)s.batch + group_count) : 0;
  const long long far = 1 << 26;
  if (!use || !aligned16(in.q) || !aligned16(in.k) || !aligned16(in.v) || !aligned16(in.output) ||
      stride_bits(in) % 8 != 0 || in.k_strides.slot >= far || in.v_strides.slot >= far || grid > kMostGroups)
    return bc_chunk_attention(s, in, bch::short_window(s, in) ? nullptr : workspace, workspace_bytes, stream);
  if (!in.q || !in.output) return BC_ERROR_INVALID_VALUE;
  MoreParams M{};
  M.t.c = chunk_params(s, in);
  M.groups = groups;
  M.shared = shared;
  M.group_count = group_count;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (in.dtype == BC_FLOAT16)
    return s.dim == 64 ? launch_forks<_Float16, 64>(M, cut, workspace, (unsigned)grid, st)
                       : launch_forks<_Float16, 128>(M, cut, workspace, (unsigned)grid, st);
  return s.dim == 64 ? launch_forks<__bf16, 64>(M, cut, workspace, (unsigned)grid, st)
                     : launch_forks<__bf16, 128>(M, cut, workspace, (unsigned)grid, st);
}
