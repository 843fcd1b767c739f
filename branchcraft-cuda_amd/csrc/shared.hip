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

// W waves per workgroup, each with 32 rows of a tile, and the steps of K and V that
// LDS holds: those on their way, the one at hand, and, where half the waves lag by
// half a step, the one before it.
//  - D = 128, W = 8: one workgroup per CU, for groups of more than 128 rows, which so
//    read each page once per 256.  What is read once comes from HBM, some 2 us away
//    under load.
//  - D = 128, W = 4: two per CU.  D = 64: three, since the softmax of three waves per
//    SIMD is the bound there, not memory.
template <int D, int W>
struct Plan {
  static constexpr bool kLag = W == 8;
  static constexpr int kBuffers = kLag ? 4 : D == 64 ? 3 : 2;
  static constexpr int kAhead = kLag ? 2 : kBuffers - 1;
  static constexpr int kPerCu = kLag ? 1 : D == 64 ? 3 : 2;
  static constexpr bool kRounds = kPerCu == 1;
};

// ---------------------------------------------------------------------------
// The plan

// threadIdx.x, found anew: what is computed from it belongs to the item at hand, and
// does not take registers through the others.
__device__ __forceinline__ int own_thread() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

// Group g: its members and the tokens they share, none of fewer than two members.
struct Group {
  int g0, g1, shared;
};

__device__ __forceinline__ Group group_at(const ChunkParams& P, int g) {
  const int from = P.groups[g], to = P.groups[g + 1], tokens = P.shared[g];  // in one round
  Group x;
  x.g0 = min(max(from, 0), P.batch);
  x.g1 = min(max(to, 0), P.batch);
  x.shared = x.g1 - x.g0 > 1 ? min(max(tokens, 0), P.max_pages * BC_PAGE_SIZE) : 0;
  return x;
}

// The groups i .. i + 63, a lane each; behind the last, groups of no request.
__device__ __forceinline__ Group groups_from(const ChunkParams& P, int i) {
  const int lane = threadIdx.x & 63;
  const Group x = group_at(P, min(i + lane, P.group_count - 1));
  return i + lane < P.group_count ? x : Group{0x7fffffff, 0, 0};
}

// Of the 64 groups that the lanes hold, that of request b, a lane's own; -1, and 0
// tokens, where it has none.  All lanes of the wave take part.
__device__ __forceinline__ int group_in(const Group& x, int b, int& shared) {
  const int n = count_upto(x.g0, b) - 1, from = max(n, 0);
  const int end = __shfl(x.g1, from, 64), tokens = __shfl(x.shared, from, 64);
  shared = n >= 0 && b < end ? tokens : 0;
  return n;
}

// The group of request b, a lane's own, of the first 64 (`head`) or those behind.
__device__ __forceinline__ int group_of(const ChunkParams& P, const Group& head, int b, int& shared) {
  int at = group_in(head, b, shared);
  for (int i = 64; i < P.group_count; i += 64) {
    int tokens;
    const int n = group_in(groups_from(P, i), b, tokens);
    if (n >= 0) {
      at = i + n;
      shared = tokens;
    }
  }
  return at;
}

// The entries of a batch in blocks of 64, one per lane: the requests' blocks, then
// the groups'.  The first two of the requests and the first of the groups stay, and
// all that these do not depend on each other for is loaded in one round.
template <int W>
struct Entries {
  int lane, own_blocks, blocks;
  Group head;  // a lane's of the first 64 groups
  AskedEntry own0, own1, groups0;

  __device__ __forceinline__ explicit Entries(const ChunkParams& C) : lane(own_thread() & 63), own1{} {
    own_blocks = (C.batch + 63) / 64;
    blocks = own_blocks + (C.group_count + 63) / 64;
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
      ask_work<32 * W>(C, a, floor, true);
    }
    return a;
  }
  __device__ __forceinline__ AskedEntry group(const ChunkParams& C, const Group& m, int g) const {
    AskedEntry a{};
    // Where the lanes hold all requests, the ends of its rows are theirs.
    int from = __shfl(own0.start, m.g0, 64), to = __shfl(own0.start + own0.n, m.g1 - 1, 64);
    const bool is = g < C.group_count && m.shared > 0;
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
      a.tiles = wide ? (a.rows + 32 * W - 1) / (32 * W) : 0;
      a.steps = wide ? wide_steps(C, a.len, 32 * W) : 0;
      a.narrow = !wide && a.rows > 0 ? (a.len + 31) / 32 : 0;
    }
    return a;
  }
};

// How the batch is cut, see Cutting: a tile of the narrow form takes each of its
// waves about kTileTime times as long as a step of the wide one takes its
// workgroup.  What the narrow entries leave of a round of workgroups is filled with
// shares.
constexpr float kTileTime = 1.8f;
constexpr int kLeastTiles = 2;  // fewest per wave

template <int W>
__device__ __forceinline__ Cutting cut_entries(const TileParams& P, const Entries<W>& all) {
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
  const float run = ((float)c.narrow + W / kTileTime * work) / (float)P.waves;
  c.run = max(min((int)__builtin_fminf(run, 1e9f) + 1, c.narrow), (c.narrow + P.waves - 1) / P.waves);
  c.run = max(c.run, kLeastTiles);
  c.groups = ((c.narrow + c.run - 1) / c.run * C.hkv + W - 1) / W;
  // n tiles have less than work / share + n parts: one more than a round holds
  // would take the time of a second round.
  const int left = max(P.target - c.groups, P.target / 4) / C.hkv - lanes_sum(tiles);
  const float share = work / (float)max(left, P.target / (2 * C.hkv) + 1);
  c.share = max(kLeastSteps, (int)__builtin_fminf(share, 1e9f) + 1);
  return c;
}

// Item `idx` of the wide entries' tiles and their parts, see plan_item.
template <int W>
__device__ __forceinline__ Item plan_entry(const TileParams& P, const Entries<W>& all, int share, long long idx) {
  const ChunkParams& C = P.c;
  const int lane = own_thread() & 63;
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
// Tiles of rows

// The wide form, with more rows per workgroup and more steps on their way than
// wide_body has: 32 W rows, and kBuffers steps of K and V in LDS, of which one is
// worked on while others are filled.  One barrier a step, before which each wave
// waits for its own loads of the next step only.
template <typename T, int D, Form FORM, int W>
__device__ __forceinline__ void deep_body(const TileParams& A, Args args, const Item& it, int kvh,
                                          uint16_t* s_kv, int* s_ids, Seen* s_seen, int* s_bad) {
  const ChunkParams& C = A.c;
  const Request& rq = it.r;
  typedef Plan<D, W> L;
  constexpr int BUFFERS = L::kBuffers, AHEAD = L::kAhead, THREADS = 64 * W;
  constexpr int KS = D / 16, CPR = D / 8;
  constexpr int NX = kStep * CPR / THREADS;   // chunks per thread and step, of K and of V each
  constexpr int HALF = kStep * D;             // halves of a step's K, then as many of V
  constexpr int WINDOW = THREADS / 4;         // steps whose page ids LDS holds
  const int tid = own_thread(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, lr = lane & 31;
  const int tile0 = it.tile * (32 * W), row0 = tile0 + wave * 32;
  const int32_t* const table = C.pages + (size_t)rq.b * C.max_pages;
  Rows<D> R;
  u32x4 qB[KS];
  Seen mine, wg;
  int t0, tend;
  auto range = [&] {  // this part's steps of those that the workgroup's rows see
    const int first = wg.any_lo / kStep;
    const int steps = wg.any_hi >= wg.any_lo ? wg.any_hi / kStep - first + 1 : 0;
    t0 = first + (int)((long long)steps * it.part / it.parts);
    tend = first + (int)((long long)steps * (it.part + 1) / it.parts);
  };

  const int lrow = tid / CPR, lcol = 8 * (tid % CPR ^ swz<D>(lrow));
  const unsigned koff = (unsigned)(((lrow % BC_PAGE_SIZE) * C.ks + lcol) * 2);
  const unsigned voff = (unsigned)(((lrow % BC_PAGE_SIZE) * C.vs + lcol) * 2);
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)s_kv + wave * 1024);
  Pages<false> pg;
  unsigned pages = 0;  // in the pool, four bits for each step from the one at hand on
  // The pages of step u and the 15 behind it, a lane each, from the window that LDS
  // holds; all waves come here for the same u.
  auto take = [&](int u) {
    if ((u - t0) % WINDOW == 0) {
      __syncthreads();
      s_ids[tid] = table[min(u * 4 + tid, C.max_pages - 1)];
      __syncthreads();
    }
    pg.take(C, kvh, s_ids[(u - t0) % WINDOW * 4 + lane]);
  };
  auto issue_chunk = [&](int x, int at, int buf) {
    const int from = 4 * at + (x * (THREADS / CPR) + wave * (64 / CPR)) / BC_PAGE_SIZE;
    const unsigned dst = lds0 + buf * (4 * HALF) + x * (THREADS * 16);
    load2_to_lds(Pages<false>::at(pg.k, from), Pages<false>::at(pg.v, from), koff, voff, dst, dst + 2 * HALF);
  };
  auto issue = [&](int u) {  // step t0 + u of the first ones
    if (t0 + u >= tend) return;
    if (u == 0) take(t0);
#pragma unroll
    for (int x = 0; x < NX; ++x) issue_chunk(x, u, u);
    pages |= ((unsigned)(pg.in_pool >> (4 * u)) & 15u) << (4 * u);
  };
  auto issue_first = [&] {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) issue(u);
  };
  // Where the rows' places do not matter to what is read, the first steps go out
  // ahead of them: a group's rows see all that it shares.
  const bool ahead = !C.first && (is_group(rq) ? C.window == 0 : true);
  if (tid < 4) s_bad[tid] = 0;
  if (ahead) {
    wg = is_group(rq) ? Seen{0, rq.len - 1, 0, 0} : rows_seen(C, rq, tile0, min(tile0 + 32 * W, rq.rows));
    range();
    issue_first();
  }
  load_rows<T, D, FORM, true>(C, rq, row0 + lr, kvh, g, R, qB);
  mine = wave_seen(R, row0 + lr < rq.rows);
  if (lane == 0) s_seen[wave] = mine;
  __syncthreads();
  wg = s_seen[0];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    wg.any_lo = min(wg.any_lo, s_seen[w].any_lo);
    wg.any_hi = max(wg.any_hi, s_seen[w].any_hi);
    wg.all_lo = max(wg.all_lo, s_seen[w].all_lo);
    wg.all_hi = min(wg.all_hi, s_seen[w].all_hi);
  }
  wg.any_lo = __builtin_amdgcn_readfirstlane(wg.any_lo);
  wg.any_hi = __builtin_amdgcn_readfirstlane(wg.any_hi);
  wg.all_lo = __builtin_amdgcn_readfirstlane(wg.all_lo);
  wg.all_hi = __builtin_amdgcn_readfirstlane(wg.all_hi);
  if (!ahead) {
    range();
    issue_first();
  }
  // Steps whole_lo .. whole_hi - 1 are seen whole by every row, given their pages.
  const int whole_lo = wg.all_lo / kStep + (wg.all_lo % kStep != 0);
  const int whole_hi = (min(wg.all_hi, rq.len - 1) + 1) / kStep;
  auto is_whole = [&](int t) { return (pages & 15u) == 15u && t >= whole_lo && t < whole_hi; };
  // Each thread tidies the chunks that its own loads, already waited for,
  // have filled.
  auto inspect = [&](int t, int buf) {
    const unsigned long long ok = tokens_of<4>(rq.len - t * kStep, pages & 15u);
    uint16_t* const v = s_kv + buf * (2 * HALF) + HALF;
    bool bad = false;
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      u32x4* const at = reinterpret_cast<u32x4*>(v + (tid + THREADS * x) * 8);
      bad |= tidy<T>(at, (ok >> (lrow + THREADS / CPR * x)) & 1u);
    }
    return bad;
  };
  // Until the loads of a step are there, of which those of `behind` more steps may
  // be on their way.
  auto wait_step = [&](int behind) {
    if (AHEAD > 1 && behind > 0)
      wait_to<2 * NX>();
    else
      wait_loads();
  };

  const Offsets<D> o = read_offsets<D>(lane);
  const float scale2 = scale2_of(C, FORM);
  f32x16 sc[2];
  // Of the step at hand: its buffer, and what was taken out of it.
  int buf = 0;
  bool bad = false;
  wait_rows(qB);
  if (t0 < tend) {
    wait_step(min(tend - 1 - t0, AHEAD - 1));
    if (!is_whole(t0)) bad = inspect(t0, 0);
    bad = __builtin_amdgcn_readfirstlane(__syncthreads_or(bad));
  }
  auto scores = [&](int t, Edges& e) {
    const uint16_t* const kt = s_kv + buf * (2 * HALF);
    const int u = t + AHEAD, at = (u - t0) % 16;
    const int to = buf + AHEAD < BUFFERS ? buf + AHEAD : buf + AHEAD - BUFFERS;
    const bool next = u < tend;
    if (next && at == 0) take(u);
    u32x4 kf[2][KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) kf[i][s] = lds16(kt + i * 32 * D + o.k[s]);
    const f32x16 zero = {};
    if (FORM == Form::kBias) start_scores<D, 2>(C, sc, R, t * kStep, g);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        sc[i] = Num<T>::mfma(kf[i][s], qB[s], FORM != Form::kBias && s == 0 ? zero : sc[i]);
      if (s % 2 == 1 && s / 2 < NX) {
        if (next) issue_chunk(s / 2, at, to);
      }
    }
    e = Edges{t * kStep < mine.all_lo, t * kStep + kStep - 1 > mine.all_hi, (pages & 15u) != 15u, 0};
    if (e.pages) e.valid = tokens_of<4>(rq.len - t * kStep, pages & 15u);
    if (next) pages |= ((unsigned)(pg.in_pool >> (4 * at)) & 15u) << (4 * AHEAD);
  };
  auto product = [&](int t, const Edges& e, int of, bool untidy) {
    finish_scores<D, FORM, 2>(C, sc, R, t * kStep, g, e);
    constexpr bool kAhead = D == 128 && FORM != Form::kCap;  // as in wide_body
    if (kAhead) __builtin_amdgcn_s_setprio(2);
    weigh<T, D, 2>(sc, R, s_kv + of * (2 * HALF) + HALF, o, scale2);
    if (kAhead) __builtin_amdgcn_s_setprio(0);
    if (untidy) add_untidy<T, D, false>(C, rq, kvh, R, t * kStep, kStep, g);
  };
  auto end_step = [&](int t) {
    pages >>= 4;
    buf = buf + 1 < BUFFERS ? buf + 1 : 0;
    // Step s of the part sets flag s % 4 before the barrier that ends the step
    // before it; the flag is read behind that barrier and cleared behind the
    // next, two barriers before it is set again.
    const int s = t - t0;
    const bool look = t + 1 < tend && !is_whole(t + 1);
    if (t + 1 < tend) {
      wait_step(min(tend - 2 - t, AHEAD - 1));
      if (look && inspect(t + 1, buf)) s_bad[(s + 1) & 3] = 1;
    }
    __syncthreads();
    if (bad && tid == 0) s_bad[s & 3] = 0;
    bad = look && __builtin_amdgcn_readfirstlane(s_bad[(s + 1) & 3]);
  };
  if (!L::kLag || wave < W / 2) {
#pragma unroll 1
    for (int t = t0; t < tend; ++t) {
      Edges e;
      scores(t, e);
      product(t, e, buf, bad);
      end_step(t);
    }
  } else if (t0 < tend) {
    // The other half of a SIMD's waves: a step's product behind the barrier that ends
    // the step, so that it runs beside the scores of the first half, and the reverse.
    Edges e;
    scores(t0, e);
    bool untidy = bad;
    end_step(t0);
#pragma unroll 1
    for (int t = t0 + 1; t < tend; ++t) {
      product(t - 1, e, buf > 0 ? buf - 1 : BUFFERS - 1, untidy);
      scores(t, e);
      untidy = bad;
      end_step(t);
    }
    product(tend - 1, e, buf > 0 ? buf - 1 : BUFFERS - 1, untidy);
  }

  const TileParams& P = reread(args);
  R.l += shfl_xor_f(R.l, 32);
  const int r = row0 + lr;
  if (it.parts > 1 || joined(rq)) {
    const int first = it.parts > 1 ? P.narrow_rows + (it.slot + it.part) * P.part_rows : single_row(P, rq) + tile0;
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
  const float inv = one_over(R.l);
  if (r < rq.rows) {
    uint16_t* const out = out_row<T, D>(P.c, rq, r, kvh) + 4 * g;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int jq = 0; jq < 4; ++jq)
        *reinterpret_cast<uint2*>(out + 32 * dt + 8 * jq) =
            make_uint2(pack2<T>(R.acc[dt][4 * jq] * inv, R.acc[dt][4 * jq + 1] * inv),
                       pack2<T>(R.acc[dt][4 * jq + 2] * inv, R.acc[dt][4 * jq + 3] * inv));
  }
}

template <typename T, int D, Form FORM, int W>
__global__ __launch_bounds__(64 * W, D == 64 ? 3 : 2) void fork_tile_kernel(TileParams) {
  constexpr int kWide = Plan<D, W>::kBuffers * 2 * kStep * D, kFlat = W * 64 * D;
  __shared__ __attribute__((aligned(256))) uint16_t s_kv[kWide > kFlat ? kWide : kFlat];
  __shared__ int s_ids[64 * W];
  __shared__ Seen s_seen[W];
  __shared__ int s_bad[4];
  const Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  // Where a workgroup fills a CU, a round of them is launched, and each takes its
  // share of what is more: those without work, which see that in 4 us, would start
  // behind the others' end.  It finds its next item anew, so that the plan's registers
  // do not live through an item.
  for (int round = 0;; ++round) {
    const TileParams& P = reread(args);
    asm volatile("" ::"s"(P.c.groups), "s"(P.c.shared), "s"(P.c.group_count));
    pin_plan(P);
    const Entries<W> all(P.c);
    const Cutting cut = cut_entries<W>(P, all);
    // The narrow entries first, as in chunk_tile_kernel.
    if ((int)blockIdx.x < cut.groups) {
      const TileParams& A = reread(args);
      pin_rows<false>(A);
      auto ask = [&](int b0) { return all.at(A.c, b0 / 64); };
      flat_body<T, D, FORM, false, true, W>(A, all.own0, 64 * all.blocks, ask, cut, s_kv);
      return;
    }
    const int wide = gridDim.x - cut.groups;
    const long long idx = blockIdx.x - cut.groups + (long long)round * wide, at = idx / P.c.hkv;
    const int kvh = (int)(idx - at * P.c.hkv);
    const Item it = plan_entry<W>(P, all, cut.share, at);
    if (!it.found) {
      const long long items = Plan<D, W>::kRounds ? 0 : it.items * P.c.hkv;
      clear_rows<D, 64 * W>(P.c, blockIdx.x - cut.groups - items, wide - items);
      return;
    }
    if (it.part == 0 && kvh == 0 && threadIdx.x == 0)
      put_fork_record(P, it.r, it.tile, it.parts,
                      it.parts > 1 ? P.narrow_rows + it.slot * P.part_rows
                                   : single_row(P, it.r) + it.tile * P.part_rows,
                      P.part_rows);
    const TileParams& A = reread(args);
    pin_rows<false>(A);
    deep_body<T, D, FORM, W>(A, args, it, kvh, s_kv, s_ids, s_seen, s_bad);
    if (!Plan<D, W>::kRounds) return;
    __syncthreads();
  }
}

// The join with groups: `apart` waves share the rows of a new token and KV head; of
// a wave, each group of D / 4 lanes takes the parts of the request's own tokens and
// then of its group's in turn.  Rows that their entry has written as output are
// left.
template <typename T, int D>
__global__ __launch_bounds__(256) void fork_join_kernel(TileParams P, int apart) {
  constexpr int LPR = D / 4, GW = 64 / LPR;
  const ChunkParams& C = P.c;
  const int lane = threadIdx.x & 63, grp = lane / LPR, c = lane % LPR;
  const long long total = (long long)C.tokens * C.hkv * apart, step = 4ll * gridDim.x;
  for (long long x = 4ll * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); x < total; x += step) {
    const long long pair = x / apart;
    const int sub = (int)(x - pair * apart), t = (int)(pair / C.hkv), kvh = (int)(pair - (long long)t * C.hkv);
    // The request of token t, the first of its rows, and its group, of loads in one
    // round for up to 64 of either.
    const Group head = groups_from(C, 0);
    int b = 0, own0 = 0;
    for (int i = 0; i < C.batch; i += 64) {
      const int from = C.starts[min(i + lane, C.batch - 1)], to = C.starts[min(i + lane, C.batch - 1) + 1];
      const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i + lane < C.batch && to <= t));
      b += n;
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
    const int all0 = shared > 0 ? start_of(C.starts[group_at(C, g).g0]) : 0;
    for (int r = sub; r < C.group; r += apart) {
      int parts[2] = {}, first[2] = {}, stride[2] = {};
      auto look = [&](int i, int entry, int from) {
        if (t < from) return;
        const int row = (t - from) * C.group + r, tile = row / P.part_rows;
        const int4 rec = P.records[record_of(P, entry, from, tile)];
        // Where starts decrease, a record may be another's or no one's.
        const long long last = rec.y + (long long)max(rec.x - 1, 0) * rec.z + row - tile * P.part_rows;
        const bool sane = rec.x > 0 && rec.x <= 2 * (P.waves + P.most_parts) && rec.y >= 0 && rec.z > 0 &&
                          last < P.total_rows;
        parts[i] = sane ? rec.x : 0;
        first[i] = rec.y + row - tile * P.part_rows;
        stride[i] = rec.z;
      };
      look(0, b, own0);
      if (shared > 0)
        look(1, C.batch + g, all0);
      else if (parts[0] < 2)
        continue;
      float m = kNegInf, l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int p = grp; p < parts[0] + parts[1]; p += GW) {
        const bool own = p < parts[0];
        const int at = own ? first[0] + p * stride[0] : first[1] + (p - parts[0]) * stride[1];
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

// ---------------------------------------------------------------------------
// The call

struct ForkCut : Cut {
  int single_rows, total_rows, own_records;
};

// Waves per workgroup, see Plan.
int waves_of(const bc_shape& s, int tokens, int groups) {
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  return s.dim == 128 && rows > 128ll * groups ? 8 : 4;
}

// How a call cuts its work; bytes 0: every request reads its own pages.
ForkCut fork_cut(const bc_shape& s, int tokens, int groups) {
  ForkCut c{};
  const long long rows = (long long)tokens * (s.query_heads / s.kv_heads);
  if (groups < 1 || s.batch < 2 || rows < 1 || rows > 1 << 28 ||
      (s.batch + (long long)groups) * (s.max_pages + 1ll) > 1 << 28 ||
      (long long)s.batch * s.query_heads > 1 << 26)
    return c;
  const int W = waves_of(s, tokens, groups);
  c.target = (W == 8 ? Plan<128, 8>::kPerCu : s.dim == 128 ? Plan<128, 4>::kPerCu : Plan<64, 4>::kPerCu) *
             bch::device_cus();  // workgroups in a round
  c.waves = W * c.target / s.kv_heads > 1 ? W * c.target / s.kv_heads : 1;
  const long long own = rows < 32ll * s.batch ? rows : 32ll * s.batch;
  const long long of_groups = rows < 32ll * groups ? rows : 32ll * groups;
  const long long narrow = 32ll * c.waves + own + of_groups;
  c.most_parts = 2 * c.target / s.kv_heads;
  c.part_rows = 32 * W;
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

template <typename T, int D, int W>
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
    fork_tile_kernel<T, D, Form::kCap, W><<<dim3(grid), 64 * W, 0, st>>>(P);
  else if (C.slopes)
    fork_tile_kernel<T, D, Form::kBias, W><<<dim3(grid), 64 * W, 0, st>>>(P);
  else
    fork_tile_kernel<T, D, Form::kPlain, W><<<dim3(grid), 64 * W, 0, st>>>(P);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  // A round of waves, eight workgroups per CU, with the rows of a token and KV head
  // apart where there is room.
  const long long pairs = (long long)C.tokens * C.hkv, most = 8ll * bch::device_cus();
  long long apart = 4 * most / pairs;
  apart = apart < 1 ? 1 : apart < C.group ? apart : C.group;
  const long long join = (pairs * apart + 3) / 4;
  fork_join_kernel<T, D><<<dim3((unsigned)(join < most ? join : most)), 256, 0, st>>>(P, (int)apart);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_forks(const ChunkParams& C, int dim, int W, const ForkCut& cut, void* ws, unsigned grid,
                        hipStream_t st) {
  return dim == 64 ? launch_forks<T, 64, 4>(C, cut, ws, grid, st)
         : W == 4  ? launch_forks<T, 128, 4>(C, cut, ws, grid, st)
                   : launch_forks<T, 128, 8>(C, cut, ws, grid, st);
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
  const int W = waves_of(s, in.tokens, group_count);
  const long long bound = split_grid(s, cut, 2 * rows + few, (long long)s.batch + group_count, W);
  const long long grid = W == 8 && bound > cut.target ? cut.target : bound, far = 1 << 26;
  if (!use || !aligned16(in.q) || !aligned16(in.k) || !aligned16(in.v) || !aligned16(in.output) ||
      stride_bits(in) % 8 != 0 || in.k_strides.slot >= far || in.v_strides.slot >= far || grid > kMostGroups)
    return bc_chunk_attention(s, in, nullptr, 0, stream);
  if (!in.q || !in.output) return BC_ERROR_INVALID_VALUE;
  ChunkParams P = chunk_params(s, in);
  P.groups = groups;
  P.shared = shared;
  P.group_count = group_count;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return in.dtype == BC_FLOAT16 ? launch_forks<_Float16>(P, s.dim, W, cut, workspace, (unsigned)grid, st)
                                : launch_forks<__bf16>(P, s.dim, W, cut, workspace, (unsigned)grid, st);
}
