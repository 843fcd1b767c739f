// A paged cache of 8 bits, for gfx950: new tokens' K and V rows rounded as they
// enter it (bc_append_fp8_kv), rows of it back in 16 bits (bc_read_fp8_kv), and
// the attention of new tokens over it (bc_fp8_chunk_attention); its pages copied
// (bc_copy_fp8_pages).
//
// Every 32 values of one head of one token share a power of two, 2^e: the least
// with which they stay within 448, the largest e4m3 value.  A value is its code
// times that.  A power of two costs a code with an exponent of its own no
// precision, it makes the rounding one exact product and one conversion, and the
// values are exact in BF16 (and in FP16, if the rows were FP16), so that the
// attention converts two codes and applies their power in one instruction.
//
// No reference counterpart: the reference's cache is FP16.
#include "bc_tiles.h"

namespace {

struct Fp8Params {
  const uint16_t* rows[2];   // K's and V's
  uint8_t* pool[2];
  uint8_t* scale[2];         // [P][Hkv][16][D / 32]
  uint16_t* out[2];
  const int32_t* slots;
  long long ts[2], hs[2];               // rows' token and head strides
  long long page[2], slot[2], head[2];  // pools'
  int tokens, phys_pages, hkv;
};

// A thread takes eight values of a head, of K and of V: a block is four lanes, a
// head of D values D / 8.
constexpr int kPiece = 8;

// Which piece of the rows thread x has, and where its slot is; `inside`: the slot
// is one of the pool's.
template <int D>
struct Piece {
  unsigned t;
  int h, e, page, in;
  bool inside;
  __device__ __forceinline__ Piece(const Fp8Params& P, unsigned x) {
    const unsigned piece = x % (D / kPiece), head = x / (D / kPiece);
    t = head / (unsigned)P.hkv;
    h = head - t * P.hkv;
    e = piece * kPiece;
    const int slot = P.slots[t];
    page = slot >> 4;
    in = slot & 15;
    inside = slot >= 0 && page < P.phys_pages;
  }
  __device__ __forceinline__ size_t code(const Fp8Params& P, int kv) const {
    return page * P.page[kv] + in * P.slot[kv] + h * P.head[kv] + e;
  }
  __device__ __forceinline__ size_t powers(const Fp8Params& P) const {  // the head's first
    return (((size_t)page * P.hkv + h) * BC_PAGE_SIZE + in) * (D / kFp8Block);
  }
};

// Eight values of T as codes, and their block's power.
template <typename T>
__device__ __forceinline__ uint2 codes_of(const uint4& w, uint32_t& power) {
  constexpr float kMost = std::is_same<T, _Float16>::value ? 0x1.ep15f : 0x1.ep127f;
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  float val[kPiece], top = 0.f;
#pragma unroll
  for (int i = 0; i < kPiece; ++i) {
    const float x = to_float(__builtin_bit_cast(T, (uint16_t)(words[i / 2] >> (16 * (i & 1)))));
    const float size = __builtin_fminf(__builtin_fabsf(x), kMost);
    const bool finite = __builtin_fabsf(x) < -kNegInf;
    top = finite ? __builtin_fmaxf(top, size) : top;
    val[i] = finite ? __builtin_copysignf(size, x) : __builtin_nanf("");
  }
  top = __builtin_fmaxf(top, dpp_f<kDppQuadXor1>(top));
  top = __builtin_fmaxf(top, dpp_f<kDppQuadXor2>(top));
  // Biased: the largest's exponent, one more where its fraction is above that of
  // 448 = 1.75 * 2^8, less 8; and at least 1, so that the power and its inverse
  // are normal numbers.
  power = (uint32_t)max((int)((__builtin_bit_cast(uint32_t, top) + 0x1fffffu) >> 23) - 8, 1);
  const float unit = power_of(254 - power);
  uint32_t code[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(val[4 * i] * unit, val[4 * i + 1] * unit, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(val[4 * i + 2] * unit, val[4 * i + 3] * unit, c, true);
    code[i] = (uint32_t)c;
  }
  return make_uint2(code[0], code[1]);
}

// A head's powers from its blocks' lanes, four apart, to its first lane.
template <int D>
__device__ __forceinline__ uint32_t gather_powers(uint32_t power) {
  uint32_t all = power | (uint32_t)dpp_i<0x104>((int)power) << 8;  // row_shl 4
  if (D == 128)
    all |= (uint32_t)dpp_i<0x108>((int)power) << 16 | (uint32_t)dpp_i<0x10c>((int)power) << 24;
  return all;
}

template <int D>
using Powers = typename std::conditional<D == 128, uint32_t, uint16_t>::type;

// The largest magnitude of a block is that of four lanes.  Infinities and NaN become
// the NaN code and have no part in the block's power.  Values past 1.875 times the
// type's largest power of two count as that: they would be rounded to the next
// power, which the type does not have.
// Memory-bound: 8192 fused rows (8 heads of 128, FP16; 51 MB moved) 12.2 us, 4.2
// TB/s, rows of 2 KB out of 12 KB; 64 rows 3.2, the launch.  Eight values a thread
// are one load of 16 bytes; with sixteen, and K and V in different workgroups, storing
// and reading these rows back took 23.4 us in place of 21.6.
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads) void append_fp8_kernel(Fp8Params P) {
  const unsigned x = blockIdx.x * kThreads + threadIdx.x;
  if (x >= (unsigned)P.tokens * P.hkv * (D / kPiece)) return;  // the lanes of a head together
  const Piece<D> at(P, x);
  uint4 w[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    w[kv] = load8<VEC>(P.rows[kv] + at.t * P.ts[kv] + at.h * P.hs[kv] + at.e);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t power;
    const uint2 codes = codes_of<T>(w[kv], power);
    const uint32_t all = gather_powers<D>(power);
    if (!at.inside) continue;
    *reinterpret_cast<uint2*>(P.pool[kv] + at.code(P, kv)) = codes;
    if (at.e == 0) *reinterpret_cast<Powers<D>*>(P.scale[kv] + at.powers(P)) = (Powers<D>)all;
  }
}

// Rows without a slot are zeros.  Memory-bound: 32768 rows (8 heads of 128, BF16; 204
// MB) 34 us, 6.0 TB/s (a large copy 5.3), 36 with stores through the caches; 8192 rows
// 9.9, 5.1 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void read_fp8_kernel(Fp8Params P) {
  const unsigned x = blockIdx.x * kThreads + threadIdx.x;
  if (x >= (unsigned)P.tokens * P.hkv * (D / kPiece)) return;
  const Piece<D> at(P, x);
  uint2 codes[2] = {};
  float power[2] = {};
  if (at.inside)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[kv] = *reinterpret_cast<const uint2*>(P.pool[kv] + at.code(P, kv));
      power[kv] = power_of(P.scale[kv][at.powers(P) + at.e / kFp8Block]);
    }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    __builtin_nontemporal_store(
        u32x4{values2<T, false>(codes[kv].x, power[kv]), values2<T, true>(codes[kv].x, power[kv]),
              values2<T, false>(codes[kv].y, power[kv]), values2<T, true>(codes[kv].y, power[kv])},
        reinterpret_cast<u32x4*>(P.out[kv] + (size_t)x * kPiece));
}

// Pages src[i] to pages dst[i]: grid = (pairs, slices), a slice being kCopyPieces
// pieces of 16 codes of K and of V each, or of four powers, which follow the codes.
// A call of one page (8 heads of 128) 4.3 us, its launch; 32 5.1; 1000 (68 MB moved)
// 10.4, 6.5 TB/s, through the caches.
constexpr int kCopyPieces = 2 * kThreads;

__global__ __launch_bounds__(kThreads) void copy_fp8_pages_kernel(Fp8Params P, const int32_t* __restrict__ src,
                                                                  int codes, int powers, int per_head) {
  const int from = src[blockIdx.x], to = P.slots[blockIdx.x];
  if (from < 0 || from >= P.phys_pages || to < 0 || to >= P.phys_pages || from == to) return;
  const int lo = blockIdx.y * kCopyPieces, hi = min(lo + kCopyPieces, codes + powers);
  for (int x = lo + (int)threadIdx.x; x < hi; x += kThreads) {
    if (x < codes) {
      const int row = x / per_head, e = 16 * (x - row * per_head), slot = row / P.hkv, h = row - slot * P.hkv;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint8_t* const at = P.pool[kv] + slot * P.slot[kv] + h * P.head[kv] + e;
        *reinterpret_cast<uint4*>(at + to * P.page[kv]) = *reinterpret_cast<const uint4*>(at + from * P.page[kv]);
      }
    } else {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint32_t* const at = reinterpret_cast<uint32_t*>(P.scale[kv]) + (x - codes);
        at[(size_t)to * powers] = at[(size_t)from * powers];
      }
    }
  }
}

// Codes go by eight and 16 bytes, powers by two and four.
bool pool_ok(const bc_shape& s, const bc_fp8_pool& p) {
  if (!p.k || !p.v || !p.k_scale || !p.v_scale || s.physical_pages < 1 || s.kv_heads < 1 ||
      s.kv_heads > BC_MAX_CHUNK_HEADS || (s.dim != 64 && s.dim != 128) || !aligned16(p.k) || !aligned16(p.v) ||
      (reinterpret_cast<uintptr_t>(p.k_scale) | reinterpret_cast<uintptr_t>(p.v_scale)) % 4 != 0)
    return false;
  const long long bits = p.k_strides.page | p.k_strides.slot | p.k_strides.head | p.v_strides.page |
                         p.v_strides.slot | p.v_strides.head;
  return bits >= 0 && bits % 16 == 0;
}

Fp8Params fp8_params(const bc_shape& s, const bc_fp8_pool& p, const int32_t* slots) {
  Fp8Params P{};
  P.pool[0] = p.k;
  P.pool[1] = p.v;
  P.scale[0] = p.k_scale;
  P.scale[1] = p.v_scale;
  P.slots = slots;
  const bc_pool_strides* const strides[] = {&p.k_strides, &p.v_strides};
  for (int i = 0; i < 2; ++i) {
    P.page[i] = strides[i]->page;
    P.slot[i] = strides[i]->slot;
    P.head[i] = strides[i]->head;
  }
  P.phys_pages = s.physical_pages;
  P.hkv = s.kv_heads;
  return P;
}

// Launches for at most this many rows each, so that none has 2^24 workgroups.
int most_rows(const bc_shape& s) {
  return (int)((long long)kMostGroups * kThreads / (s.kv_heads * (s.dim / kPiece)));
}

dim3 pieces_grid(const bc_shape& s, int tokens) {
  const long long pieces = (long long)tokens * s.kv_heads * (s.dim / kPiece);
  return dim3((unsigned)((pieces + kThreads - 1) / kThreads));
}

template <typename T, bool VEC>
void launch_append(const bc_shape& s, const Fp8Params& P, hipStream_t st) {
  const dim3 grid = pieces_grid(s, P.tokens);
  if (s.dim == 64)
    append_fp8_kernel<T, 64, VEC><<<grid, kThreads, 0, st>>>(P);
  else
    append_fp8_kernel<T, 128, VEC><<<grid, kThreads, 0, st>>>(P);
}

template <typename T>
void launch_read(const bc_shape& s, const Fp8Params& P, hipStream_t st) {
  const dim3 grid = pieces_grid(s, P.tokens);
  if (s.dim == 64)
    read_fp8_kernel<T, 64><<<grid, kThreads, 0, st>>>(P);
  else
    read_fp8_kernel<T, 128><<<grid, kThreads, 0, st>>>(P);
}

}  // namespace

extern "C" int bc_append_fp8_kv(bc_shape s, const bc_half* k, const bc_half* v, bc_row_strides ks,
                                bc_row_strides vs, int dtype, bc_fp8_pool pool, const int32_t* slots,
                                int tokens, bc_stream_t stream) {
  const long long bits = ks.token | ks.head | vs.token | vs.head;
  if (!pool_ok(s, pool) || !k || !v || !slots || tokens < 0 || bits < 0 ||
      (dtype != BC_FLOAT16 && dtype != BC_BFLOAT16))
    return BC_ERROR_INVALID_VALUE;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool vec = aligned16(k) && aligned16(v) && bits % 8 == 0;
  Fp8Params P = fp8_params(s, pool, slots);
  P.ts[0] = ks.token;
  P.ts[1] = vs.token;
  P.hs[0] = ks.head;
  P.hs[1] = vs.head;
  const int most = most_rows(s);
  for (long long t0 = 0; t0 < tokens; t0 += most) {
    P.rows[0] = k + t0 * ks.token;
    P.rows[1] = v + t0 * vs.token;
    P.slots = slots + t0;
    P.tokens = (int)(tokens - t0 < most ? tokens - t0 : most);
    if (dtype == BC_FLOAT16)
      vec ? launch_append<_Float16, true>(s, P, st) : launch_append<_Float16, false>(s, P, st);
    else
      vec ? launch_append<__bf16, true>(s, P, st) : launch_append<__bf16, false>(s, P, st);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return BC_SUCCESS;
}

extern "C" int bc_read_fp8_kv(bc_shape s, bc_fp8_pool pool, const int32_t* slots, int tokens,
                              int dtype, bc_half* k, bc_half* v, bc_stream_t stream) {
  if (!pool_ok(s, pool) || tokens < 0 || (tokens > 0 && (!slots || !k || !v)) || !aligned16(k) ||
      !aligned16(v) || (dtype != BC_FLOAT16 && dtype != BC_BFLOAT16))
    return BC_ERROR_INVALID_VALUE;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  Fp8Params P = fp8_params(s, pool, slots);
  const int most = most_rows(s);
  for (long long t0 = 0; t0 < tokens; t0 += most) {
    P.out[0] = k + t0 * s.kv_heads * s.dim;
    P.out[1] = v + t0 * s.kv_heads * s.dim;
    P.slots = slots + t0;
    P.tokens = (int)(tokens - t0 < most ? tokens - t0 : most);
    dtype == BC_FLOAT16 ? launch_read<_Float16>(s, P, st) : launch_read<__bf16>(s, P, st);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return BC_SUCCESS;
}

extern "C" int bc_copy_fp8_pages(bc_shape s, bc_fp8_pool pool, const int32_t* src_pages,
                                 const int32_t* dst_pages, int count, bc_stream_t stream) {
  if (!pool_ok(s, pool) || count < 0 || (count > 0 && (!src_pages || !dst_pages))) return BC_ERROR_INVALID_VALUE;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int codes = s.kv_heads * s.dim, powers = BC_PAGE_SIZE * s.kv_heads * s.dim / (4 * kFp8Block);
  const int slices = (codes + powers + kCopyPieces - 1) / kCopyPieces, most = kMostGroups / slices;
  for (long long i = 0; i < count; i += most) {
    const Fp8Params P = fp8_params(s, pool, dst_pages + i);
    const int n = (int)(count - i < most ? count - i : most);
    copy_fp8_pages_kernel<<<dim3(n, slices), kThreads, 0, st>>>(P, src_pages + i, codes, powers, s.dim / 16);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return BC_SUCCESS;
}

extern "C" size_t bc_fp8_chunk_attention_workspace_size(bc_shape s, int tokens) {
  return chunk_shape_ok(s, tokens) ? cut_of(s, tokens, true).bytes : 0;
}

extern "C" int bc_fp8_chunk_attention(bc_shape s, bc_chunk_inputs in, const uint8_t* k_scale,
                                      const uint8_t* v_scale, void* workspace,
                                      size_t workspace_bytes, bc_stream_t stream) {
  if (!chunk_shape_ok(s, in.tokens) || !chunk_inputs_ok(in) || !k_scale || !v_scale)
    return BC_ERROR_INVALID_VALUE;
  const long long pool_bits = in.k_strides.page | in.k_strides.slot | in.k_strides.head |
                              in.v_strides.page | in.v_strides.slot | in.v_strides.head;
  // Powers are read four at a time (two at D = 64).
  const uintptr_t scales = reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale);
  if (!aligned16(in.k) || !aligned16(in.v) || pool_bits % 16 != 0 || scales % 4 != 0)
    return BC_ERROR_INVALID_VALUE;
  if (in.tokens == 0) return BC_SUCCESS;
  if (!in.q || !in.output) return BC_ERROR_INVALID_VALUE;
  MoreParams M{};
  M.t.c = chunk_params(s, in);
  M.k_scale = k_scale;
  M.v_scale = v_scale;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // As in bc_chunk_attention, which cuts tables also under a short window.
  const Cut cut = cut_of(s, in.tokens, true);
  const bool use = cut.bytes > 0 && workspace && aligned16(workspace) && workspace_bytes >= cut.bytes &&
                   !bch::short_window(s, in);
  const long long rows = (long long)in.tokens * M.t.c.group;
  const long long grid = use ? split_grid(s, cut, rows, s.batch) : tile_grid(s, in.tokens, cut, false);
  const long long far = 1 << 27;  // bytes: offsets inside a page are 32-bit
  const bool tiled = aligned16(in.q) && aligned16(in.output) &&
                     (in.q_strides.token | in.q_strides.head) % 8 == 0 && in.k_strides.slot < far &&
                     in.v_strides.slot < far && rows <= 1 << 30 &&
                     grid <= kMostGroups;
  void* const ws = use ? workspace : nullptr;
  if (tiled) return launch_tiles<true>(M, s.dim, in.dtype, cut, ws, grid, st);
  return launch_rows<true>(M, s.dim, in.dtype, st);
}
