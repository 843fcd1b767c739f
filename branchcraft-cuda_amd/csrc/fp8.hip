// A paged cache of 8 bits, for gfx950: new tokens' K and V rows rounded as they
// enter it (bc_append_fp8_kv), rows of it back in 16 bits (bc_read_fp8_kv), and
// the attention of new tokens over it (bc_fp8_chunk_attention).
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

// A thread takes 16 values of a head: half a block.
constexpr int kPiece = 16;

// Which piece of the rows of K (0) or V (1) thread x has, and where its slot is;
// false where the slot is outside the pool.
template <int D>
struct Piece {
  int kv, t, h, e;
  int page, in;
  bool inside;
  __device__ __forceinline__ Piece(const Fp8Params& P, long long x) {
    const int per_row = P.hkv * (D / kPiece);
    const long long row = x / per_row;
    const int c = (int)(x - row * per_row);
    kv = blockIdx.y;
    t = (int)row;
    h = c / (D / kPiece);
    e = c % (D / kPiece) * kPiece;
    const int slot = P.slots[t];
    page = slot >> 4;
    in = slot & 15;
    inside = slot >= 0 && page < P.phys_pages;
  }
  __device__ __forceinline__ size_t code(const Fp8Params& P) const {
    return page * P.page[kv] + in * P.slot[kv] + h * P.head[kv] + e;
  }
  __device__ __forceinline__ size_t power(const Fp8Params& P) const {
    return (((size_t)page * P.hkv + h) * BC_PAGE_SIZE + in) * (D / kFp8Block) + e / kFp8Block;
  }
};

// Sixteen values of T at p; VEC: two 16-byte loads.
template <typename T, bool VEC>
__device__ __forceinline__ void load_values(const uint16_t* p, float (&x)[kPiece]) {
#pragma unroll
  for (int i = 0; i < kPiece; i += 8) {
    const uint4 w = load8<VEC>(p + i);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int y = 0; y < 8; ++y)
      x[i + y] = to_float(__builtin_bit_cast(T, (uint16_t)(words[y / 2] >> (16 * (y & 1)))));
  }
}

// grid = (pieces, 2).  The largest magnitude of a block is that of two lanes side
// by side.  Infinities and NaN become the NaN code and have no part in the
// block's power.  Values past 1.875 times the type's largest power of two count as
// that: they would be rounded to the next power, which the type does not have.
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads) void append_fp8_kernel(Fp8Params P) {
  const long long x = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (x >= (long long)P.tokens * P.hkv * (D / kPiece)) return;  // pairs of lanes leave together
  const Piece<D> at(P, x);
  constexpr float kMost = std::is_same<T, _Float16>::value ? 0x1.ep15f : 0x1.ep127f;
  float val[kPiece], top = 0.f;
  load_values<T, VEC>(P.rows[at.kv] + at.t * P.ts[at.kv] + at.h * P.hs[at.kv] + at.e, val);
#pragma unroll
  for (int i = 0; i < kPiece; ++i) {
    const float size = __builtin_fabsf(val[i]);
    const bool finite = size < -kNegInf;
    val[i] = __builtin_copysignf(__builtin_fminf(size, kMost), val[i]);
    top = finite ? __builtin_fmaxf(top, __builtin_fabsf(val[i])) : top;
    val[i] = finite ? val[i] : __builtin_nanf("");
  }
  top = __builtin_fmaxf(top, dpp_f<kDppQuadXor1>(top));
  // Biased: the largest's exponent, one more where its fraction is above that of
  // 448 = 1.75 * 2^8, less 8; and at least 1, so that the power and its inverse
  // are normal numbers.
  const uint32_t power =
      (uint32_t)max((int)((__builtin_bit_cast(uint32_t, top) + 0x1fffffu) >> 23) - 8, 1);
  const float unit = power_of(254 - power);
  uint32_t w[kPiece / 4];
#pragma unroll
  for (int i = 0; i < kPiece / 4; ++i) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(val[4 * i] * unit, val[4 * i + 1] * unit, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(val[4 * i + 2] * unit, val[4 * i + 3] * unit, c, true);
    w[i] = (uint32_t)c;
  }
  if (!at.inside) return;
  *reinterpret_cast<uint4*>(P.pool[at.kv] + at.code(P)) = make_uint4(w[0], w[1], w[2], w[3]);
  if (at.e % kFp8Block == 0) P.scale[at.kv][at.power(P)] = (uint8_t)power;
}

// grid = (pieces, 2).  Rows without a slot are zeros.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void read_fp8_kernel(Fp8Params P) {
  const long long x = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (x >= (long long)P.tokens * P.hkv * (D / kPiece)) return;
  const Piece<D> at(P, x);
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (at.inside) {
    const uint4 w = *reinterpret_cast<const uint4*>(P.pool[at.kv] + at.code(P));
    const float power = power_of(P.scale[at.kv][at.power(P)]);
    lo = make_uint4(values2<T, false>(w.x, power), values2<T, true>(w.x, power),
                    values2<T, false>(w.y, power), values2<T, true>(w.y, power));
    hi = make_uint4(values2<T, false>(w.z, power), values2<T, true>(w.z, power),
                    values2<T, false>(w.w, power), values2<T, true>(w.w, power));
  }
  uint4* const out = reinterpret_cast<uint4*>(P.out[at.kv] + x * kPiece);
  out[0] = lo;
  out[1] = hi;
}

// Codes go by 16 bytes.
bool pool_ok(const bc_shape& s, const bc_fp8_pool& p) {
  if (!p.k || !p.v || !p.k_scale || !p.v_scale || s.physical_pages < 1 || s.kv_heads < 1 ||
      s.kv_heads > BC_MAX_CHUNK_HEADS || (s.dim != 64 && s.dim != 128) || !aligned16(p.k) || !aligned16(p.v))
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
  return dim3((unsigned)((pieces + kThreads - 1) / kThreads), 2);
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

extern "C" size_t bc_fp8_chunk_attention_workspace_size(bc_shape s, int tokens) {
  return chunk_shape_ok(s, tokens) ? cut_of(s, tokens).bytes : 0;
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
  ChunkParams P = chunk_params(s, in);
  P.k_scale = k_scale;
  P.v_scale = v_scale;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // As in bc_chunk_attention.
  const Cut cut = cut_of(s, in.tokens);
  const bool use = cut.bytes > 0 && workspace && aligned16(workspace) && workspace_bytes >= cut.bytes;
  const long long grid = tile_grid(s, in.tokens, cut, use);
  const long long far = 1 << 27;  // bytes: offsets inside a page are 32-bit
  const bool tiled = aligned16(in.q) && aligned16(in.output) &&
                     (in.q_strides.token | in.q_strides.head) % 8 == 0 && in.k_strides.slot < far &&
                     in.v_strides.slot < far && (long long)in.tokens * P.group <= 1 << 30 &&
                     grid <= kMostGroups;
  void* const ws = use ? workspace : nullptr;
  if (tiled) return launch_tiles<true>(P, s.dim, in.dtype, cut, ws, grid, st);
  return launch_rows<true>(P, s.dim, in.dtype, st);
}
