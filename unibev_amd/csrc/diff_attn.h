// Differential attention: what the host passes to the kernels, and the pieces they share.
//
//   A_m = softmax_j(scale q_m . k_m + mask), m = 1, 2;     out = (D o (A_1 - lam_h A_2)) v;     a row that sees no key gives 0
//
// Rows: the G = H / Hk query heads that share a key / value head are walked as one list of G Nq rows (row r = head r / Nq of
// the group, query r % Nq), so that shared heads read their keys once and their gradients are sums inside one block.
//
// All products run on 32 x 32 MFMA tiles whose output gives a lane ONE item of its own (column lane & 31) and 16 items of
// the staged tile, rows 8 (i >> 2) + 4 (lane >> 5) + (i & 3).  Forward and grad_q: own = rows, staged = keys; grad_k / grad_v:
// own = keys, staged = rows.  The second product of each pair contracts over the staged items, whose order does not
// matter: registers 8 s .. 8 s + 7 of the tile, rounded, ARE its B operand for the 16 staged items of step s (f32: eight
// operands of one), and the A operand is read transposed from the same staged rows (ds_read_b64_tr_b16).  So no score ever
// goes through memory or LDS, and the softmax of a row is arithmetic of its own lane and the one 32 lanes away.
#pragma once
#include <algorithm>
#include <type_traits>

#include "ubv_common.h"

namespace ubv {

struct DiffAttnArgs {
  const void *q, *k, *v, *go;              // [B, N, heads, (2,) D] with element strides below, D contiguous
  int64_t qs[4], ks[4], vs[3], gs[3];      // batch, token, head, map
  const float* lam;                        // [H]
  const uint8_t* kpm;                      // [B, Nk] contiguous, nonzero hides the key; or null
  const void* mask;                        // element strides ms; kind 0: none, 1: bytes (nonzero hides), 2: f32 (added)
  int64_t ms[4];
  int mask_kind, causal;
  int B, H, Hk, G, Nq, Nk, Dh, Dv, R;      // R = G Nq rows of a group
  float scale;                             // > 0
  uint32_t t16;                            // dropout threshold of a 16-bit field, 0: none
  float up;                                // scale of what dropout keeps
  uint64_t seed;
  const uint64_t* seed_dev;
  int n4;                                  // ceil(Nk / 4) field groups per row
  void* out;                               // [B, Nq, H, Dv] contiguous
  float4* stat;                            // [B H Nq] {a_1, l_1, a_2, l_2}: see row_probability
  float* o;                                // [2][B H Nq][Dv] the two maps' normalised products (D's scale included)
  float4* row;                             // [B H Nq] {A_1, A_2, del_1, del_2}, del_m = grad_out . o_m
  float2* rowl;                            // [B H Nq] {l_1, l_2}, with a float mask only
  float* dlrow;                            // [B H Nq] - sum_j A_2 G
  void *gq, *gk, *gv;                      // contiguous gradients
  int work;                                // blocks with work (the grid is rounded up)
  int splits;                              // most blocks that share the staged items of an own tile, 1: none
  int chunk;                               // staged tiles of each of them (fewer in the last)
  int own, n;                              // own items of a block, items of a staged tile
  int halves;                              // forward: blocks that share a row tile's output columns
  float* part;                             // splits > 1: [32 own items][half][split][64 lanes][floats] the blocks' sums
};

constexpr int kAttnSplits = 256;         // most splits of an own tile's staged items

// f16 holds nothing below 2^-24 and loses bits below 2^-14, which the probabilities of a long row reach: they enter the matrix
// instructions 2^8 larger and their products leave 2^8 smaller.  dS enters at its size: a common factor would take from its upper
// range, which a scaled loss uses, what it gives below.
template <typename T> constexpr float kProbShift = std::is_same<T, f16_t>::value ? 8.0f : 0.0f;
template <typename T> constexpr float kProbScale = std::is_same<T, f16_t>::value ? 256.0f : 1.0f;

// a value that is the wave's in every lane: kept in a scalar register
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// What grad_k / grad_v's pass takes lam by on top of that: f16's A_1 - lam A_2 and dS_2 would leave its range beside a |lam| past 255
// though the gradients may not.  A power of two s with (1 + |lam|) 2^8 s below 2^15 for every query head that shares key head hk
// (they are added in one sum); 1 up to 255 and in the other types.
// In two steps, a load that need not be waited for at once (lam_top) and what follows from it.
template <typename T> __device__ __forceinline__ float lam_top(const float* lam, int hk, int G, int lane) {
  float m = 0.0f;
  if constexpr (std::is_same<T, f16_t>::value)
    for (int g = lane; g < G; g += 64) m = fmaxf(m, fabsf(lam[hk * G + g]));
  return m;
}
template <typename T> __device__ __forceinline__ float lam_scale(float m) {
  if constexpr (!std::is_same<T, f16_t>::value) return 1.0f;
  if (!__any(m > 255.0f)) return 1.0f;
#pragma unroll
  for (int w = 32; w >= 1; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
  return uniform(ldexpf(1.0f, 6 - ilogbf(1.0f + fminf(m, 3.0e38f))));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

typedef __attribute__((ext_vector_type(16))) float af32x16_t;
typedef __attribute__((ext_vector_type(4))) uint32_t au32x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t au32x2_t;
typedef __attribute__((ext_vector_type(8))) __bf16 abf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 af16x8_t;
typedef __attribute__((ext_vector_type(4))) short ai16x4_t;

// ---- staged rows in LDS ---------------------------------------------------------------------------------------------------------
// A row of L 16-byte chunks (a power of two) lies unpadded; chunk c of row r is stored at place c ^ fold(r).  fold takes the row bits
// that the bank (4 L r dwords mod 64) does not see, so that the 16 rows which one phase of a 16-byte read touches at one chunk, and
// the 4 rows x 4 chunks which one phase of a transposing read touches, each cover all 64 banks once.  (Rows padded by 16 bytes
// instead: a third of the LDS time was bank conflicts of the transposing reads.)  fold is linear over XOR, and so are addresses:
// a lane's part ^ a constant.
template <int L> __host__ __device__ constexpr int row_fold(int r) {
  return L <= 4 ? (r >> 2) & 3 : L == 8 ? 4 * ((r >> 1) & 1) + ((r >> 2) & 3) : 4 * (r & 3) + ((r >> 2) & 3);
}

// ---- one 16-deep step of a 32 x 32 product: a lane holds items 8 (lane >> 5) + 0 .. 7 of the contraction -------------------
// load<L>: row r0 + (lane & 31) (r0 a multiple of 32) of a tile, elements 16 s .. of the part that begins at chunk `c0`
// load_tr<L>: column 32 d + (lane & 31) of that part, rows k0 + 8 (j >> 2) + 4 (lane >> 5) + (j & 3), j = 0 .. 7 (k0 a multiple of 16)
template <typename T> struct amma {                       // 16-bit types: one MFMA
  static constexpr bool SPLIT = true;                     // what split gives is in two operands
  struct frag { au32x4_t d; };
  static __device__ __forceinline__ af32x16_t mul(const frag& a, const frag& b, af32x16_t c) {
    if constexpr (std::is_same<T, f16_t>::value)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(af16x8_t, a.d), __builtin_bit_cast(af16x8_t, b.d), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf16x8_t, a.d), __builtin_bit_cast(abf16x8_t, b.d), c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag own(const T* t) { return {*reinterpret_cast<const au32x4_t*>(t)}; }
  // probabilities, rounded to the inputs' type: the matrix instruction takes no wider operand.  Half a step of each, random: out and
  // grad_v, which are rounded to the type themselves, are off by 1.1 to 1.4 times that one rounding, by norm over many rows (a row
  // by itself up to 2).  (The rest of each, as for dS, would make that 1.0 and the forward pass 13 to 28 % longer.)
  static __device__ __forceinline__ frag pack(const float* p) {
    frag f;
    if constexpr (std::is_same<T, f16_t>::value) {
      af16x8_t h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (_Float16)p[i];
      f.d = __builtin_bit_cast(au32x4_t, h);
    } else {
      // (the compiler's conversion, not cvt_pk_bf16: beside matrix instructions in flight its wait states are the compiler's to
      //  place, which it does not do around inline assembly)
      abf16x8_t h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (__bf16)p[i];
      f.d = __builtin_bit_cast(au32x4_t, h);
    }
    return f;
  }
  // dS, as the sum of two operands.  Its rows sum to zero, so that errors of one rounding weigh more in grad_q and grad_k than in out
  // (1.45 to 1.55 times the roundings of the results themselves, 1.0 to 1.1 with the rest of each).  bf16 is cut off, not rounded: the
  // upper part is there in f32 without a conversion back.  The second product costs where the VALU is short: 4 heads of 32 / 64,
  // 10 000 x 10 000 bf16, grad_q 290 -> 345 us, grad_k / grad_v 500 -> 575; 2 x 8 heads of 64 / 128, 4096: 373 -> 421, 604 -> 617.
  static __device__ __forceinline__ void split(const float* p, frag& hi, frag& lo) {
    float r[8];
    if constexpr (std::is_same<T, f16_t>::value) {
      hi = pack(p);
      const af16x8_t h = __builtin_bit_cast(af16x8_t, hi.d);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __builtin_fmaf((float)h[i], -1.0f, p[i]);
    } else {
      uint32_t u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { u[i] = __float_as_uint(p[i]); r[i] = p[i] - __uint_as_float(u[i] & 0xffff0000u); }
      hi.d = au32x4_t{__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u),
                      __builtin_amdgcn_perm(u[5], u[4], 0x07060302u), __builtin_amdgcn_perm(u[7], u[6], 0x07060302u)};
    }
    lo = pack(r);
  }
  template <int L> static __device__ __forceinline__ frag load(const char* tile, int r0, int c0, int s, int lane) {
    const int r = lane & 31, base = r * 16 * L + (((lane >> 5) ^ row_fold<L>(r)) << 4);
    return {*reinterpret_cast<const au32x4_t*>(tile + r0 * 16 * L + (base ^ ((c0 + 2 * s) << 4)))};
  }
  template <int L> static __device__ __forceinline__ frag load_tr(const char* tile, int k0, int c0, int d, int lane) {
    typedef __attribute__((address_space(3))) ai16x4_t lds_v4;
    const int rr = (lane & 15) >> 2, r = 4 * (lane >> 5) + rr;
    const int base = r * 16 * L + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ row_fold<L>(r)) << 4) + (lane & 1) * 8;
    const char* t = tile + k0 * 16 * L;
    const ai16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(t + (base ^ ((c0 + 4 * d) << 4))));
    const ai16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(t + 8 * 16 * L + (base ^ (((c0 + 4 * d) ^ row_fold<L>(8)) << 4))));
    const au32x2_t ua = __builtin_bit_cast(au32x2_t, a), ub = __builtin_bit_cast(au32x2_t, b);
    return {au32x4_t{ua.x, ua.y, ub.x, ub.y}};
  }
};
template <> struct amma<float> {                          // f32: eight MFMAs of depth 2 (lane halves), IEEE products
  static constexpr bool SPLIT = false;
  struct frag { float d[8]; };
  static __device__ __forceinline__ af32x16_t mul(const frag& a, const frag& b, af32x16_t c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.d[j], b.d[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag own(const float* t) {
    frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.d[i] = t[i];
    return f;
  }
  static __device__ __forceinline__ frag pack(const float* p) { return own(p); }
  static __device__ __forceinline__ void split(const float* p, frag& hi, frag&) { hi = own(p); }
  template <int L> static __device__ __forceinline__ frag load(const char* tile, int r0, int c0, int s, int lane) {
    const int r = lane & 31, base = r * 16 * L + (((2 * (lane >> 5)) ^ row_fold<L>(r)) << 4);
    const char* t = tile + r0 * 16 * L;
    frag f;
    *reinterpret_cast<float4*>(f.d) = *reinterpret_cast<const float4*>(t + (base ^ ((c0 + 4 * s) << 4)));
    *reinterpret_cast<float4*>(f.d + 4) = *reinterpret_cast<const float4*>(t + (base ^ ((c0 + 4 * s + 1) << 4)));
    return f;
  }
  template <int L> static __device__ __forceinline__ frag load_tr(const char* tile, int k0, int c0, int d, int lane) {
    const int r = 4 * (lane >> 5), base = r * 16 * L + ((((lane & 31) >> 2) ^ row_fold<L>(r)) << 4) + 4 * (lane & 3);
    const char* t = tile + k0 * 16 * L;
    frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int rj = 8 * (j >> 2) + (j & 3);
      f.d[j] = *reinterpret_cast<const float*>(t + rj * 16 * L + (base ^ (((c0 + 8 * d) ^ row_fold<L>(rj)) << 4)));
    }
    return f;
  }
};

__device__ __forceinline__ int tile_item(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

__device__ __forceinline__ float aexp2(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32: 1 ulp, 0 below 2^-126

// v and the value of the lane 32 away, joined
__device__ __forceinline__ float half_max(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// 16 bytes at base + off + soff; 0 from an offset past 2^31 (the buffer descriptor's bound), which kOutside is
constexpr uint32_t kOutside = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t attn_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00027000);
}
__device__ __forceinline__ au32x4_t attn_piece(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff) {
  return __builtin_bit_cast(au32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, soff, 0));
}

// A row's probability of raw score x (q . k, a float mask added over scale), c = scale log2 e.  Without a float mask
// a = log2 of the row's sum (its reference included) and one fma serves.  A float mask may hold the type's lowest value, beside
// which a f32 product loses the score: there the reference a is subtracted first (raw) and l is log2 of the sum.
// A row that sees no key: without a float mask a = +inf, with one a = 0 and l = +inf; both give 0.
__device__ __forceinline__ float row_probability(bool fm, float x, float c, float a, float l) {
  return fm ? aexp2(fmaf(x - a, c, -l)) : aexp2(fmaf(x, c, -a));
}

// what a float mask adds to a raw score: a finite value stays finite (the lowest value alone hides nothing: a row of it is a
// uniform row), -inf hides
__device__ __forceinline__ float mask_raw(float m, float rscale) {
  const float v = m * rscale;
  return m == kNegInf ? kNegInf : v < -3.0e38f ? -3.0e38f : v > 3.0e38f ? 3.0e38f : v;
}
__device__ __forceinline__ float mask_add(float x, float bias) { return bias == kNegInf ? kNegInf : x + bias; }

// 64 bits of the dropout generator from seed's part and a group's number (drop_mix64 of the two)
__device__ __forceinline__ uint64_t attn_seed(uint64_t seed, const uint64_t* dev) {
  return (seed + (dev != nullptr ? *dev : 0)) * 0x9E3779B97F4A7C15ull;
}
__device__ __forceinline__ uint64_t attn_mix(uint64_t z) { return drop_mix64(0, z); }
// field e of a group's bits against the threshold in the upper half of a word
__device__ __forceinline__ bool attn_keep(uint32_t word, int odd, uint32_t t32) { return (odd ? word : word << 16) >= t32; }

}  // namespace ubv
