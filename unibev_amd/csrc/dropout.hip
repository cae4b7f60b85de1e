// Dropout from a counter-based generator, with or without the residual:  y = identity + D o x,  D = keep / (1 - t / 2^16).
//
// The mask is a function of (seed, element index) and is never stored: the backward pass is the same kernel over grad_y.
// One 64-bit mix serves the four elements of a group (drop_mix64): element i is kept where the 16-bit field i % 4 of group
// i / 4 is at least t = round(p 2^16).  The scale uses t, not p, so that E[D] = 1 holds exactly at this resolution; p = 1 is
// t = 2^16 (nothing kept, scale 0).
//
// Bound by memory: 6 bytes per 16-bit element with the residual against ~11 VALU slots of hash.  A thread takes 8 elements a
// step, 16-byte accesses; buffers that start off a 16-byte border take the same kernel with element-aligned accesses.
// 41 M bf16 elements with the residual 45 to 47 us (5.2 to 5.5 TB/s), without it 27 to 28 us (5.9 to 6.0 TB/s, part of it cached);
// below ~1 M elements the launch is what it takes (2.6 to 2.8 us).
#include "ubv_common.h"

namespace ubv {

typedef __attribute__((ext_vector_type(4))) uint32_t du32x4_t;

// 8 consecutive elements as f32; ALN: p is 16-byte aligned
template <typename T, bool ALN> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  constexpr int W = 8 * elem<T>::kBytes / 16, PER = 16 / elem<T>::kBytes;
  T t[8];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if constexpr (ALN) *reinterpret_cast<du32x4_t*>(t + w * PER) = *reinterpret_cast<const du32x4_t*>(p + w * PER);
    else __builtin_memcpy(t + w * PER, p + w * PER, 16);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = elem<T>::to_float(t[i]);
}
template <typename T, bool ALN> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  constexpr int W = 8 * elem<T>::kBytes / 16, PER = 16 / elem<T>::kBytes;
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = elem<T>::from_float(v[i]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if constexpr (ALN) *reinterpret_cast<du32x4_t*>(p + w * PER) = *reinterpret_cast<const du32x4_t*>(t + w * PER);
    else __builtin_memcpy(p + w * PER, t + w * PER, 16);
  }
}

// TX: type of x; TY: type of identity and y
template <typename TX, typename TY, bool RES, bool ALN>
__global__ __launch_bounds__(256) void dropout_kernel(const TX* x, const TY* identity, TY* y, long n, uint32_t t16,
                                                      float scale, uint64_t seed, const uint64_t* __restrict__ seed_dev) {
  if (seed_dev != nullptr) seed += *seed_dev;   // per-step base kept on the device (graph replays)
  const long stride = (long)gridDim.x * 256 * 8;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += stride) {
    const uint64_t mix[2] = {drop_mix64(seed, (uint64_t)i >> 2), drop_mix64(seed, ((uint64_t)i >> 2) + 1)};
    if (i + 8 <= n) {
      float v[8], r[8];
      load8<TX, ALN>(x + i, v);
      if constexpr (RES) load8<TY, ALN>(identity + i, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool keep = (uint32_t)((mix[e >> 2] >> (16 * (e & 3))) & 0xffffull) >= t16;
        const float d = keep ? v[e] * scale : 0.0f;
        v[e] = RES ? r[e] + d : d;
      }
      store8<TY, ALN>(y + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e) {
        if (i + e < n) {
          const bool keep = (uint32_t)((mix[e >> 2] >> (16 * (e & 3))) & 0xffffull) >= t16;
          const float d = keep ? elem<TX>::to_float(x[i + e]) * scale : 0.0f;
          y[i + e] = elem<TY>::from_float(RES ? elem<TY>::to_float(identity[i + e]) + d : d);
        }
      }
    }
  }
}

template <typename TX, typename TY>
static void dropout_launch(const void* x, const void* identity, void* y, long n, uint32_t t16, float scale, uint64_t seed,
                           const uint64_t* seed_dev, hipStream_t st) {
  const long units = (n + 7) / 8;
  const dim3 grid((unsigned)min((units + 255) / 256, 16384L));
  const bool aln = (((uintptr_t)x | (uintptr_t)y | (uintptr_t)identity) % 16) == 0;
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, (const TX*)x, (const TY*)identity, (TY*)y, n, t16, scale, seed, seed_dev);
  };
  if (identity != nullptr) {
    if (aln) run(dropout_kernel<TX, TY, true, true>); else run(dropout_kernel<TX, TY, true, false>);
  } else {
    if (aln) run(dropout_kernel<TX, TY, false, true>); else run(dropout_kernel<TX, TY, false, false>);
  }
}

}  // namespace ubv

extern "C" int ubv_dropout(const void* x, const void* identity, void* y, int64_t n, float p, uint64_t seed,
                           const uint64_t* seed_dev, int x_dtype, int y_dtype, void* stream) {
  using namespace ubv;
  UBV_CHECK_ARG(n >= 0 && (n == 0 || (x && y)), "dropout: bad arguments");
  UBV_CHECK_ARG(x_dtype >= 0 && x_dtype <= 2 && y_dtype >= 0 && y_dtype <= 2, "dropout: unknown dtype %d / %d", x_dtype, y_dtype);
  UBV_CHECK_ARG(x_dtype == y_dtype || x_dtype == UBV_F32 || y_dtype == UBV_F32, "dropout: x and y of two 16-bit types");
  UBV_CHECK_ARG(p >= 0.0f && p <= 1.0f, "dropout: p = %g must be in [0, 1]", (double)p);
  if (n == 0) return UBV_OK;
  uint32_t t16; float sc;
  drop_params16(p, t16, sc);
  hipStream_t st = as_stream(stream);
#define UBV_DROP(TX, TY) dropout_launch<TX, TY>(x, identity, y, (long)n, t16, sc, seed, seed_dev, st)
  switch (x_dtype * 3 + y_dtype) {
    case UBV_F32 * 3 + UBV_F32: UBV_DROP(float, float); break;
    case UBV_F16 * 3 + UBV_F16: UBV_DROP(f16_t, f16_t); break;
    case UBV_BF16 * 3 + UBV_BF16: UBV_DROP(bf16_t, bf16_t); break;
    case UBV_F16 * 3 + UBV_F32: UBV_DROP(f16_t, float); break;
    case UBV_BF16 * 3 + UBV_F32: UBV_DROP(bf16_t, float); break;
    case UBV_F32 * 3 + UBV_F16: UBV_DROP(float, f16_t); break;
    default: UBV_DROP(float, bf16_t); break;
  }
#undef UBV_DROP
  UBV_CHECK_LAUNCH("dropout");
  return UBV_OK;
}
