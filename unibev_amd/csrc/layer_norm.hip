// Layer norm over the last axis, forward and backward, any width:
//
//   y = (x - mean) rstd gamma + beta;     h = (x - mean) rstd,  u = grad_y gamma
//   grad_x = rstd (u - mean_C(u) - h mean_C(u h));   grad_gamma = sum_rows grad_y h;   grad_beta = sum_rows grad_y
//
// Bound by memory: x in, y out forward; x and grad_y in, grad_x out backward.  A row lives in the registers of TPR threads
// (K 16-byte pieces each) between its one load and its one store, with the variance taken around the mean in a second pass
// over those registers; a row of a few pieces shares its wave with others (TPR < 64), a row of more than 256 pieces takes a
// block.  Rows whose width is no multiple of a 16-byte piece start at any element border: the same kernels with
// element-aligned accesses (one instruction too) and a last piece that overlaps the one before.  Rows wider than 8192 elements
// are streamed (ln_plan).  80 000 x 256 f32: forward 27 to 31 us (5.3 to 6.0 TB/s),
// backward 42 (5.9 TB/s) + 4, bf16: 15 (5.3), 22 (5.6) + 4; 5001 x 1021 f16: 7.1, 12.4 + 4.9, bf16: 7.0, 12.6 + 4.9.
//
// The weight's gradient: a thread owns the same columns of every row that its block visits and keeps their sums in f32
// registers; the block's threads are added through LDS, the blocks' sums [block][2][C] go to a workspace and are added in
// fixed order by a second small launch: the same bits on every run.
#include <type_traits>

#include "ubv_common.h"

namespace ubv {

typedef __attribute__((ext_vector_type(4))) uint32_t lu32x4_t;

// rows that start at 16-byte borders and are whole pieces | of at least one piece | narrower than a piece
constexpr int kLnAligned = 0, kLnAny = 1, kLnNarrow = 2;

// Where the piece of VEC elements that begins at column c is taken from: the last one of a row that is no whole number of pieces
// is moved back to end with the row, and one past the row's end is that piece again; ln_in: the elements that are the piece's own.
// Both holders of an element compute and store the same value.  (A scalar tail, whose loads wait for one another: 5001 x 1021 f16
// forward 9.2 us, 7.3 so; backward 19.8, 13.1.)
template <int VEC> __device__ __forceinline__ int ln_place(int c, int C) { return max(0, min(c, C - VEC)); }
template <int AL> __device__ __forceinline__ bool ln_in(int c, int at, int i, int C) { return AL == kLnAligned ? c < C : at + i >= c && at + i < C; }

// the piece at `at` (ln_place); a row narrower than a piece repeats its last element
template <typename T, int AL>
__device__ __forceinline__ void ln_load(const T* p, int at, int C, float (&v)[16 / elem<T>::kBytes]) {
  constexpr int VEC = 16 / elem<T>::kBytes;
  T t[VEC];
  if constexpr (AL == kLnAligned) *reinterpret_cast<lu32x4_t*>(t) = *reinterpret_cast<const lu32x4_t*>(p + at);
  else if constexpr (AL == kLnAny) __builtin_memcpy(t, p + at, 16);
  else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = p[min(i, C - 1)];
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = elem<T>::to_float(t[i]);
}
template <typename T, int AL>
__device__ __forceinline__ void ln_store(T* p, int at, int C, const float (&v)[16 / elem<T>::kBytes]) {
  constexpr int VEC = 16 / elem<T>::kBytes;
  T t[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) t[i] = elem<T>::from_float(v[i]);
  if constexpr (AL == kLnAligned) *reinterpret_cast<lu32x4_t*>(p + at) = *reinterpret_cast<const lu32x4_t*>(t);
  else if constexpr (AL == kLnAny) __builtin_memcpy(p + at, t, 16);
  else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < C) p[i] = t[i];
  }
}
// VEC f32 weights (gamma or beta; any alignment), `fill` where there are none
template <int AL, int VEC>
__device__ __forceinline__ void ln_weight(const float* w, int at, int C, float fill, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = fill;
  if (w == nullptr) return;
  if constexpr (AL != kLnNarrow) __builtin_memcpy(v, w + at, 4 * VEC);
  else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = w[min(i, C - 1)];
  }
}

// sums of a and b over the TPR threads of a row, handed to all of them
template <int TPR>
__device__ __forceinline__ void ln_sum2(float& a, float& b, float (*red)[2]) {
#pragma unroll
  for (int m = (TPR < 64 ? TPR : 64) >> 1; m >= 1; m >>= 1) { a += __shfl_xor(a, m, 64); b += __shfl_xor(b, m, 64); }
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __syncthreads();                                 // (the row before may still be read)
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6][0] = a; red[threadIdx.x >> 6][1] = b; }
    __syncthreads();
    a = 0.0f; b = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) { a += red[w][0]; b += red[w][1]; }
  }
}

// the same for one sum
template <int TPR> __device__ __forceinline__ void ln_sum(float& a, float (*red)[2]) {
#pragma unroll
  for (int m = (TPR < 64 ? TPR : 64) >> 1; m >= 1; m >>= 1) a += __shfl_xor(a, m, 64);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = a;
    __syncthreads();
    a = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) a += red[w][0];
  }
}

constexpr int ln_block(int tpr) { return tpr < 256 ? 256 : tpr; }

template <typename T, int AL, int TPR, int K>
__global__ __launch_bounds__(ln_block(TPR)) void layer_norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                     const float* __restrict__ beta, T* __restrict__ y,
                                                                     float* __restrict__ mean, float* __restrict__ rstd, long R,
                                                                     int C, float eps) {
  constexpr int VEC = 16 / elem<T>::kBytes, ROWS = ln_block(TPR) / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1][2];
  const int sub = threadIdx.x / TPR, tc = (threadIdx.x % TPR) * VEC;
  const float inv = 1.0f / (float)C;
  constexpr bool HOLD = K * VEC <= 16;                         // weights held for all the block's rows, else read for each
  float gh[HOLD ? K : 1][VEC], bh[HOLD ? K : 1][VEC];
  if constexpr (HOLD) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = ln_place<VEC>(tc + k * TPR * VEC, C);
      ln_weight<AL, VEC>(gamma, at, C, 1.0f, gh[k]);
      ln_weight<AL, VEC>(beta, at, C, 0.0f, bh[k]);
    }
  }
  for (long r0 = (long)blockIdx.x * ROWS; r0 < R; r0 += (long)gridDim.x * ROWS) {
    const long r = r0 + sub;
    const bool ok = r < R;
    const T* xr = x + (ok ? r : R - 1) * C;
    float v[K][VEC], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = tc + k * TPR * VEC, at = ln_place<VEC>(c, C);
      ln_load<T, AL>(xr, at, C, v[k]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += ln_in<AL>(c, at, i, C) ? v[k][i] : 0.0f;
    }
    ln_sum<TPR>(sum, red);
    const float mu = sum * inv;
    float var = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = tc + k * TPR * VEC, at = ln_place<VEC>(c, C);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[k][i] -= mu;
        const float d = ln_in<AL>(c, at, i, C) ? v[k][i] : 0.0f;
        var = fmaf(d, d, var);
      }
    }
    ln_sum<TPR>(var, red);
    const float rs = 1.0f / sqrtf(var * inv + eps);
    if (ok) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = tc + k * TPR * VEC, at = ln_place<VEC>(c, C);
        if (c < C) {
          float o[VEC];
          float (&g)[VEC] = gh[HOLD ? k : 0], (&b)[VEC] = bh[HOLD ? k : 0];
          if constexpr (!HOLD) {
            ln_weight<AL, VEC>(gamma, at, C, 1.0f, g);
            ln_weight<AL, VEC>(beta, at, C, 0.0f, b);
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = fmaf(v[k][i] * rs, g[i], b[i]);
          ln_store<T, AL>(y + r * C, at, C, o);
        }
      }
      if (threadIdx.x % TPR == 0 && mean != nullptr) { mean[r] = mu; rstd[r] = rs; }
    }
  }
}

template <typename T, int AL, int TPR, int K>
__global__ __launch_bounds__(ln_block(TPR)) void layer_norm_bwd_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                                                                     const float* __restrict__ gamma,
                                                                     const float* __restrict__ mean,
                                                                     const float* __restrict__ rstd, T* __restrict__ gx,
                                                                     float* __restrict__ part, long R, int C) {
  constexpr int VEC = 16 / elem<T>::kBytes, BLK = ln_block(TPR), ROWS = BLK / TPR;
  constexpr int GW = TPR < 64 ? TPR : 64;                      // threads of one wave that hold different columns
  __shared__ float red[TPR > 64 ? TPR / 64 : 1][2];
  __shared__ float cols[TPR > 64 ? 1 : 3][TPR > 64 ? 1 : GW * VEC * K];
  const int sub = threadIdx.x / TPR, tc = (threadIdx.x % TPR) * VEC;
  const float inv = 1.0f / (float)C;
  constexpr bool HOLD = K * VEC <= 16;
  float ag[K][VEC], ab[K][VEC], gh[HOLD ? K : 1][VEC];
  if constexpr (HOLD) {
#pragma unroll
    for (int k = 0; k < K; ++k) ln_weight<AL, VEC>(gamma, ln_place<VEC>(tc + k * TPR * VEC, C), C, 1.0f, gh[k]);
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) { ag[k][i] = 0.0f; ab[k][i] = 0.0f; }
  for (long r0 = (long)blockIdx.x * ROWS; r0 < R; r0 += (long)gridDim.x * ROWS) {
    const long r = r0 + sub;
    const bool ok = r < R;
    const long rr = ok ? r : R - 1;
    const float mu = mean[rr], rs = rstd[rr];
    float h[K][VEC], u[K][VEC], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = tc + k * TPR * VEC, at = ln_place<VEC>(c, C);
      float (&g)[VEC] = gh[HOLD ? k : 0];
      ln_load<T, AL>(x + rr * C, at, C, h[k]);
      ln_load<T, AL>(gy + rr * C, at, C, u[k]);
      if constexpr (!HOLD) ln_weight<AL, VEC>(gamma, at, C, 1.0f, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const bool in = ok && ln_in<AL>(c, at, i, C);
        h[k][i] = (h[k][i] - mu) * rs;
        const float hi = in ? h[k][i] : 0.0f, go = in ? u[k][i] : 0.0f;
        u[k][i] *= g[i];
        ag[k][i] = fmaf(go, hi, ag[k][i]);
        ab[k][i] += go;
        const float ui = in ? u[k][i] : 0.0f;
        s1 += ui;
        s2 = fmaf(ui, hi, s2);
      }
    }
    ln_sum2<TPR>(s1, s2, red);
    s1 *= inv; s2 *= inv;
    if (ok && gx != nullptr) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = tc + k * TPR * VEC;
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = rs * (u[k][i] - s1 - h[k][i] * s2);
        if (c < C) ln_store<T, AL>(gx + r * C, ln_place<VEC>(c, C), C, o);
      }
    }
  }
  if (part == nullptr) return;
  float* out = part + (long)blockIdx.x * 2 * C;
  if constexpr (TPR > 64) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = tc + k * TPR * VEC, at = ln_place<VEC>(c, C);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (ln_in<AL>(c, at, i, C)) { out[at + i] = ag[k][i]; out[C + at + i] = ab[k][i]; }
    }
  } else {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float (&a)[K][VEC] = half == 0 ? ag : ab;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
#pragma unroll
          for (int m = 32; m >= TPR; m >>= 1) a[k][i] += __shfl_xor(a[k][i], m, 64);
          if (wv > 0 && lane < GW) cols[wv - 1][(k * GW + lane) * VEC + i] = a[k][i];
        }
      __syncthreads();
      if (wv == 0 && lane < GW) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = tc + k * TPR * VEC, at = ln_place<VEC>(c, C);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int o = (k * GW + lane) * VEC + i;
            if (ln_in<AL>(c, at, i, C)) out[half * C + at + i] = ((a[k][i] + cols[0][o]) + cols[1][o]) + cols[2][o];
          }
        }
      }
      __syncthreads();
    }
  }
}

// ---- rows too wide for a block's registers: a block walks a row, which it reads again for each pass (from L2) --------------
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_wide_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta, T* __restrict__ y,
                                                                  float* __restrict__ mean, float* __restrict__ rstd, long R, int C,
                                                                  float eps) {
  constexpr int VEC = 16 / elem<T>::kBytes;
  __shared__ float red[16][2];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    const T* xr = x + r * C;
    T* yr = y + r * C;
    float sum = 0.0f, var = 0.0f, v[VEC];
    for (int c = threadIdx.x * VEC; c < C; c += 1024 * VEC) {
      const int at = ln_place<VEC>(c, C);
      ln_load<T, kLnAny>(xr, at, C, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += at + i >= c ? v[i] : 0.0f;
    }
    ln_sum<1024>(sum, red);
    const float mu = sum / (float)C;
    for (int c = threadIdx.x * VEC; c < C; c += 1024 * VEC) {
      const int at = ln_place<VEC>(c, C);
      ln_load<T, kLnAny>(xr, at, C, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) { const float d = at + i >= c ? v[i] - mu : 0.0f; var = fmaf(d, d, var); }
    }
    ln_sum<1024>(var, red);
    const float rs = 1.0f / sqrtf(var / (float)C + eps);
    for (int c = threadIdx.x * VEC; c < C; c += 1024 * VEC) {
      const int at = ln_place<VEC>(c, C);
      float g[VEC], b[VEC];
      ln_load<T, kLnAny>(xr, at, C, v);
      ln_weight<kLnAny, VEC>(gamma, at, C, 1.0f, g);
      ln_weight<kLnAny, VEC>(beta, at, C, 0.0f, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mu) * rs, g[i], b[i]);
      ln_store<T, kLnAny>(yr, at, C, v);
    }
    if (threadIdx.x == 0 && mean != nullptr) { mean[r] = mu; rstd[r] = rs; }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_wide_bwd_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                                                                  const float* __restrict__ gamma, const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, T* __restrict__ gx, long R, int C) {
  constexpr int VEC = 16 / elem<T>::kBytes;
  __shared__ float red[16][2];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    const long base = r * C;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.0f, s2 = 0.0f, v[VEC], go[VEC], g[VEC];
    for (int c = threadIdx.x * VEC; c < C; c += 1024 * VEC) {
      const int at = ln_place<VEC>(c, C);
      ln_load<T, kLnAny>(x + base, at, C, v);
      ln_load<T, kLnAny>(gy + base, at, C, go);
      ln_weight<kLnAny, VEC>(gamma, at, C, 1.0f, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float u = at + i >= c ? go[i] * g[i] : 0.0f;
        s1 += u;
        s2 = fmaf(u, (v[i] - mu) * rs, s2);
      }
    }
    ln_sum2<1024>(s1, s2, red);
    s1 /= (float)C; s2 /= (float)C;
    for (int c = threadIdx.x * VEC; c < C; c += 1024 * VEC) {
      const int at = ln_place<VEC>(c, C);
      ln_load<T, kLnAny>(x + base, at, C, v);
      ln_load<T, kLnAny>(gy + base, at, C, go);
      ln_weight<kLnAny, VEC>(gamma, at, C, 1.0f, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = rs * (go[i] * g[i] - s1 - (v[i] - mu) * rs * s2);
      ln_store<T, kLnAny>(gx + base, at, C, v);
    }
  }
}

// column sums of such rows: blockIdx.x = 256 columns, blockIdx.y = a slab of rows
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_wide_cols_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                  float* __restrict__ part, long R, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float ag = 0.0f, ab = 0.0f;
  for (long r = blockIdx.y; r < R; r += gridDim.y) {
    const float go = elem<T>::to_float(gy[r * C + c]);
    ag = fmaf(go, (elem<T>::to_float(x[r * C + c]) - mean[r]) * rstd[r], ag);
    ab += go;
  }
  part[((long)blockIdx.y * 2) * C + c] = ag;
  part[((long)blockIdx.y * 2 + 1) * C + c] = ab;
}

// out[t] = sum over the blocks' rows in fixed order, t < 2 C: 16 columns x 64 groups of rows per block (626 x 2042: 4.8 us; 16
// groups and 1024 x 2042: 7.5)
__global__ __launch_bounds__(1024) void layer_norm_cols_final_kernel(const float* __restrict__ part, int nrows, int C,
                                                                    float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int t = blockIdx.x * 16 + cl;
  const int per = (nrows + 63) / 64;
  float sum = 0.0f;
  if (t < 2 * C) {
    const int r1 = min(nrows, (rg + 1) * per);
#pragma unroll 8
    for (int r = rg * per; r < r1; ++r) sum += part[(long)r * 2 * C + t];
  }
  red[rg][cl] = sum;
  __syncthreads();
  if (rg == 0 && t < 2 * C) {
    float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < 64; ++g) q[g >> 4] += red[g][cl];
    const float tot = (q[0] + q[1]) + (q[2] + q[3]);
    if (t < C) { if (dgamma != nullptr) dgamma[t] = tot; }
    else if (dbeta != nullptr) dbeta[t - C] = tot;
  }
}

constexpr int kLnBwdBlocks = 1024;      // most blocks of a backward launch = rows of the workspace
constexpr int kLnWideSlabs = 64;        // the same where rows are streamed
constexpr int kLnHeld = 8192;           // widest row that ln_plan holds in registers, of every type

// f(TPR, K) for a row of C elements of 16 / VEC bytes; false: stream the row
template <int VEC, typename F>
static bool ln_plan(int C, F&& f) {
  if (C > kLnHeld) return false;
  const long n = ((long)C + VEC - 1) / VEC;
#define UBV_LN(TPR, K) (f(std::integral_constant<int, TPR>{}, std::integral_constant<int, K>{}), true)
  if (n <= 4) return UBV_LN(4, 1);
  if (n <= 8) return UBV_LN(8, 1);
  if (n <= 16) return UBV_LN(16, 1);
  if (n <= 32) return UBV_LN(32, 1);
  if (n <= 64) return UBV_LN(64, 1);
  if (n <= 128) return UBV_LN(64, 2);
  if (n <= 256) return UBV_LN(64, 4);
  if (n <= 512) return UBV_LN(256, 2);
  if (n <= 1024) return UBV_LN(256, 4);
  // f32 up to kLnHeld.  16-bit rows of as many pieces are wider than that and streamed: 1024 threads have 128 registers each, which
  // the backward kernel's x, grad_y and sums of 2 x 8 elements pass by 16 to 37.  2000 x 10 000 f16, us, streamed / held: forward
  // 25 / 30, backward 57 / 159 (300 x 9001 bf16: 7.7 / 8.9, 31 / 50; only very many rows gain, 20 000 x 16 384: 395 / 298, 842 / 774).
  if constexpr (VEC == 4) {
    if (n <= 2048) return UBV_LN(1024, 2);
  }
#undef UBV_LN
  return false;
}

template <typename T>
static void ln_fwd(const void* xv, const float* gamma, const float* beta, void* yv, float* mean, float* rstd, long R, int C,
                   float eps, hipStream_t st) {
  constexpr int VEC = 16 / elem<T>::kBytes;
  const T* x = (const T*)xv;
  T* y = (T*)yv;
  const bool aln = C % VEC == 0 && ((uintptr_t)xv | (uintptr_t)yv) % 16 == 0;
  const bool held = ln_plan<VEC>(C, [&](auto tpr, auto k) {
    constexpr int TPR = decltype(tpr)::value, K = decltype(k)::value, ROWS = ln_block(TPR) / TPR;
    const dim3 grid((unsigned)min((R + ROWS - 1) / ROWS, 4096L)), blk(ln_block(TPR));
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, blk, 0, st, x, gamma, beta, y, mean, rstd, R, C, eps); };
    if (aln) return run(layer_norm_fwd_kernel<T, kLnAligned, TPR, K>);
    if constexpr (TPR == 4)
      if (C < VEC) return run(layer_norm_fwd_kernel<T, kLnNarrow, TPR, K>);
    run(layer_norm_fwd_kernel<T, kLnAny, TPR, K>);
  });
  if (!held)
    hipLaunchKernelGGL(layer_norm_wide_fwd_kernel<T>, dim3((unsigned)min(R, 4096L)), dim3(1024), 0, st, x, gamma, beta, y, mean, rstd, R, C, eps);
}

template <typename T>
static void ln_bwd(const void* gyv, const void* xv, const float* gamma, const float* mean, const float* rstd, void* gxv,
                   float* dgamma, float* dbeta, float* part, long R, int C, hipStream_t st) {
  constexpr int VEC = 16 / elem<T>::kBytes;
  const T *gy = (const T*)gyv, *x = (const T*)xv;
  T* gx = (T*)gxv;
  const bool aln = C % VEC == 0 && ((uintptr_t)xv | (uintptr_t)gyv | (uintptr_t)gxv) % 16 == 0;
  int nrows = 0;
  const bool held = ln_plan<VEC>(C, [&](auto tpr, auto k) {
    constexpr int TPR = decltype(tpr)::value, K = decltype(k)::value, ROWS = ln_block(TPR) / TPR;
    const long steps = (R + ROWS - 1) / ROWS, each = (steps + kLnBwdBlocks - 1) / kLnBwdBlocks;
    nrows = (int)((steps + each - 1) / each);          // as few blocks as take the same number of steps
    const dim3 grid((unsigned)nrows), blk(ln_block(TPR));
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, blk, 0, st, gy, x, gamma, mean, rstd, gx, part, R, C); };
    if (aln) return run(layer_norm_bwd_kernel<T, kLnAligned, TPR, K>);
    if constexpr (TPR == 4)
      if (C < VEC) return run(layer_norm_bwd_kernel<T, kLnNarrow, TPR, K>);
    run(layer_norm_bwd_kernel<T, kLnAny, TPR, K>);
  });
  if (!held) {
    if (gx != nullptr)
      hipLaunchKernelGGL(layer_norm_wide_bwd_kernel<T>, dim3((unsigned)min(R, 4096L)), dim3(1024), 0, st, gy, x, gamma, mean, rstd, gx, R, C);
    nrows = (int)min(R, (long)kLnWideSlabs);
    if (part != nullptr)
      hipLaunchKernelGGL(layer_norm_wide_cols_kernel<T>, dim3((C + 255) / 256, nrows), dim3(256), 0, st, gy, x, mean, rstd, part, R, C);
  }
  if (part != nullptr)
    hipLaunchKernelGGL(layer_norm_cols_final_kernel, dim3((2 * C + 15) / 16), dim3(1024), 0, st, part, nrows, C, dgamma, dbeta);
}

static int ln_check(int64_t R, int C, int dtype, const char* who) {
  UBV_CHECK_ARG(R >= 0 && R < (int64_t(1) << 31) && C > 0 && C <= (1 << 29), "%s: R = %ld rows of C = %d are out of range", who, (long)R, C);
  UBV_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: unknown dtype %d", who, dtype);
  return UBV_OK;
}

}  // namespace ubv

extern "C" int ubv_layer_norm_forward(const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                                      int64_t R, int C, float eps, int dtype, void* stream) {
  using namespace ubv;
  const int rc = ln_check(R, C, dtype, "layer_norm_forward");
  if (rc) return rc;
  if (R == 0) return UBV_OK;
  UBV_CHECK_ARG(x && y && (mean == nullptr) == (rstd == nullptr), "layer_norm_forward: null pointer");
  hipStream_t st = as_stream(stream);
  switch (dtype) {
    case UBV_F32: ln_fwd<float>(x, gamma, beta, y, mean, rstd, (long)R, C, eps, st); break;
    case UBV_F16: ln_fwd<f16_t>(x, gamma, beta, y, mean, rstd, (long)R, C, eps, st); break;
    default: ln_fwd<bf16_t>(x, gamma, beta, y, mean, rstd, (long)R, C, eps, st); break;
  }
  UBV_CHECK_LAUNCH("layer_norm_forward");
  return UBV_OK;
}

extern "C" int64_t ubv_layer_norm_backward_workspace(int64_t R, int C) {
  const int64_t most = C > ubv::kLnHeld ? ubv::kLnWideSlabs : ubv::kLnBwdBlocks, rows = R < most ? R : most;
  return R <= 0 || C <= 0 ? 0 : rows * 2 * (int64_t)C * 4;
}

extern "C" int ubv_layer_norm_backward(const void* grad_y, const void* x, const float* gamma, const float* mean, const float* rstd,
                                       void* grad_x, float* grad_gamma, float* grad_beta, int64_t R, int C, int dtype,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ubv;
  const int rc = ln_check(R, C, dtype, "layer_norm_backward");
  if (rc) return rc;
  const bool cols = grad_gamma != nullptr || grad_beta != nullptr;
  UBV_CHECK_ARG(R > 0, "layer_norm_backward: no rows (the gradients are zero)");
  UBV_CHECK_ARG(grad_y && x && mean && rstd && (grad_x || cols), "layer_norm_backward: null pointer");
  UBV_CHECK_ARG(!cols || (workspace != nullptr && (uintptr_t)workspace % 4 == 0 &&
                          workspace_bytes >= ubv_layer_norm_backward_workspace(R, C)),
                "layer_norm_backward: the workspace is too small (%ld bytes)", (long)workspace_bytes);
  float* part = cols ? (float*)workspace : nullptr;
  hipStream_t st = as_stream(stream);
  switch (dtype) {
    case UBV_F32: ln_bwd<float>(grad_y, x, gamma, mean, rstd, grad_x, grad_gamma, grad_beta, part, (long)R, C, st); break;
    case UBV_F16: ln_bwd<f16_t>(grad_y, x, gamma, mean, rstd, grad_x, grad_gamma, grad_beta, part, (long)R, C, st); break;
    default: ln_bwd<bf16_t>(grad_y, x, gamma, mean, rstd, grad_x, grad_gamma, grad_beta, part, (long)R, C, st); break;
  }
  UBV_CHECK_LAUNCH("layer_norm_backward");
  return UBV_OK;
}
