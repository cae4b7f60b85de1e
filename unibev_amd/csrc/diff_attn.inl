// Kernels and launchers of differential attention for one element type: included once per type (diff_attn_f32.hip, ...),
// UBV_ATTN_T names it.
#include "diff_attn.h"

namespace ubv {

template <typename T, int DH, int DV> struct AttnTile {
  static constexpr int VEC = 16 / elem<T>::kBytes;
  static constexpr int LDK = DH + VEC, LDV = DV + VEC;      // 16 bytes of padding: fragment reads of 32 rows hit all banks alike
  static constexpr int KB = DH / 16, VB = DV / 16;          // 16-deep steps over a head's width
  static constexpr int KO = (DH + 31) / 32, VO = DV / 32;   // 32-wide output blocks
  static constexpr int bytes(int n) { return (n * (2 * LDK + LDV) + 32) * elem<T>::kBytes; }   // (+ 32: a 16-wide head's transposed reads)
  static constexpr int WK = bytes(128) <= 150 * 1024 ? 4 : 2;       // most waves that share one set of own items
};

// ---- staging: `n` items of 2 x DH (x) and DV (y) elements into LDS -----------------------------------------------------------
// the block's threads take 16-byte pieces; items past `valid`, hidden keys and columns past the head's width become zeros
template <typename T, int DH, int DV, int N> struct AttnStage {
  using S = AttnTile<T, DH, DV>;
  static constexpr int PX = 2 * DH / S::VEC, PY = DV / S::VEC, NX = N * PX / 256, NY = N * PY / 256;
  static_assert(N * PX % 256 == 0 && N * PY % 256 == 0, "pieces per thread");
  au32x4_t x[NX], y[NY];

  template <typename F> __device__ __forceinline__ void load(F&& item, int tid, int Dh, int Dv) {
#pragma unroll
    for (int c = 0; c < NX; ++c) {
      const int id = tid + 256 * c, it = id / PX, pc = id % PX, m = pc / (PX / 2), d = (pc % (PX / 2)) * S::VEC;
      x[c] = item(it, m, d, d < Dh);
    }
#pragma unroll
    for (int c = 0; c < NY; ++c) {
      const int id = tid + 256 * c, it = id / PY, d = (id % PY) * S::VEC;
      y[c] = item(it, 2, d, d < Dv);
    }
  }
  __device__ __forceinline__ void store(T* lds, int tid) {
#pragma unroll
    for (int c = 0; c < NX; ++c) {
      const int id = tid + 256 * c, it = id / PX, pc = id % PX, m = pc / (PX / 2), d = (pc % (PX / 2)) * S::VEC;
      *reinterpret_cast<au32x4_t*>(lds + (m * N + it) * S::LDK + d) = x[c];
    }
    T* ly = lds + 2 * N * S::LDK;
#pragma unroll
    for (int c = 0; c < NY; ++c) {
      const int id = tid + 256 * c, it = id / PY, d = (id % PY) * S::VEC;
      *reinterpret_cast<au32x4_t*>(ly + it * S::LDV + d) = y[c];
    }
  }
};

// a lane's own item as B operands: 8 elements at 16 s + 8 (lane >> 5) of step s
template <typename T, int NB>
__device__ __forceinline__ void own_frags(typename amma<T>::frag (&f)[NB], const T* p, bool ok, int D, int lane) {
  constexpr int VEC = 16 / elem<T>::kBytes;
#pragma unroll
  for (int s = 0; s < NB; ++s) {
    const int d = 16 * s + 8 * (lane >> 5);
    T t[8];
#pragma unroll
    for (int w = 0; w < 8 / VEC; ++w)
      *reinterpret_cast<au32x4_t*>(t + w * VEC) = piece(p + d + w * VEC, ok && d + w * VEC < D);
    f[s] = amma<T>::load(t);
  }
}

// 16 scores of own item (lane & 31) against staged items it0 .. it0 + 31
template <typename T, int NB, int LD>
__device__ __forceinline__ af32x16_t tile_dot(const T* tile, int it0, const typename amma<T>::frag (&own)[NB], int lane) {
  af32x16_t c = {0.0f};
  const T* p = tile + (it0 + (lane & 31)) * LD + 8 * (lane >> 5);
#pragma unroll
  for (int s = 0; s < NB; ++s) c = amma<T>::mul(amma<T>::load(p + 16 * s), own[s], c);
  return c;
}

// 4 consecutive elements of an output row of D elements
template <typename T> __device__ __forceinline__ void store_quad(T* row, int d, int D, const float (&v)[4]) {
  if (D % 4 == 0) {
    if (d < D) vec_io<T, 4>::store(row + d, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) row[d + i] = elem<T>::from_float(v[i]);
  }
}

// fields of the four staged rows 8 q + 4 (lane >> 5) + t of this lane's key: the four lanes of a key group each mix one row
// and hand it round
__device__ __forceinline__ void quad_fields(uint64_t mix, int lane, uint32_t (&f)[4]) {
  const int lo = (int)(uint32_t)mix, hi = (int)(uint32_t)(mix >> 32);
#define UBV_QUAD(t)                                                                             \
  {                                                                                             \
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp(lo, (t) * 0x55, 0xf, 0xf, true);     \
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp(hi, (t) * 0x55, 0xf, 0xf, true);     \
    f[t] = (((lane & 2) ? b : a) >> (16 * (lane & 1))) & 0xffffu;                              \
  }
  UBV_QUAD(0) UBV_QUAD(1) UBV_QUAD(2) UBV_QUAD(3)
#undef UBV_QUAD
}

// ---- forward -----------------------------------------------------------------------------------------------------------------
template <typename T, int DH, int DV, int WQ, int WK>
__global__ __launch_bounds__(256) void diff_attn_fwd_kernel(const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  using M = amma<T>;
  constexpr int BK = WK == 1 ? 64 : 32 * WK, SUB = BK / (32 * WK);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* lds = reinterpret_cast<T*>(smem);
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, wq = wv / WK, wk = wv % WK;
  const int tiles = (a.R + 32 * WQ - 1) / (32 * WQ);
  const int bh = blockIdx.x / tiles, rb = (blockIdx.x % tiles) * 32 * WQ;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int r = rb + 32 * wq + (lane & 31);
  const bool ok = r < a.R;
  const int rc = ok ? r : a.R - 1, h = hk * a.G + rc / a.Nq, i = rc % a.Nq;
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, rowid = ((int64_t)b * a.H + hk * a.G) * a.Nq + rc;
  const uint64_t seed = a.seed + (a.seed_dev != nullptr ? *a.seed_dev : 0);

  typename M::frag qf[2][S::KB];
#pragma unroll
  for (int m = 0; m < 2; ++m)
    own_frags<T, S::KB>(qf[m], (const T*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + m * a.qs[3], ok, a.Dh, lane);
  af32x16_t acc[2][S::VO];
  float mx[2] = {kNegInf, kNegInf}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int d = 0; d < S::VO; ++d) acc[m][d] = af32x16_t{0.0f};

  // keys that any row of the block sees
  int kend = a.Nk;
  if (a.causal) {
    const int last = min(rb + 32 * WQ, a.R) - 1;
    const int imax = rb / a.Nq == last / a.Nq ? last % a.Nq : a.Nq - 1;
    kend = max(0, min(a.Nk, imax + a.Nk - a.Nq + 1));
  }
  const T* kbase = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vbase = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const float c = a.scale * kLog2e;
  AttnStage<T, DH, DV, BK> st;
  for (int k0 = 0; k0 < kend; k0 += BK) {
    st.load([&](int it, int m, int d, bool in) {
      const int j = k0 + it;
      const bool use = in && j < a.Nk && !(a.kpm != nullptr && a.kpm[(int64_t)b * a.Nk + min(j, a.Nk - 1)]);
      return m < 2 ? piece(kbase + j * a.ks[1] + m * a.ks[3] + d, use) : piece(vbase + j * a.vs[1] + d, use);
    }, tid, a.Dh, a.Dv);
    __syncthreads();
    st.store(lds, tid);
    __syncthreads();
#pragma unroll 1
    for (int sub = 0; sub < SUB; ++sub) {
      const int it0 = (sub * WK + wk) * 32, j0 = k0 + it0;
      if (j0 >= kend) break;
      af32x16_t x[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) x[m] = tile_dot<T, S::KB, S::LDK>(lds + m * BK * S::LDK, it0, qf[m], lane);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[m][e] *= c;
      if (a.causal || a.kpm != nullptr || a.mask_kind != 0 || j0 + 32 > a.Nk) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = j0 + tile_item(e, lane);
          const float bias = j < a.Nk ? mask_bias(a, b, h, i, j) : kNegInf;
#pragma unroll
          for (int m = 0; m < 2; ++m) x[m][e] = bias == kNegInf ? kNegInf : x[m][e] + bias;
        }
      }
      float p[2][16];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float top = x[m][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, x[m][e]);
        top = fmaxf(mx[m], fmaxf(top, other_half(top)));
        if (__any(top > mx[m])) {                   // a larger maximum: what is summed so far shrinks (wave-uniform branch)
          const float al = aexp2(mx[m] - (top == kNegInf ? 0.0f : top));
          l[m] *= al;
#pragma unroll
          for (int d = 0; d < S::VO; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][d][e] *= al;
          mx[m] = top;
        }
        const float mu = mx[m] == kNegInf ? 0.0f : mx[m] - kProbShift<T>;
#pragma unroll
        for (int e = 0; e < 16; ++e) { p[m][e] = aexp2(x[m][e] - mu); l[m] += p[m][e]; }
      }
      if (a.t16 != 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint64_t mix = drop_mix64(seed, (uint64_t)(rowid * a.n4 + ((j0 + tile_item(4 * q, lane)) >> 2)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool keep = (uint32_t)((mix >> (16 * e)) & 0xffffull) >= a.t16;
#pragma unroll
            for (int m = 0; m < 2; ++m) p[m][4 * q + e] = keep ? p[m][4 * q + e] : 0.0f;
          }
        }
      }
      const T* vt = lds + 2 * BK * S::LDK;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const typename M::frag f0 = M::pack(p[0] + 8 * s), f1 = M::pack(p[1] + 8 * s);
#pragma unroll
        for (int d = 0; d < S::VO; ++d) {
          const typename M::frag vf = M::template load_tr<S::LDV>(vt, it0 + 16 * s, 32 * d, lane);
          acc[0][d] = M::mul(vf, f0, acc[0][d]);
          acc[1][d] = M::mul(vf, f1, acc[1][d]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) l[m] += other_half(l[m]);
  if constexpr (WK > 1) {                            // join the waves that walked other keys of the same rows
    float* mrg = reinterpret_cast<float*>(smem);
    constexpr int SLOT = (4 + DV) * 64;
#pragma unroll 1
    for (int half = WK / 2; half >= 1; half >>= 1) {
      __syncthreads();
      float* slot = mrg + (wq * (WK / 2) + wk % half) * SLOT + lane;
      if (wk >= half && wk < 2 * half) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          slot[(2 * m) * 64] = mx[m]; slot[(2 * m + 1) * 64] = l[m];
#pragma unroll
          for (int d = 0; d < S::VO; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) slot[(4 + (m * S::VO + d) * 16 + e) * 64] = acc[m][d][e];
        }
      }
      __syncthreads();
      if (wk < half) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float mo = slot[(2 * m) * 64], top = fmaxf(mx[m], mo), mu = top == kNegInf ? 0.0f : top;
          const float f0 = aexp2(mx[m] - mu), f1 = aexp2(mo - mu);
          l[m] = l[m] * f0 + slot[(2 * m + 1) * 64] * f1;
          mx[m] = top;
#pragma unroll
          for (int d = 0; d < S::VO; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              acc[m][d][e] = acc[m][d][e] * f0 + slot[(4 + (m * S::VO + d) * 16 + e) * 64] * f1;
        }
      }
    }
    if (wk != 0) return;
  }
  if (!ok) return;
  const float lam = a.lam[h];
  float inv[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    inv[m] = l[m] == 0.0f ? 0.0f : a.up / l[m];
    if (a.lse != nullptr && lane < 32) a.lse[m * rows + rowid] = mx[m] - kProbShift<T> + log2f(l[m]);
  }
  T* orow = (T*)a.out + (((int64_t)b * a.Nq + i) * a.H + h) * a.Dv;
#pragma unroll
  for (int d = 0; d < S::VO; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dv = 32 * d + tile_item(4 * q, lane);
      float o1[4], o2[4], o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o1[e] = acc[0][d][4 * q + e] * inv[0];
        o2[e] = acc[1][d][4 * q + e] * inv[1];
        o[e] = fmaf(-lam, o2[e], o1[e]);
      }
      store_quad<T>(orow, dv, a.Dv, o);
      if (a.o != nullptr) {
        store_quad<float>(a.o + rowid * a.Dv, dv, a.Dv, o1);
        store_quad<float>(a.o + (rows + rowid) * a.Dv, dv, a.Dv, o2);
      }
    }
}

// ---- backward: del_m = grad_out . o_m per row, 16 lanes a row -----------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void diff_attn_del_kernel(const DiffAttnArgs a) {
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, rowid = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int t = threadIdx.x & 15;
  const int64_t rr = rowid < rows ? rowid : rows - 1;
  const int i = (int)(rr % a.Nq), h = (int)(rr / a.Nq % a.H);
  const int64_t b = rr / a.Nq / a.H;
  const T* g = (const T*)a.go + b * a.gs[0] + i * a.gs[1] + h * a.gs[2];
  const float *o1 = a.o + rr * a.Dv, *o2 = a.o + (rows + rr) * a.Dv;
  float s1 = 0.0f, s2 = 0.0f;
  for (int d = t; d < a.Dv; d += 16) {
    const float gv = elem<T>::to_float(g[d]);
    s1 = fmaf(gv, o1[d], s1);
    s2 = fmaf(gv, o2[d], s2);
  }
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) { s1 += __shfl_xor(s1, m, 64); s2 += __shfl_xor(s2, m, 64); }
  if (t == 0 && rowid < rows) { a.del[rowid] = s1; a.del[rows + rowid] = s2; }
}

// sums over the waves of a block that walked other staged items of the same own items; the result is in the waves wk == 0
template <int WQ, int WK, int NB>
__device__ __forceinline__ void join_waves(af32x16_t* const (&acc)[NB], float* mrg, int wq, int wk, int lane) {
#pragma unroll 1
  for (int half = WK / 2; half >= 1; half >>= 1) {
    __syncthreads();
    float* slot = mrg + (wq * (WK / 2) + wk % half) * (NB * 16 * 64) + lane;
    if (wk >= half && wk < 2 * half) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) slot[(n * 16 + e) * 64] = (*acc[n])[e];
    }
    __syncthreads();
    if (wk < half) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) (*acc[n])[e] += slot[(n * 16 + e) * 64];
    }
  }
}

// ---- backward: grad_q and the rows' parts of grad_lam; own = rows, staged = keys ---------------------------------------------
template <typename T, int DH, int DV, int WQ, int WK>
__global__ __launch_bounds__(256) void diff_attn_bwd_q_kernel(const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  using M = amma<T>;
  constexpr int BK = WK == 1 ? 64 : 32 * WK, SUB = BK / (32 * WK);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* lds = reinterpret_cast<T*>(smem);
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, wq = wv / WK, wk = wv % WK;
  const int tiles = (a.R + 32 * WQ - 1) / (32 * WQ);
  const int bh = blockIdx.x / tiles, rb = (blockIdx.x % tiles) * 32 * WQ;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int r = rb + 32 * wq + (lane & 31);
  const bool ok = r < a.R;
  const int rc = ok ? r : a.R - 1, h = hk * a.G + rc / a.Nq, i = rc % a.Nq;
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, rowid = ((int64_t)b * a.H + hk * a.G) * a.Nq + rc;
  const uint64_t seed = a.seed + (a.seed_dev != nullptr ? *a.seed_dev : 0);

  typename M::frag qf[2][S::KB], gf[S::VB];
  float lse[2], del[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    own_frags<T, S::KB>(qf[m], (const T*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + m * a.qs[3], ok, a.Dh, lane);
    const float v = a.lse[m * rows + rowid];
    lse[m] = !ok || v == kNegInf ? -kNegInf : v;     // no key seen: every probability is exp2(x - inf) = 0
    del[m] = a.del[m * rows + rowid];
  }
  own_frags<T, S::VB>(gf, (const T*)a.go + b * a.gs[0] + i * a.gs[1] + h * a.gs[2], ok, a.Dv, lane);
  af32x16_t acc[2][S::KO];
  float dl = 0.0f;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int d = 0; d < S::KO; ++d) acc[m][d] = af32x16_t{0.0f};
  int kend = a.Nk;
  if (a.causal) {
    const int last = min(rb + 32 * WQ, a.R) - 1;
    const int imax = rb / a.Nq == last / a.Nq ? last % a.Nq : a.Nq - 1;
    kend = max(0, min(a.Nk, imax + a.Nk - a.Nq + 1));
  }
  const T* kbase = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vbase = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const float c = a.scale * kLog2e;
  AttnStage<T, DH, DV, BK> st;
  for (int k0 = 0; k0 < kend; k0 += BK) {
    st.load([&](int it, int m, int d, bool in) {
      const int j = k0 + it;
      const bool use = in && j < a.Nk && !(a.kpm != nullptr && a.kpm[(int64_t)b * a.Nk + min(j, a.Nk - 1)]);
      return m < 2 ? piece(kbase + j * a.ks[1] + m * a.ks[3] + d, use) : piece(vbase + j * a.vs[1] + d, use);
    }, tid, a.Dh, a.Dv);
    __syncthreads();
    st.store(lds, tid);
    __syncthreads();
#pragma unroll 1
    for (int sub = 0; sub < SUB; ++sub) {
      const int it0 = (sub * WK + wk) * 32, j0 = k0 + it0;
      if (j0 >= kend) break;
      af32x16_t x[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        x[m] = tile_dot<T, S::KB, S::LDK>(lds + m * BK * S::LDK, it0, qf[m], lane);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[m][e] *= c;
      }
      if (a.causal || a.kpm != nullptr || a.mask_kind != 0 || j0 + 32 > a.Nk) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = j0 + tile_item(e, lane);
          const float bias = j < a.Nk ? mask_bias(a, b, h, i, j) : kNegInf;
#pragma unroll
          for (int m = 0; m < 2; ++m) x[m][e] = bias == kNegInf ? kNegInf : x[m][e] + bias;
        }
      }
      af32x16_t g = tile_dot<T, S::VB, S::LDV>(lds + 2 * BK * S::LDK, it0, gf, lane);
      if (a.t16 != 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint64_t mix = drop_mix64(seed, (uint64_t)(rowid * a.n4 + ((j0 + tile_item(4 * q, lane)) >> 2)));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            g[4 * q + e] = (uint32_t)((mix >> (16 * e)) & 0xffffull) >= a.t16 ? g[4 * q + e] * a.up : 0.0f;
        }
      }
      float ds[2][16], dt = 0.0f;                     // (the tile's own sum first: 16 times fewer additions to the long one)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p1 = aexp2(x[0][e] - lse[0]), p2 = aexp2(x[1][e] - lse[1]);
        dt = fmaf(p2, g[e], dt);
        ds[0][e] = p1 * (g[e] - del[0]);
        ds[1][e] = p2 * (g[e] - del[1]);
      }
      dl += dt;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const typename M::frag f = M::pack(ds[m] + 8 * s);
#pragma unroll
          for (int d = 0; d < S::KO; ++d)
            acc[m][d] = M::mul(M::template load_tr<S::LDK>(lds + m * BK * S::LDK, it0 + 16 * s, 32 * d, lane), f, acc[m][d]);
        }
    }
  }
  dl += other_half(dl);
  if constexpr (WK > 1) {
    af32x16_t dlv = {dl};
    af32x16_t* ptr[2 * S::KO + 1];
#pragma unroll
    for (int d = 0; d < S::KO; ++d) { ptr[d] = &acc[0][d]; ptr[S::KO + d] = &acc[1][d]; }
    ptr[2 * S::KO] = &dlv;
    join_waves<WQ, WK>(ptr, reinterpret_cast<float*>(smem), wq, wk, lane);
    if (wk != 0) return;
    dl = dlv[0];
  }
  if (!ok) return;
  if (lane < 32) a.dlrow[rowid] = -dl;
  if (a.gq == nullptr) return;
  const float f[2] = {a.scale, -a.lam[h] * a.scale};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    T* row = (T*)a.gq + ((((int64_t)b * a.Nq + i) * a.H + h) * 2 + m) * a.Dh;
#pragma unroll
    for (int d = 0; d < S::KO; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = acc[m][d][4 * q + e] * f[m];
        store_quad<T>(row, 32 * d + tile_item(4 * q, lane), a.Dh, o);
      }
  }
}

// grad_lam[h] = sum over the batch and the queries, one block a head, fixed order
__global__ __launch_bounds__(256) static void diff_attn_lam_kernel(const float* __restrict__ dlrow, float* __restrict__ glam, int B, int H,
                                                                   int Nq) {
  __shared__ float red[4];
  const int h = blockIdx.x;
  float s = 0.0f;
  for (int b = 0; b < B; ++b)
    for (int i = threadIdx.x; i < Nq; i += 256) s += dlrow[((int64_t)b * H + h) * Nq + i];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) glam[h] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- backward: grad_k and grad_v; own = keys, staged = the rows of every head that shares them --------------------------------
template <typename T, int DH, int DV, int WQ, int WK>
__global__ __launch_bounds__(256) void diff_attn_bwd_kv_kernel(const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  using M = amma<T>;
  constexpr int BK = WK == 1 ? 64 : 32 * WK, SUB = BK / (32 * WK);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ __attribute__((aligned(16))) float stat[5][BK];     // lse_1, lse_2, del_1, del_2, lam of the staged rows
  T* lds = reinterpret_cast<T*>(smem);
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, wq = wv / WK, wk = wv % WK;
  const int tiles = (a.Nk + 32 * WQ - 1) / (32 * WQ);
  const int bh = blockIdx.x / tiles, jb = (blockIdx.x % tiles) * 32 * WQ;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int j = jb + 32 * wq + (lane & 31);
  // a hidden key's column is computed from zeros and its gradients are stored as zeros: no masking needed for it
  const bool in = j < a.Nk, ok = in && !(a.kpm != nullptr && a.kpm[(int64_t)b * a.Nk + (in ? j : 0)]);
  const int jc = in ? j : a.Nk - 1;
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, row0 = ((int64_t)b * a.H + hk * a.G) * a.Nq;
  const uint64_t seed = a.seed + (a.seed_dev != nullptr ? *a.seed_dev : 0);

  typename M::frag kf[2][S::KB], vf[S::VB];
#pragma unroll
  for (int m = 0; m < 2; ++m)
    own_frags<T, S::KB>(kf[m], (const T*)a.k + b * a.ks[0] + jc * a.ks[1] + hk * a.ks[2] + m * a.ks[3], ok, a.Dh, lane);
  own_frags<T, S::VB>(vf, (const T*)a.v + b * a.vs[0] + jc * a.vs[1] + hk * a.vs[2], ok, a.Dv, lane);
  af32x16_t ak[2][S::KO], av[S::VO];
#pragma unroll
  for (int d = 0; d < S::KO; ++d) { ak[0][d] = af32x16_t{0.0f}; ak[1][d] = af32x16_t{0.0f}; }
#pragma unroll
  for (int d = 0; d < S::VO; ++d) av[d] = af32x16_t{0.0f};
  const float c = a.scale * kLog2e;
  AttnStage<T, DH, DV, BK> st;
  for (int r0 = 0; r0 < a.R; r0 += BK) {
    if (a.causal) {                                   // no row of the tile sees a key of the block
      const int last = min(r0 + BK, a.R) - 1;
      const int imax = r0 / a.Nq == last / a.Nq ? last % a.Nq : a.Nq - 1;
      if (imax + a.Nk - a.Nq < jb) continue;
    }
    st.load([&](int it, int m, int d, bool use) {
      const int r = r0 + it, rc = r < a.R ? r : a.R - 1, h = hk * a.G + rc / a.Nq, i = rc % a.Nq;
      use = use && r < a.R;
      return m < 2 ? piece((const T*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + m * a.qs[3] + d, use)
                   : piece((const T*)a.go + b * a.gs[0] + i * a.gs[1] + h * a.gs[2] + d, use);
    }, tid, a.Dh, a.Dv);
    float sv[5] = {-kNegInf, -kNegInf, 0.0f, 0.0f, 0.0f};
    if (tid < BK && r0 + tid < a.R) {
      const int64_t rid = row0 + r0 + tid;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float v = a.lse[m * rows + rid];
        sv[m] = v == kNegInf ? -kNegInf : v;
        sv[2 + m] = a.del[m * rows + rid];
      }
      sv[4] = a.lam[hk * a.G + (r0 + tid) / a.Nq];
    }
    __syncthreads();
    st.store(lds, tid);
    if (tid < BK) {
#pragma unroll
      for (int n = 0; n < 5; ++n) stat[n][tid] = sv[n];
    }
    __syncthreads();
#pragma unroll 1
    for (int sub = 0; sub < SUB; ++sub) {
      const int it0 = (sub * WK + wk) * 32;
      if (r0 + it0 >= a.R) break;
      af32x16_t x[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        x[m] = tile_dot<T, S::KB, S::LDK>(lds + m * BK * S::LDK, it0, kf[m], lane);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[m][e] *= c;
      }
      if (a.causal || a.mask_kind != 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = min(r0 + it0 + tile_item(e, lane), a.R - 1);
          const float bias = mask_bias(a, b, hk * a.G + r / a.Nq, r % a.Nq, jc);
#pragma unroll
          for (int m = 0; m < 2; ++m) x[m][e] = bias == kNegInf ? kNegInf : x[m][e] + bias;
        }
      }
      const af32x16_t g = tile_dot<T, S::VB, S::LDV>(lds + 2 * BK * S::LDK, it0, vf, lane);
      float pc[16], ds[2][16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int t0 = it0 + tile_item(4 * q, lane);
        uint32_t fld[4];
        if (a.t16 != 0) quad_fields(drop_mix64(seed, (uint64_t)((row0 + r0 + t0 + (lane & 3)) * a.n4 + (j >> 2))), lane, fld);
        float s[5][4];
#pragma unroll
        for (int n = 0; n < 5; ++n) *reinterpret_cast<float4*>(s[n]) = *reinterpret_cast<const float4*>(&stat[n][t0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = 4 * q + e;
          const float p1 = aexp2(x[0][n] - s[0][e]), p2 = s[4][e] * aexp2(x[1][n] - s[1][e]);
          float gn = g[n], pn = p1 - p2;
          if (a.t16 != 0) {
            const bool keep = fld[e] >= a.t16;
            gn = keep ? gn * a.up : 0.0f;
            pn = keep ? pn : 0.0f;
          }
          pc[n] = kProbScale<T> == 1.0f ? pn : pn * kProbScale<T>;
          ds[0][n] = p1 * (gn - s[2][e]);
          ds[1][n] = p2 * (s[3][e] - gn);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const typename M::frag fp = M::pack(pc + 8 * s);
#pragma unroll
        for (int d = 0; d < S::VO; ++d)
          av[d] = M::mul(M::template load_tr<S::LDV>(lds + 2 * BK * S::LDK, it0 + 16 * s, 32 * d, lane), fp, av[d]);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const typename M::frag f = M::pack(ds[m] + 8 * s);
#pragma unroll
          for (int d = 0; d < S::KO; ++d)
            ak[m][d] = M::mul(M::template load_tr<S::LDK>(lds + m * BK * S::LDK, it0 + 16 * s, 32 * d, lane), f, ak[m][d]);
        }
      }
    }
  }
  if constexpr (WK > 1) {
    af32x16_t* ptr[2 * S::KO + S::VO];
#pragma unroll
    for (int d = 0; d < S::KO; ++d) { ptr[d] = &ak[0][d]; ptr[S::KO + d] = &ak[1][d]; }
#pragma unroll
    for (int d = 0; d < S::VO; ++d) ptr[2 * S::KO + d] = &av[d];
    join_waves<WQ, WK>(ptr, reinterpret_cast<float*>(smem), wq, wk, lane);
    if (wk != 0) return;
  }
  if (!in) return;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    T* row = (T*)a.gk + ((((int64_t)b * a.Nk + j) * a.Hk + hk) * 2 + m) * a.Dh;
#pragma unroll
    for (int d = 0; d < S::KO; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = ok ? ak[m][d][4 * q + e] * a.scale : 0.0f;
        store_quad<T>(row, 32 * d + tile_item(4 * q, lane), a.Dh, o);
      }
  }
  const float fv = a.up / kProbScale<T>;
  T* row = (T*)a.gv + (((int64_t)b * a.Nk + j) * a.Hk + hk) * a.Dv;
#pragma unroll
  for (int d = 0; d < S::VO; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = ok ? av[d][4 * q + e] * fv : 0.0f;
      store_quad<T>(row, 32 * d + tile_item(4 * q, lane), a.Dv, o);
    }
}

// ---- launch -----------------------------------------------------------------------------------------------------------------------
template <typename K>
static int attn_launch(K kernel, int64_t blocks, int lds, const DiffAttnArgs& a, hipStream_t st, const char* who) {
  if (blocks >= (int64_t(1) << 31)) { set_error("%s: %ld blocks", who, (long)blocks); return UBV_ERR_UNSUPPORTED; }
  if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), (size_t)lds, st, a);
  UBV_CHECK_LAUNCH(who);
  return UBV_OK;
}

constexpr int64_t kAttnFill = 512;      // blocks of 4 waves that keep the 256 CUs busy

template <typename T, int DH, int DV>
static int attn_forward(const DiffAttnArgs& a, hipStream_t st) {
  using S = AttnTile<T, DH, DV>;
  constexpr int WK = S::WK, WQ = 4 / WK, MRG = WQ * (WK / 2) * (4 + DV) * 64 * 4;
  const int64_t heads = (int64_t)a.B * a.Hk, wide = heads * ((a.R + 127) / 128);
  if (wide >= kAttnFill)
    return attn_launch(diff_attn_fwd_kernel<T, DH, DV, 4, 1>, wide, S::bytes(64), a, st, "diff_attention_forward");
  constexpr int lds = S::bytes(32 * WK) > MRG ? S::bytes(32 * WK) : MRG;
  return attn_launch(diff_attn_fwd_kernel<T, DH, DV, WQ, WK>, heads * ((a.R + 32 * WQ - 1) / (32 * WQ)), lds, a, st, "diff_attention_forward");
}

template <typename T, int DH, int DV>
static int attn_backward(const DiffAttnArgs& a, float* glam, hipStream_t st) {
  using S = AttnTile<T, DH, DV>;
  constexpr int WK = S::WK, WQ = 4 / WK;
  constexpr int MQ = WQ * (WK / 2) * (2 * S::KO + 1) * 16 * 64 * 4, MKV = WQ * (WK / 2) * (2 * S::KO + S::VO) * 16 * 64 * 4;
  constexpr int TL = S::bytes(32 * WK);
  const int64_t heads = (int64_t)a.B * a.Hk, rows = (int64_t)a.B * a.H * a.Nq;
  hipLaunchKernelGGL(diff_attn_del_kernel<T>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a);
  UBV_CHECK_LAUNCH("diff_attention_backward");
  int rc = UBV_OK;
  if (a.gq != nullptr || glam != nullptr) {
    const int64_t wide = heads * ((a.R + 127) / 128);
    if (wide >= kAttnFill)
      rc = attn_launch(diff_attn_bwd_q_kernel<T, DH, DV, 4, 1>, wide, S::bytes(64), a, st, "diff_attention_backward");
    else
      rc = attn_launch(diff_attn_bwd_q_kernel<T, DH, DV, WQ, WK>, heads * ((a.R + 32 * WQ - 1) / (32 * WQ)), TL > MQ ? TL : MQ, a, st,
                       "diff_attention_backward");
    if (rc != UBV_OK) return rc;
    if (glam != nullptr) {
      hipLaunchKernelGGL(diff_attn_lam_kernel, dim3((unsigned)a.H), dim3(256), 0, st, a.dlrow, glam, a.B, a.H, a.Nq);
      UBV_CHECK_LAUNCH("diff_attention_backward");
    }
  }
  if (a.gk != nullptr) {
    const int64_t wide = heads * ((a.Nk + 127) / 128);
    if (wide >= kAttnFill)
      rc = attn_launch(diff_attn_bwd_kv_kernel<T, DH, DV, 4, 1>, wide, S::bytes(64), a, st, "diff_attention_backward");
    else
      rc = attn_launch(diff_attn_bwd_kv_kernel<T, DH, DV, WQ, WK>, heads * ((a.Nk + 32 * WQ - 1) / (32 * WQ)), TL > MKV ? TL : MKV, a, st,
                       "diff_attention_backward");
  }
  return rc;
}

// the smallest pair of widths that holds the call's
#define UBV_ATTN_PAIRS(DO)                                                                    \
  if (a.Dh <= 16 && a.Dv <= 32) DO(16, 32)                                                    \
  if (a.Dh <= 32 && a.Dv <= 64) DO(32, 64)                                                    \
  if (a.Dh <= 64 && a.Dv <= 64) DO(64, 64)                                                    \
  if (a.Dh <= 64 && a.Dv <= 128) DO(64, 128)                                                  \
  if (a.Dh <= 128 && a.Dv <= 128) DO(128, 128)                                                \
  DO(128, 256)

int UBV_ATTN_NAME(forward)(const DiffAttnArgs& a, hipStream_t st) {
#define UBV_DO(DH, DV) return attn_forward<UBV_ATTN_T, DH, DV>(a, st);
  UBV_ATTN_PAIRS(UBV_DO)
#undef UBV_DO
}

int UBV_ATTN_NAME(backward)(const DiffAttnArgs& a, float* glam, hipStream_t st) {
#define UBV_DO(DH, DV) return attn_backward<UBV_ATTN_T, DH, DV>(a, glam, st);
  UBV_ATTN_PAIRS(UBV_DO)
#undef UBV_DO
}

}  // namespace ubv
