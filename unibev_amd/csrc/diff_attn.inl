// Kernels and launchers of differential attention for one element type: included once per type (diff_attn_f32.hip, ...),
// UBV_ATTN_T names it.
//
// Two arrangements of the same wave program (a wave: 32 own items against a stream of 32-item tiles):
//   shared   the block's four waves have 128 own items and share each staged tile (two LDS buffers, one barrier a tile)
//   private  the block's waves have the SAME 32 own items, every wave stages tiles of its own (one buffer, no barrier: a wave's
//            LDS accesses are in order) and the waves' sums are joined through LDS at the end: four times the blocks
// In both the next tile's global loads are issued before the present tile is worked on.  Loads are buffer loads whose offset is
// sent out of bounds where a zero is wanted: items past the end, hidden keys, columns past the head's width.
#include "diff_attn.h"

namespace ubv {

template <typename T, int DH, int DV> struct AttnTile {
  static constexpr int VEC = 16 / elem<T>::kBytes;
  static constexpr int LX = 2 * DH / VEC, LY = DV / VEC;    // 16-byte chunks of a staged row: x of both maps, y
  static constexpr int KB = DH / 16, VB = DV / 16;          // 16-deep steps over a head's width
  static constexpr int KO = (DH + 31) / 32, VO = DV / 32;   // 32-wide output blocks
  // a staged tile of n items: x, y, and the rows' statistics of the backward pass (float4 + float2 each)
  static constexpr int xbytes(int n) { return n * 16 * LX; }
  static constexpr int xybytes(int n) { return n * 16 * (LX + LY); }
  static constexpr int bytes(int n) { return xybytes(n) + 24 * n; }
  static constexpr int QFLOATS = 32 * KO + 4, KFLOATS = 16 * (2 * KO + VO);      // a lane's sums in a split's workspace
  // two waves a SIMD (256 registers each) up to 32 / 64, where a 16-bit type's accumulators, operands and tile in flight about fit
  // (grad_k / grad_v at 32 / 64 spills 2 to 11, with masks 27); wider heads take one (64 / 128, f16: forward 244 us with two waves that
  // spill, 167 with one that does not).  f32's operands are twice as long: its grad_k / grad_v spills at 32 / 64, 2 to 33 registers as
  // private blocks and 45 to 137 as shared ones.
  static constexpr int MINW = DH <= 32 && DV <= 64 ? 2 : 1;
  // own operands in registers: 2 KB + VB operands of 4 registers, f32 8: at 128 / 256 that is 256 beside the accumulators, and read
  // again they cost less than spilled (8 heads, 1024 x 1024, us: grad_q 1360 spilled, 369; held where they fit: 64 / 128 1500 x 1500
  // 188, read again 266).  16-bit heads past 64 keep them and spill up to 84 others, most in shared blocks of grad_k at 128 / 256.
  static constexpr bool KEEP = elem<T>::kBytes == 2 || DH <= 64;
  static constexpr int fit(int w) { return w > 2 && w * bytes(32) > 150 * 1024 ? fit(w / 2) : w; }
  // waves of a private block.  16-bit heads up to 32 / 64: all of a CU's, which halves a block's time where blocks are few (2 x 4
  // heads, 900 x 900 bf16, us: 56 with eight waves, 64 with four; 4 heads, 10 000 x 10 000: 1090, 1050); f32's tiles are longer
  // (8 heads of 16 / 32, 2 x 900: 173, 148)
  static constexpr int WK = fit(elem<T>::kBytes == 2 ? 4 * MINW : 4);
  static constexpr int NS = 2 * bytes(64) <= 76 * 1024 ? 64 : 32;                // items of a shared tile
};

template <typename T, int DH, int DV, bool SHARED> struct AttnPlan {
  using S = AttnTile<T, DH, DV>;
  static constexpr int WK = SHARED ? 1 : S::WK, WQ = SHARED ? 4 : 1;             // waves per own items / groups of own items
  static constexpr int NW = WK * WQ, NT = 64 * NW;
  static constexpr int N = SHARED ? S::NS : 32;                                  // items of a staged tile
  static constexpr int LT = SHARED ? NT : 64;                                    // threads that stage a tile
  static constexpr int LDS = (SHARED ? 2 : WK) * S::bytes(N);
  static constexpr int merge(int floats) { return SHARED ? 0 : (WK / 2) * floats * 64 * 4; }     // joining `floats` per lane
  static constexpr int lds(int floats) { return LDS > merge(floats) ? LDS : merge(floats); }
  static constexpr int MINW = S::MINW;
  // 16-byte pieces of a tile that a thread holds: at most a quarter of its registers
  static constexpr bool PREF = S::xybytes(N) / LT / 16 <= (MINW == 2 ? 8 : 16);
  static_assert(PREF || !SHARED, "a shared tile passes through registers");
};

// What a call may hold beside hidden keys.  Each has kernels of its own: what a kernel can never meet costs it registers, and
// with them a wave per SIMD (32 / 64 wide heads, bf16, 10 000 x 10 000: grad_k / grad_v 738 us with everything, 448 plain,
// dS in one operand).
constexpr int kAttnPlain = 0, kAttnDrop = 1, kAttnCausal = 2, kAttnAny = 3;       // nothing | dropout | causal | masks, any of it together

// ---- staging ------------------------------------------------------------------------------------------------------------------
// PREF: a tile's pieces wait in registers until the present tile is done with; else they pass through in groups of 8
template <typename T, int DH, int DV, int N, int LT, bool PREF> struct AttnStage {
  using S = AttnTile<T, DH, DV>;
  static constexpr int PX = S::LX, PY = S::LY, NX = N * PX / LT, NY = N * PY / LT;
  static_assert(N * PX % LT == 0 && N * PY % LT == 0 && LT % PX == 0 && LT % PY == 0, "a thread keeps its column");
  au32x4_t x[PREF ? NX : 1], y[PREF ? NY : 1];
  uint32_t xoff, yoff;               // this thread's byte offset inside a tile, kOutside past the head's width

  __device__ __forceinline__ void init(int t, uint32_t xrow, uint32_t xmap, uint32_t yrow, int Dh, int Dv) {
    const int pc = t % PX, m = pc / (PX / 2), dx = (pc % (PX / 2)) * S::VEC, dy = (t % PY) * S::VEC;
    xoff = dx < Dh ? (t / PX) * xrow + m * xmap + dx * elem<T>::kBytes : kOutside;
    yoff = dy < Dv ? (t / PY) * yrow + dy * elem<T>::kBytes : kOutside;
  }
  // byte offset of piece c of x (y): kOutside where bit `item` of hid is set (the item becomes zeros)
  __device__ __forceinline__ uint32_t at(uint32_t off, int item, uint64_t hid) const { return hid != 0 && ((hid >> item) & 1) ? kOutside : off; }
  __device__ __forceinline__ void load(const char* xb, uint32_t xrow, const char* yb, uint32_t yrow, uint64_t hid, int t) {
    const __amdgpu_buffer_rsrc_t rx = attn_rsrc(xb), ry = attn_rsrc(yb);
    if (hid == 0) {
#pragma unroll
      for (int c = 0; c < NX; ++c) x[c] = attn_piece(rx, xoff, c * (LT / PX) * xrow);
#pragma unroll
      for (int c = 0; c < NY; ++c) y[c] = attn_piece(ry, yoff, c * (LT / PY) * yrow);
    } else {
#pragma unroll
      for (int c = 0; c < NX; ++c) x[c] = attn_piece(rx, at(xoff, t / PX + c * (LT / PX), hid), c * (LT / PX) * xrow);
#pragma unroll
      for (int c = 0; c < NY; ++c) y[c] = attn_piece(ry, at(yoff, t / PY + c * (LT / PY), hid), c * (LT / PY) * yrow);
    }
  }
  // place of piece c (a thread's rows are its first one plus multiples of a power of two above it: their folds XOR)
  template <int L> static __device__ __forceinline__ char* place(char* lds, int t, int c) {
    const int o = (t / L) * 16 * L + (((t % L) ^ row_fold<L>(t / L)) << 4);
    return lds + c * (LT / L) * 16 * L + (o ^ (row_fold<L>(c * (LT / L)) << 4));
  }
  __device__ __forceinline__ void store(char* lds, int t) {
#pragma unroll
    for (int c = 0; c < NX; ++c) *reinterpret_cast<au32x4_t*>(place<PX>(lds, t, c)) = x[c];
#pragma unroll
    for (int c = 0; c < NY; ++c) *reinterpret_cast<au32x4_t*>(place<PY>(lds + S::xbytes(N), t, c)) = y[c];
  }
  template <int L, int COUNT> __device__ __forceinline__ void pass(const char* base, uint32_t row, uint32_t off, uint64_t hid, char* lds, int t) const {
    const __amdgpu_buffer_rsrc_t r = attn_rsrc(base);
    constexpr int G = COUNT < 8 ? COUNT : 8;
#pragma unroll
    for (int c0 = 0; c0 < COUNT; c0 += G) {
      au32x4_t v[G];
#pragma unroll
      for (int c = 0; c < G; ++c) v[c] = attn_piece(r, at(off, t / L + (c0 + c) * (LT / L), hid), (c0 + c) * (LT / L) * row);
#pragma unroll
      for (int c = 0; c < G; ++c) *reinterpret_cast<au32x4_t*>(place<L>(lds, t, c0 + c)) = v[c];
      __builtin_amdgcn_sched_barrier(0);               // (or all groups' loads would be drawn together, and need the registers)
    }
  }
  __device__ __forceinline__ void through(const char* xb, uint32_t xrow, const char* yb, uint32_t yrow, uint64_t hid, char* lds, int t) const {
    pass<PX, NX>(xb, xrow, xoff, hid, lds, t);
    pass<PY, NY>(yb, yrow, yoff, hid, lds + S::xbytes(N), t);
  }
};

// the staged tile is there for every lane that reads it
template <bool SHARED> __device__ __forceinline__ void tile_ready() {
  if constexpr (SHARED) __syncthreads();
  else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// A lane's own item as B operands: 8 elements at 16 s + 8 (lane >> 5) of step s.  KEEP: held in registers; else (f32 heads past 64)
// read again for every tile, where the accumulators leave no room for them: 48 to 64 KB a tile in a private block, 192 to 256 KB in a
// shared one, more than the L1, so from L2.  Four rows of waves to a tile make up for it: 2 x 16 heads of 128 / 128, 1024 x 1024, us,
// shared / private: forward 445 / 862, grad_q 610 / 1293.
template <typename T, int NB, bool KEEP> struct OwnRow {
  static constexpr int VEC = 16 / elem<T>::kBytes;
  typename amma<T>::frag f[KEEP ? NB : 1];
  const T* p;
  bool ok;
  int D, d0;

  // p: a row of the tensor also where !ok (loaded, then dropped)
  __device__ __forceinline__ void init(const T* row, bool ok_, int D_, int lane) {
    p = row; ok = ok_; D = D_; d0 = 8 * (lane >> 5);
    if constexpr (KEEP) {
#pragma unroll
      for (int s = 0; s < NB; ++s) f[s] = read(s);
    }
  }
  __device__ __forceinline__ typename amma<T>::frag read(int s) const {
    T t[8];
#pragma unroll
    for (int w = 0; w < 8 / VEC; ++w) {
      const int d = 16 * s + d0 + w * VEC;
      const bool in = ok && d < D;
      const au32x4_t v = *reinterpret_cast<const au32x4_t*>(p + (in ? d : 0)), z = {0u, 0u, 0u, 0u};
      *reinterpret_cast<au32x4_t*>(t + w * VEC) = in ? v : z;
    }
    return amma<T>::own(t);
  }
  __device__ __forceinline__ typename amma<T>::frag get(int s) const {
    if constexpr (KEEP) return f[s];
    else return read(s);
  }
  // a new tile: what was read for the last one is not to be kept
  __device__ __forceinline__ void again() {
    if constexpr (!KEEP) asm volatile("" : "+v"(p));
  }
};

// 16 dot products of own item (lane & 31) with staged items it0 .. it0 + 31, over the part of their rows from chunk c0
template <typename T, int NB, int L, bool KEEP>
__device__ __forceinline__ af32x16_t tile_dot(const char* tile, int it0, int c0, OwnRow<T, NB, KEEP>& own, int lane) {
  af32x16_t c = {0.0f};
  own.again();
#pragma unroll
  for (int s = 0; s < NB; ++s) c = amma<T>::mul(amma<T>::template load<L>(tile, it0, c0, s, lane), own.get(s), c);
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

// words (lower field row t even, ...) of the four staged rows 8 q + 4 (lane >> 5) + t of this lane's key: the four lanes of a key
// group each mix one row and hand it round; w[t] is the word that holds this key's field
__device__ __forceinline__ void quad_words(uint64_t mix, int lane, uint32_t (&w)[4]) {
  const int lo = (int)(uint32_t)mix, hi = (int)(uint32_t)(mix >> 32);
#define UBV_QUAD(t)                                                                           \
  {                                                                                           \
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp(lo, (t) * 0x55, 0xf, 0xf, true);   \
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp(hi, (t) * 0x55, 0xf, 0xf, true);   \
    w[t] = (lane & 2) ? b : a;                                                                \
  }
  UBV_QUAD(0) UBV_QUAD(1) UBV_QUAD(2) UBV_QUAD(3)
#undef UBV_QUAD
}

// keys j0 .. j0 + n - 1 that no row may see: past the end or padded (this lane's part; the wave's ballot is the tile's)
__device__ __forceinline__ bool key_hidden(const DiffAttnArgs& a, int b, int j0, int n, int lane) {
  const int j = j0 + lane;
  bool hide = j >= a.Nk;
  if (a.kpm != nullptr) hide = hide || a.kpm[(int64_t)b * a.Nk + min(j, a.Nk - 1)] != 0;
  return hide && lane < n;
}

// hides keys of a tile from the lane's row (query i of head h): `hid` bits of the 32 keys from j0, causal, the call's mask
template <int MODE> __device__ __forceinline__ void mask_tile(const DiffAttnArgs& a, af32x16_t (&x)[2], uint32_t hid, int b, int h, int i, int j0, float rscale,
                                          int lane) {
  const int half = 4 * (lane >> 5);
  if (hid != 0) {
    const uint32_t w = hid >> half;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (w & (1u << (8 * (e >> 2) + (e & 3)))) { x[0][e] = kNegInf; x[1][e] = kNegInf; }
  }
  if constexpr (MODE < kAttnCausal) return;
  if (MODE == kAttnCausal || a.causal) {
    const int lim = i + a.Nk - a.Nq - j0 - half;
    if (__any(lim < 31 - half)) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (8 * (e >> 2) + (e & 3) > lim) { x[0][e] = kNegInf; x[1][e] = kNegInf; }
    }
  }
  if (MODE != kAttnAny || a.mask_kind == 0) return;
  const int64_t o = b * a.ms[0] + h * a.ms[1] + i * a.ms[2] + (j0 + half) * a.ms[3];
  const bool whole = j0 + 32 <= a.Nk;
  const int last = a.Nk - 1 - j0 - half;               // (keys past the end, which `hid` hides, read the last one's)
  if (a.mask_kind == 1) {
    const uint8_t* m = (const uint8_t*)a.mask + o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w = 0;
      if (whole && a.ms[3] == 1) __builtin_memcpy(&w, m + 8 * q, 4);
      else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= (uint32_t)(m[min(8 * q + e, last) * a.ms[3]] != 0 ? 1u : 0u) << (8 * e);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (w & (0xffu << (8 * e))) { x[0][4 * q + e] = kNegInf; x[1][4 * q + e] = kNegInf; }
    }
  } else {
    const float* m = (const float*)a.mask + o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (whole && a.ms[3] == 1) __builtin_memcpy(w, m + 8 * q, 16);
      else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = m[min(8 * q + e, last) * a.ms[3]];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float bias = mask_raw(w[e], rscale);
        x[0][4 * q + e] = mask_add(x[0][4 * q + e], bias);
        x[1][4 * q + e] = mask_add(x[1][4 * q + e], bias);
      }
    }
  }
}

// Blocks go round-robin over the 8 XCDs: XCD x takes the x-th eighth of the tiles, so that the tiles of a head, which read the
// same keys (or rows), meet in one L2 (2 x 8 heads of 64 / 128, 4096 x 4096: forward 389 -> 376 us; causal, f16, 2 x 2 shared heads,
// 2047 x 2047: 153 -> 128).  Not in a padded batch, whose samples are unequal work, nor where splits of one tile share nothing.
// The grid is rounded up; a tile past the end has no work.
__device__ __forceinline__ int xcd_tile(const DiffAttnArgs& a) {
  return a.kpm != nullptr || (a.splits > 1 && !a.causal) ? blockIdx.x : xcd_remap(blockIdx.x, gridDim.x >> 3);
}
// block `id`'s own tile and which of its splits.  Causal tiles of a head are unequal: where an eighth is a part of a head (m parts),
// the parts take its tiles in turns, there and back, longest first; the last splits, short or empty, come last
__device__ __forceinline__ int2 tile_split(const DiffAttnArgs& a, int id) {
  if (!a.causal) return make_int2(id / a.splits, id % a.splits);
  const int heads = a.B * a.Hk, units = a.work / heads, tiles = units / a.splits, bh = id / units, u = id - bh * units;
  const int m = heads & 1 ? 8 : heads & 2 ? 4 : heads & 4 ? 2 : 1, q = units / m, r = units - q * m;
  const int longer = r * (q + 1);                      // (r parts have a unit more)
  const int part = u < longer ? u / (q + 1) : r + (u - longer) / max(q, 1);
  const int at = u < longer ? u - part * (q + 1) : u - longer - (part - r) * q;
  const int o = at * m + ((at & 1) && at < q ? m - 1 - part : part);
  return make_int2(bh * tiles + o % tiles, o / tiles);
}

// keys that some row of rb .. rb + n - 1 sees: [0, rows_end)
__device__ __forceinline__ int rows_end(const DiffAttnArgs& a, int rb, int n) {
  if (!a.causal) return a.Nk;
  const int last = (rb + n < a.R ? rb + n : a.R) - 1;
  const int imax = rb / a.Nq == last / a.Nq ? last % a.Nq : a.Nq - 1;
  const int end = imax + a.Nk - a.Nq + 1;
  return end < 0 ? 0 : end < a.Nk ? end : a.Nk;
}

// what forward and grad_q share: own = rows
struct RowWave {
  int wave, lane, wq, wk, b, hk, rb, r, h, i;
  bool ok;
  int64_t rowid;
  int kend;                            // keys that some row of the block sees: [0, kend)

  template <int WQ, int WK, bool MASK> __device__ __forceinline__ void init(const DiffAttnArgs& a, int tile) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    wq = wave / WK; wk = wave % WK;
    const int tiles = (a.R + 32 * WQ - 1) / (32 * WQ), bh = tile / tiles;
    int at = tile - bh * tiles;
    if (MASK && a.causal) at = tiles - 1 - at;         // the rows that see most keys first: no long block at the end
    rb = at * 32 * WQ;
    b = bh / a.Hk; hk = bh - b * a.Hk;
    r = rb + 32 * wq + (lane & 31);
    ok = r < a.R;
    const int rc = ok ? r : a.R - 1, g = rc / a.Nq;
    h = hk * a.G + g; i = rc - g * a.Nq;
    rowid = ((int64_t)b * a.H + hk * a.G) * a.Nq + rc;
    kend = MASK ? rows_end(a, rb, 32 * WQ) : a.Nk;
  }
  // this wave's 32 rows among those of all heads
  __device__ __forceinline__ int64_t tile32(const DiffAttnArgs& a) const {
    return ((int64_t)b * a.Hk + hk) * ((a.R + 31) / 32) + rb / 32 + wq;
  }
};

// the stream of staged key tiles: f(tile, it0, hid of its 32 keys, j0) for every 32 keys that are not all hidden
template <typename T, int DH, int DV, bool SHARED, typename F>
__device__ __forceinline__ void key_tiles(const DiffAttnArgs& a, const RowWave& w, int col, int t0, int t1, char* smem, F&& f) {
  using S = AttnTile<T, DH, DV>;
  using P = AttnPlan<T, DH, DV, SHARED>;
  constexpr int N = P::N, STEP = P::WK;
  constexpr uint64_t ALL = N == 64 ? ~0ull : 0xffffffffull;
  const int st = SHARED ? threadIdx.x : w.lane;
  AttnStage<T, DH, DV, N, P::LT, P::PREF> sg;
  const uint32_t xrow = (uint32_t)(a.ks[1] * elem<T>::kBytes), yrow = (uint32_t)(a.vs[1] * elem<T>::kBytes);
  sg.init(st, xrow, (uint32_t)(a.ks[3] * elem<T>::kBytes), yrow, a.Dh, a.Dv - col);
  const char* kb = (const char*)a.k + (w.b * a.ks[0] + w.hk * a.ks[2]) * elem<T>::kBytes;
  const char* vb = (const char*)a.v + (w.b * a.vs[0] + w.hk * a.vs[2] + col) * elem<T>::kBytes;
  int t = t0 + w.wk;
  if (t >= t1) return;                                       // (private waves only: no barrier inside)
  auto load = [&](int tt, uint64_t hid, char* lds) {
    const int64_t j0 = (int64_t)tt * N;
    if (hid == ALL) return;
    if constexpr (P::PREF) sg.load(kb + j0 * xrow, xrow, vb + j0 * yrow, yrow, hid, st);
    else sg.through(kb + j0 * xrow, xrow, vb + j0 * yrow, yrow, hid, lds, st);
  };
  uint64_t hid = __ballot(key_hidden(a, w.b, t * N, N, w.lane));
  char* const buf = smem + (SHARED ? 0 : w.wk * S::bytes(N));
  load(t, hid, buf);
  if constexpr (P::PREF) sg.store(buf, st);
  tile_ready<SHARED>();
  bool nb = t + STEP < t1 && key_hidden(a, w.b, (t + STEP) * N, N, w.lane);
  int cur = 0;
#pragma unroll 1
  for (; t < t1; t += STEP) {
    const bool more = t + STEP < t1;
    const uint64_t nhid = __ballot(nb);
    if (P::PREF && more) load(t + STEP, nhid, nullptr);
    nb = t + 2 * STEP < t1 && key_hidden(a, w.b, (t + 2 * STEP) * N, N, w.lane);
    const char* tile = SHARED ? smem + cur * S::bytes(N) : buf;
#pragma unroll 1
    for (int it0 = 0; it0 < N; it0 += 32) {
      const uint32_t h32 = (uint32_t)(hid >> it0);
      if (h32 != 0xffffffffu && t * N + it0 < w.kend) f(tile, it0, h32, t * N + it0);
    }
    if (more) {
      if constexpr (SHARED) cur ^= 1;
      else tile_ready<false>();
      if constexpr (P::PREF) sg.store(SHARED ? smem + cur * S::bytes(N) : buf, st);
      else load(t + STEP, nhid, buf);
      tile_ready<SHARED>();
    }
    hid = nhid;
  }
}

// 16 floats of a lane as 4 pieces, `step` floats apart
__device__ __forceinline__ void put_block(float* at, const af32x16_t& v, int step) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<float4*>(at + q * step) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

// ---- forward ------------------------------------------------------------------------------------------------------------------
template <typename T, int DV> struct FwdState {
  static constexpr int VO = DV / 32;
  af32x16_t acc[2][VO];
  float top[2], l[2];              // the row's reference (raw score) and this lane half's sum beside it

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      top[m] = kNegInf; l[m] = 0.0f;
#pragma unroll
      for (int d = 0; d < VO; ++d) acc[m][d] = af32x16_t{0.0f};
    }
  }
  __device__ __forceinline__ void scale(int m, float f) {
    l[m] *= f;
#pragma unroll
    for (int d = 0; d < VO; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[m][d][e] *= f;
  }
  static constexpr int FLOATS = 4 + DV;
  __device__ __forceinline__ void put(float* slot) const {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      slot[(2 * m) * 64] = top[m]; slot[(2 * m + 1) * 64] = l[m];
#pragma unroll
      for (int d = 0; d < VO; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) slot[(4 + (m * VO + d) * 16 + e) * 64] = acc[m][d][e];
    }
  }
  // the same for the splits' workspace, pieces of 4 floats.  Rows by the wave: piece by piece, 1 KB each; few rows: a lane's in one
  // stretch (only the lanes of rows are written: few bytes)
  static __device__ __forceinline__ int64_t lane_at(bool few, int lane) { return few ? lane * FLOATS : lane * 4; }
  static __device__ __forceinline__ int piece(bool few) { return few ? 4 : 256; }
  __device__ __forceinline__ void put_row(float* at, int step) const {
    *reinterpret_cast<float4*>(at) = make_float4(top[0], l[0], top[1], l[1]);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int d = 0; d < VO; ++d) put_block(at + (1 + (m * VO + d) * 4) * step, acc[m][d], step);
  }
  // joins what another wave put for the same rows
  __device__ __forceinline__ void join(const float* slot, float c) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float to = slot[(2 * m) * 64], t = fmaxf(top[m], to);
      const float f0 = top[m] == kNegInf ? 0.0f : aexp2((top[m] - t) * c), f1 = to == kNegInf ? 0.0f : aexp2((to - t) * c);
      scale(m, f0);
      l[m] = fmaf(slot[(2 * m + 1) * 64], f1, l[m]);
      top[m] = t;
#pragma unroll
      for (int d = 0; d < VO; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[m][d][e] = fmaf(slot[(4 + (m * VO + d) * 16 + e) * 64], f1, acc[m][d][e]);
    }
  }
};

// the rows' outputs and what the backward pass wants, from the joined state
template <typename T, int DV>
__device__ __forceinline__ void fwd_finish(const DiffAttnArgs& a, const FwdState<T, DV>& s, const RowWave& w, int col, float c) {
  if (!w.ok) return;
  const bool fm = a.mask_kind == 2;
  const int64_t rows = (int64_t)a.B * a.H * a.Nq;
  const float lam = a.lam[w.h];
  float inv[2], st[4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float l = half_sum(s.l[m]);
    const bool dead = l == 0.0f;
    inv[m] = dead ? 0.0f : a.up / l;
    st[2 * m] = dead ? 0.0f : fm ? s.top[m] : s.top[m] * c - kProbShift<T>;
    st[2 * m + 1] = dead ? -kNegInf : fm ? log2f(l) - kProbShift<T> : log2f(l);
  }
  if (a.stat != nullptr && w.lane < 32 && col == 0) a.stat[w.rowid] = make_float4(st[0], st[1], st[2], st[3]);
  T* orow = (T*)a.out + (((int64_t)w.b * a.Nq + w.i) * a.H + w.h) * a.Dv;
#pragma unroll
  for (int d = 0; d < DV / 32; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dv = col + 32 * d + tile_item(4 * q, w.lane);
      float o1[4], o2[4], o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o1[e] = s.acc[0][d][4 * q + e] * inv[0];
        o2[e] = s.acc[1][d][4 * q + e] * inv[1];
        o[e] = fmaf(-lam, o2[e], o1[e]);
      }
      store_quad<T>(orow, dv, a.Dv, o);
      if (a.o != nullptr) {
        store_quad<float>(a.o + w.rowid * a.Dv, dv, a.Dv, o1);
        store_quad<float>(a.o + (rows + w.rowid) * a.Dv, dv, a.Dv, o2);
      }
    }
}

// One pass over the keys with a running reference and sum for each map.  Per pair and map: Dh + Dv multiply-adds on the matrix cores
// against one exponential (a quarter of the VALU's rate), a fma, a maximum, an addition and a rounding.  A wave's products and its
// softmax follow one another, and one or two waves a SIMD do not fill the gaps: at 32 / 64, 10 000 x 10 000, the VALU issues 52 % of
// the time and the matrix cores are busy 23 %; at 64 / 128, 4096 x 4096, 46 and 22 %.  4 heads of 32 / 64, 10 000 x 10 000 bf16: 267 us
// (575 TFLOP/s); 2 x 8 heads of 64 / 128, 4096 x 4096: 380 us (542 TFLOP/s); one query, 8 x 4 heads of 32 / 64, 40 000 keys ragged:
// 54 to 61 us (4.2 to 4.7 TB/s, bound by memory).
template <typename T, int DH, int DV, bool SHARED, int MODE>
__global__ __launch_bounds__((AttnPlan<T, DH, DV, SHARED>::NT), (AttnPlan<T, DH, DV, SHARED>::MINW)) void diff_attn_fwd_kernel(
    const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  using P = AttnPlan<T, DH, DV, SHARED>;
  using M = amma<T>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int id = xcd_tile(a);
  if (id >= a.work) return;
  const int2 cut = tile_split(a, id);
  const int split = cut.y, tile = cut.x / a.halves, col = (cut.x - tile * a.halves) * DV;
  RowWave w;
  w.init<P::WQ, P::WK, (MODE >= kAttnCausal)>(a, tile);
  const int tn = (w.kend + P::N - 1) / P::N, t0 = split * a.chunk;
  if (split > 0 && t0 >= tn) return;                   // (an own tile that sees less has fewer splits)
  OwnRow<T, S::KB, S::KEEP> qf[2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
    qf[m].init((const T*)a.q + w.b * a.qs[0] + w.i * a.qs[1] + w.h * a.qs[2] + m * a.qs[3], w.ok, a.Dh, w.lane);
  const float c = a.scale * kLog2e, rscale = 1.0f / a.scale, grow = 6.0f / c;
  constexpr bool MASK = MODE >= kAttnCausal;
  const bool fm = MODE == kAttnAny && a.mask_kind == 2, drop = (MODE == kAttnDrop || MODE == kAttnAny) && a.t16 != 0;
  const uint32_t t32 = a.t16 << 16;
  const uint64_t zrow = attn_seed(a.seed, a.seed_dev) + (uint64_t)(w.rowid * a.n4) + (w.lane >> 5);
  FwdState<T, DV> s;
  s.init();
  float mu[2] = {0.0f, 0.0f};
  key_tiles<T, DH, DV, SHARED>(a, w, col, t0, min(tn, t0 + a.chunk), smem,
                               [&](const char* kt, int it0, uint32_t hid, int j0) {
    af32x16_t x[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) x[m] = tile_dot<T, S::KB, S::LX, S::KEEP>(kt, it0, m * S::LX / 2, qf[m], w.lane);
    if (hid != 0 || MASK) mask_tile<MODE>(a, x, hid, w.b, w.h, w.i, j0, rscale, w.lane);
    float p[2][16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float t = x[m][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) t = fmaxf(t, x[m][e]);
      t = half_max(t);
      // the reference moves, and what is summed so far shrinks, only where a score is over it by 2^6: the sums have room for
      // that, and after a row's first tiles this (wave-uniform) branch is hardly taken
      if (__any(t > s.top[m] + grow)) {
        t = fmaxf(t, s.top[m]);
        s.scale(m, s.top[m] == kNegInf ? 0.0f : aexp2((s.top[m] - t) * c));
        s.top[m] = t;
        mu[m] = t == kNegInf ? 0.0f : fm ? t : t * c - kProbShift<T>;
      }
      if (fm) {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[m][e] = aexp2(fmaf(x[m][e] - mu[m], c, kProbShift<T>));
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[m][e] = aexp2(fmaf(x[m][e], c, -mu[m]));
      }
      float t0 = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) t0 += p[m][e];
      s.l[m] += t0;
    }
    if (drop) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint64_t mix = attn_mix(zrow + (uint64_t)((j0 >> 2) + 2 * q));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool keep = attn_keep((uint32_t)(e < 2 ? mix : mix >> 32), e & 1, t32);
#pragma unroll
          for (int m = 0; m < 2; ++m) p[m][4 * q + e] = keep ? p[m][4 * q + e] : 0.0f;
        }
      }
    }
    const char* vt = kt + S::xbytes(P::N);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const typename M::frag f0 = M::pack(p[0] + 8 * st), f1 = M::pack(p[1] + 8 * st);
#pragma unroll
      for (int d = 0; d < S::VO; ++d) {
        const typename M::frag vf = M::template load_tr<S::LY>(vt, it0 + 16 * st, 0, d, w.lane);
        s.acc[0][d] = M::mul(vf, f0, s.acc[0][d]);
        s.acc[1][d] = M::mul(vf, f1, s.acc[1][d]);
      }
    }
  });
  if constexpr (!SHARED) {                            // join the waves that walked other keys of the same rows
    float* slots = reinterpret_cast<float*>(smem);
#pragma unroll 1
    for (int half = P::WK / 2; half >= 1; half >>= 1) {
      __syncthreads();
      float* slot = slots + (w.wk % half) * (s.FLOATS * 64) + w.lane;
      if (w.wk >= half && w.wk < 2 * half) s.put(slot);
      __syncthreads();
      if (w.wk < half) s.join(slot, c);
    }
    if (w.wk != 0) return;
  }
  if (tn > a.chunk) {
    const bool few = a.R < 32;
    if (w.ok) s.put_row(a.part + ((w.tile32(a) * a.halves + col / DV) * a.splits + split) * 64 * s.FLOATS + s.lane_at(few, w.lane), s.piece(few));
    return;
  }
  fwd_finish<T, DV>(a, s, w, col, c);
}

// Joins the splits of 32 rows: one wave a tile and 32 columns of a half
template <typename T, int DV>
__global__ __launch_bounds__(64) void diff_attn_join_rows_kernel(const DiffAttnArgs a) {
  constexpr int VO = DV / 32, FLOATS = FwdState<T, DV>::FLOATS;
  const int part = blockIdx.x / VO, d = blockIdx.x - part * VO, tile = part / a.halves, half = part - tile * a.halves;
  RowWave w;
  w.init<1, 1, true>(a, tile);
  const int parts = ((rows_end(a, w.rb / a.own * a.own, a.own) + a.n - 1) / a.n + a.chunk - 1) / a.chunk;
  if (!w.ok || parts <= 1) return;                     // (written by its one block)
  const float c = a.scale * kLog2e;
  const float* at = a.part + (w.tile32(a) * a.halves + half) * a.splits * 64 * FLOATS + w.lane * 4;
  FwdState<T, 32> s;
  s.init();
#pragma unroll 2
  for (int p = 0; p < parts; ++p) {
    const float* f = at + (int64_t)p * 64 * FLOATS;
    const float4 r = *reinterpret_cast<const float4*>(f);
    const float to[2] = {r.x, r.z}, lo[2] = {r.y, r.w};
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float t = fmaxf(s.top[m], to[m]);
      const float f0 = s.top[m] == kNegInf ? 0.0f : aexp2((s.top[m] - t) * c), f1 = to[m] == kNegInf ? 0.0f : aexp2((to[m] - t) * c);
      s.scale(m, f0);
      s.l[m] = fmaf(lo[m], f1, s.l[m]);
      s.top[m] = t;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(f + (1 + (m * VO + d) * 4 + q) * 256);
        s.acc[m][0][4 * q] = fmaf(v.x, f1, s.acc[m][0][4 * q]);
        s.acc[m][0][4 * q + 1] = fmaf(v.y, f1, s.acc[m][0][4 * q + 1]);
        s.acc[m][0][4 * q + 2] = fmaf(v.z, f1, s.acc[m][0][4 * q + 2]);
        s.acc[m][0][4 * q + 3] = fmaf(v.w, f1, s.acc[m][0][4 * q + 3]);
      }
    }
  }
  fwd_finish<T, 32>(a, s, w, half * DV + 32 * d, c);
}

// Joins the splits of few rows (under 32 a group): one block a row (and column half), a thread an element of one map's product.  Weights of the splits
// first (one exponential each, in LDS), then the products' sum in split order.
template <typename T, int DV>
__global__ __launch_bounds__(256) void diff_attn_join_kernel(const DiffAttnArgs a) {
  constexpr int FLOATS = FwdState<T, DV>::FLOATS, VO = DV / 32;
  __shared__ float wt[2][kAttnSplits], red[4][4], o2s[128];
  const float c = a.scale * kLog2e;
  const int part = blockIdx.x, half = part % a.halves, row = part / a.halves, bh = row / a.R, r = row - bh * a.R;
  const int parts = ((rows_end(a, r / a.own * a.own, a.own) + a.n - 1) / a.n + a.chunk - 1) / a.chunk;
  if (parts <= 1) return;                              // (written by its one block)
  const int lane = r % 32, col = half * DV;
  const int64_t tile = (int64_t)bh * ((a.R + 31) / 32) + r / 32;
  const int b = bh / a.Hk, hk = bh - b * a.Hk, h = hk * a.G + r / a.Nq, i = r % a.Nq;
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, rowid = ((int64_t)b * a.H + h) * a.Nq + i;
  const float* p = a.part + ((tile * a.halves + half) * a.splits * 64 + lane) * FLOATS;      // split n, lane half: + (64 n + 32 s) FLOATS
  const int t = threadIdx.x, wave = t >> 6;
  auto block = [&](float x, float y, bool is_max, float& ox, float& oy) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const float u = __shfl_xor(x, m, 64), v = __shfl_xor(y, m, 64);
      x = is_max ? fmaxf(x, u) : x + u;
      y = is_max ? fmaxf(y, v) : y + v;
    }
    __syncthreads();
    if ((t & 63) == 0) { red[wave][0] = x; red[wave][1] = y; }
    __syncthreads();
    ox = red[0][0]; oy = red[0][1];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      ox = is_max ? fmaxf(ox, red[w][0]) : ox + red[w][0];
      oy = is_max ? fmaxf(oy, red[w][1]) : oy + red[w][1];
    }
  };
  float m1 = kNegInf, m2 = kNegInf, top[2], l[2], l1 = 0.0f, l2 = 0.0f;
  for (int n = t; n < parts; n += 256) {
    const float4 s = *reinterpret_cast<const float4*>(p + (int64_t)64 * n * FLOATS);
    m1 = fmaxf(m1, s.x); m2 = fmaxf(m2, s.z);
  }
  block(m1, m2, true, top[0], top[1]);
  for (int n = t; n < parts; n += 256) {
    const float4 s = *reinterpret_cast<const float4*>(p + (int64_t)64 * n * FLOATS);
    const float4 s2 = *reinterpret_cast<const float4*>(p + (int64_t)(64 * n + 32) * FLOATS);
    wt[0][n] = s.x == kNegInf ? 0.0f : aexp2((s.x - top[0]) * c);
    wt[1][n] = s.z == kNegInf ? 0.0f : aexp2((s.z - top[1]) * c);
    l1 = fmaf(s.y + s2.y, wt[0][n], l1);
    l2 = fmaf(s.w + s2.w, wt[1][n], l2);
  }
  block(l1, l2, false, l[0], l[1]);                  // (its barriers also order the weights)
  const int m = t >> 7, d = t & 127;
  float o = 0.0f;
  if (d < DV) {
    const float* e = p + (int64_t)(32 * ((d >> 2) & 1)) * FLOATS + 4 + (m * VO + (d >> 5)) * 16 + 4 * ((d >> 3) & 3) + (d & 3);
#pragma unroll 8
    for (int n = 0; n < parts; ++n) o = fmaf(e[(int64_t)64 * n * FLOATS], wt[m][n], o);
  }
  const bool fm = a.mask_kind == 2, dead = l[m] == 0.0f;
  o *= dead ? 0.0f : a.up / l[m];
  if (m == 1) o2s[d] = o;
  __syncthreads();
  const bool in = d < DV && col + d < a.Dv;
  if (a.o != nullptr && in) a.o[(m * rows + rowid) * a.Dv + col + d] = o;
  if (m == 0 && in)
    ((T*)a.out)[(((int64_t)b * a.Nq + i) * a.H + h) * a.Dv + col + d] = elem<T>::from_float(fmaf(-a.lam[h], o2s[d], o));
  if (a.stat != nullptr && col == 0 && d == 0)
    reinterpret_cast<float2*>(a.stat + rowid)[m] =
        make_float2(dead ? 0.0f : fm ? top[m] : top[m] * c - kProbShift<T>, dead ? -kNegInf : fm ? log2f(l[m]) - kProbShift<T> : log2f(l[m]));
}

// ---- backward: del_m = grad_out . o_m of a row by 16 lanes (t: this lane's number); all of them get the sums --------------------
template <typename T>
__device__ __forceinline__ float2 row_del(const DiffAttnArgs& a, int64_t rowid, int64_t b, int h, int i, int t) {
  const int64_t rows = (int64_t)a.B * a.H * a.Nq;
  const T* g = (const T*)a.go + b * a.gs[0] + i * a.gs[1] + h * a.gs[2];
  const float *o1 = a.o + rowid * a.Dv, *o2 = a.o + (rows + rowid) * a.Dv;
  float s1 = 0.0f, s2 = 0.0f;
  for (int d = t; d < a.Dv; d += 16) {
    const float gv = elem<T>::to_float(g[d]);
    s1 = fmaf(gv, o1[d], s1);
    s2 = fmaf(gv, o2[d], s2);
  }
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) { s1 += __shfl_xor(s1, m, 64); s2 += __shfl_xor(s2, m, 64); }
  return make_float2(s1, s2);
}
// the row's numbers as row_probability takes them
__device__ __forceinline__ void row_stats(const DiffAttnArgs& a, bool fm, int64_t rowid, float2 del, float4& rw, float2& rl) {
  const float4 st = a.stat[rowid];
  rw = fm ? make_float4(st.x, st.z, del.x, del.y) : make_float4(st.x + st.y, st.z + st.w, del.x, del.y);
  rl = fm ? make_float2(st.y, st.w) : make_float2(0.0f, 0.0f);
}
// what grad_q's pass leaves for grad_k's, by itself where that pass does not run
template <typename T>
__global__ __launch_bounds__(256) void diff_attn_del_kernel(const DiffAttnArgs a) {
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, rowid = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int64_t rr = rowid < rows ? rowid : rows - 1;
  const float2 del = row_del<T>(a, rr, rr / a.Nq / a.H, (int)(rr / a.Nq % a.H), (int)(rr % a.Nq), threadIdx.x & 15);
  if ((threadIdx.x & 15) == 0 && rowid < rows) {
    float4 rw;
    float2 rl;
    row_stats(a, a.mask_kind == 2, rr, del, rw, rl);
    a.row[rr] = rw;
    if (a.mask_kind == 2) a.rowl[rr] = rl;
  }
}

// sums over the waves of a private block; the result is in wave 0
template <int WK, int NB>
__device__ __forceinline__ void join_waves(af32x16_t* const (&acc)[NB], float* slots, int wk, int lane) {
#pragma unroll 1
  for (int half = WK / 2; half >= 1; half >>= 1) {
    __syncthreads();
    float* slot = slots + (wk % half) * (NB * 16 * 64) + lane;
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

// sum over the splits of a lane's 16 floats, in split order
__device__ __forceinline__ af32x16_t sum_block(const float* at, int splits, int64_t step) {
  af32x16_t v = {0.0f};
#pragma unroll 2
  for (int n = 0; n < splits; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(at + n * step + 256 * q);
      v[4 * q] += f.x; v[4 * q + 1] += f.y; v[4 * q + 2] += f.z; v[4 * q + 3] += f.w;
    }
  return v;
}
template <typename T> __device__ __forceinline__ void store_block(T* row, int d0, int D, const af32x16_t& v, float f, int lane) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = f != 0.0f ? v[4 * q + e] * f : 0.0f;
    store_quad<T>(row, d0 + tile_item(4 * q, lane), D, o);
  }
}
// block n of a row's gradient: map n / KO, columns 32 (n % KO) ..
template <typename T, int KO>
__device__ __forceinline__ void store_gq(const DiffAttnArgs& a, const RowWave& w, int n, const af32x16_t& v) {
  // a single key has probability 1 whatever its score: its gradient is zero, not the rounding of G - del
  const float one = a.Nk > 1 ? a.scale : 0.0f;
  store_block<T>((T*)a.gq + ((((int64_t)w.b * a.Nq + w.i) * a.H + w.h) * 2 + n / KO) * a.Dh, 32 * (n % KO), a.Dh, v,
                 n < KO ? one : -a.lam[w.h] * one, w.lane);
}
// block n of a key's gradients: grad_k's 2 KO, then grad_v's; `ok`: a key that is seen; ls: lam_scale of its head
template <typename T, int KO>
__device__ __forceinline__ void store_gkv(const DiffAttnArgs& a, int b, int hk, int j, bool ok, int n, const af32x16_t& v, float ls, int lane) {
  const int64_t row = ((int64_t)b * a.Nk + j) * a.Hk + hk;
  if (n < 2 * KO)
    store_block<T>((T*)a.gk + (row * 2 + n / KO) * a.Dh, 32 * (n % KO), a.Dh, v, !ok || a.Nk <= 1 ? 0.0f : n < KO ? a.scale : a.scale / ls, lane);
  else
    store_block<T>((T*)a.gv + row * a.Dv, 32 * (n - 2 * KO), a.Dv, v, ok ? a.up / (kProbScale<T> * ls) : 0.0f, lane);
}

// ---- backward: grad_q and the rows' parts of grad_lam; own = rows, staged = keys -----------------------------------------------
// dq_m = scale sum_j dS_m k_m,  dS_1 = A_1 o (G - del_1),  dS_2 = -lam A_2 o (G - del_2),  G = D o (grad_out v^T);  A from the row's
// statistics.  Bound as the forward pass: 10 000 x 10 000, 4 heads of 32 / 64 bf16 340 us (VALU 60 %, matrix
// cores 25 %; the scores computed again, dS in two operands).
template <typename T, int DH, int DV, bool SHARED, int MODE>
__global__ __launch_bounds__((AttnPlan<T, DH, DV, SHARED>::NT), (AttnPlan<T, DH, DV, SHARED>::MINW)) void diff_attn_bwd_q_kernel(
    const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  using P = AttnPlan<T, DH, DV, SHARED>;
  using M = amma<T>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int id = xcd_tile(a);
  if (id >= a.work) return;
  const int2 cut = tile_split(a, id);
  const int tile = cut.x, split = cut.y;
  RowWave w;
  w.init<P::WQ, P::WK, (MODE >= kAttnCausal)>(a, tile);
  const int tn = (w.kend + P::N - 1) / P::N, t0 = split * a.chunk;
  if (split > 0 && t0 >= tn) return;
  constexpr bool MASK = MODE >= kAttnCausal;
  const bool fm = MODE == kAttnAny && a.mask_kind == 2, drop = (MODE == kAttnDrop || MODE == kAttnAny) && a.t16 != 0;
  OwnRow<T, S::KB, S::KEEP> qf[2];
  OwnRow<T, S::VB, S::KEEP> gf;
#pragma unroll
  for (int m = 0; m < 2; ++m)
    qf[m].init((const T*)a.q + w.b * a.qs[0] + w.i * a.qs[1] + w.h * a.qs[2] + m * a.qs[3], w.ok, a.Dh, w.lane);
  gf.init((const T*)a.go + w.b * a.gs[0] + w.i * a.gs[1] + w.h * a.gs[2], w.ok, a.Dv, w.lane);
  // del of the own rows, 16 lanes a row, the waves of the same rows taking turns; kept for the pass of grad_k
  __shared__ float2 dels[P::WQ][32];
  for (int n = 4 * w.wk + (w.lane >> 4); n < 32; n += 4 * P::WK) {
    const int r = min(w.rb + 32 * w.wq + n, a.R - 1), g = r / a.Nq;
    const float2 del = row_del<T>(a, ((int64_t)w.b * a.H + w.hk * a.G) * a.Nq + r, w.b, w.hk * a.G + g, r - g * a.Nq, w.lane & 15);
    if ((w.lane & 15) == 0) dels[w.wq][n] = del;
  }
  __syncthreads();
  float4 rw;
  float2 rl;
  row_stats(a, fm, w.rowid, dels[w.wq][w.lane & 31], rw, rl);
  if (w.ok && w.wk == 0 && split == 0 && w.lane < 32) {
    a.row[w.rowid] = rw;
    if (fm) a.rowl[w.rowid] = rl;
  }
  const float c = a.scale * kLog2e, rscale = 1.0f / a.scale;
  const uint32_t t32 = a.t16 << 16;
  const uint64_t zrow = attn_seed(a.seed, a.seed_dev) + (uint64_t)(w.rowid * a.n4) + (w.lane >> 5);
  af32x16_t acc[2][S::KO];
  float dl = 0.0f;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int d = 0; d < S::KO; ++d) acc[m][d] = af32x16_t{0.0f};
  key_tiles<T, DH, DV, SHARED>(a, w, 0, t0, min(tn, t0 + a.chunk), smem, [&](const char* kt, int it0, uint32_t hid, int j0) {
    af32x16_t x[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) x[m] = tile_dot<T, S::KB, S::LX, S::KEEP>(kt, it0, m * S::LX / 2, qf[m], w.lane);
    af32x16_t g = tile_dot<T, S::VB, S::LY, S::KEEP>(kt + S::xbytes(P::N), it0, 0, gf, w.lane);
    if (hid != 0 || MASK) mask_tile<MODE>(a, x, hid, w.b, w.h, w.i, j0, rscale, w.lane);
    if (drop) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint64_t mix = attn_mix(zrow + (uint64_t)((j0 >> 2) + 2 * q));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          g[4 * q + e] = attn_keep((uint32_t)(e < 2 ? mix : mix >> 32), e & 1, t32) ? g[4 * q + e] * a.up : 0.0f;
      }
    }
    float dt = 0.0f;                                  // (the tile's own sum first: 16 times fewer additions to the long one)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p1 = row_probability(fm, x[0][e], c, rw.x, rl.x), p2 = row_probability(fm, x[1][e], c, rw.y, rl.y);
      dt = fmaf(p2, g[e], dt);
      x[0][e] = p1 * (g[e] - rw.z);
      x[1][e] = p2 * (g[e] - rw.w);
    }
    dl += dt;
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float ds[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) ds[e] = x[m][8 * st + e];
        typename M::frag f, rest;
        M::split(ds, f, rest);
#pragma unroll
        for (int d = 0; d < S::KO; ++d) {
          const typename M::frag kf = M::template load_tr<S::LX>(kt, it0 + 16 * st, m * S::LX / 2, d, w.lane);
          acc[m][d] = M::mul(kf, f, acc[m][d]);
          if constexpr (M::SPLIT) acc[m][d] = M::mul(kf, rest, acc[m][d]);
        }
      }
  });
  if constexpr (!SHARED) {
    af32x16_t dlv = {dl};
    af32x16_t* ptr[2 * S::KO + 1];
#pragma unroll
    for (int d = 0; d < S::KO; ++d) { ptr[d] = &acc[0][d]; ptr[S::KO + d] = &acc[1][d]; }
    ptr[2 * S::KO] = &dlv;
    join_waves<P::WK>(ptr, reinterpret_cast<float*>(smem), w.wk, w.lane);
    if (w.wk != 0) return;
    dl = dlv[0];
  }
  if (!w.ok) return;
  if (tn > a.chunk) {
    float* at = a.part + (w.tile32(a) * a.splits + split) * 64 * S::QFLOATS + w.lane * 4;
#pragma unroll
    for (int n = 0; n < 2 * S::KO; ++n) put_block(at + 1024 * n, acc[n / S::KO][n % S::KO], 256);
    at[2048 * S::KO] = dl;
    return;
  }
  dl = half_sum(dl);
  if (w.lane < 32) a.dlrow[w.rowid] = -dl;
  if (a.gq == nullptr) return;
#pragma unroll
  for (int n = 0; n < 2 * S::KO; ++n) store_gq<T, S::KO>(a, w, n, acc[n / S::KO][n % S::KO]);
}

// grad_lam[h] = sum over the batch and the queries, one block a head, fixed order (256 threads: 11 us for 10 000 rows)
__global__ __launch_bounds__(1024) static void diff_attn_lam_kernel(const float* __restrict__ dlrow, float* __restrict__ glam, int B, int H,
                                                                    int Nq) {
  __shared__ float red[16];
  const int h = blockIdx.x;
  float s = 0.0f;
  for (int b = 0; b < B; ++b) {
    const float* row = dlrow + ((int64_t)b * H + h) * Nq;
#pragma unroll 8
    for (int i = threadIdx.x; i < Nq; i += 1024) s += row[i];
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x < 16) {
    s = red[threadIdx.x];
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
    if (threadIdx.x == 0) glam[h] = s;
  }
}

// ---- backward: grad_k and grad_v; own = keys, staged = the rows of every head that shares them ----------------------------------
// A tile of rows stays inside one head (its rows are one stretch of queries), heads one after the other.
// dk_m = scale sum_i dS_m q_m,  dv = sum_i (D o (A_1 - lam A_2)) grad_out.  10 000 x 10 000, 4 heads of 32 / 64 bf16: 513 to 590 us
// by card and clock; bound as the others (VALU 49 %, matrix cores 19 %) with LDS reads on top (the rows' statistics, 4 floats each).
// PART 0: both gradients in one pass; 1: grad_k, 2: grad_v by a pass of its own, where the accumulators of both (2 DH + DV
// floats a lane's item pair) would not fit the register file (the scores are computed twice: less than spilling costs).
template <typename T, int DH, int DV, bool SHARED, int MODE, int PART>
__global__ __launch_bounds__((AttnPlan<T, DH, DV, SHARED>::NT), (AttnPlan<T, DH, DV, SHARED>::MINW)) void diff_attn_bwd_kv_kernel(
    const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  using P = AttnPlan<T, DH, DV, SHARED>;
  using M = amma<T>;
  constexpr int N = P::N;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, wq = wave / P::WK, wk = wave % P::WK;
  const int id = xcd_tile(a);
  if (id >= a.work) return;
  const int2 cut = tile_split(a, id);
  const int tile = cut.x, split = cut.y;
  const int tiles = (a.Nk + 32 * P::WQ - 1) / (32 * P::WQ), bh = tile / tiles, jb = (tile - bh * tiles) * 32 * P::WQ;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const int j = jb + 32 * wq + (lane & 31);
  // a hidden key's column is computed from zeros and its gradients are stored as zeros: no masking needed for it
  const bool in = j < a.Nk, ok = in && !(a.kpm != nullptr && a.kpm[(int64_t)b * a.Nk + (in ? j : 0)]);
  const int jc = in ? j : a.Nk - 1, off = a.Nk - a.Nq;
  constexpr bool MASK = MODE >= kAttnCausal;
  const bool fm = MODE == kAttnAny && a.mask_kind == 2, drop = (MODE == kAttnDrop || MODE == kAttnAny) && a.t16 != 0;

  OwnRow<T, S::KB, S::KEEP> kf[2];
  OwnRow<T, S::VB, S::KEEP> vf;
#pragma unroll
  for (int m = 0; m < 2; ++m)
    kf[m].init((const T*)a.k + b * a.ks[0] + jc * a.ks[1] + hk * a.ks[2] + m * a.ks[3], ok, a.Dh, lane);
  if constexpr (PART != 2) vf.init((const T*)a.v + b * a.vs[0] + jc * a.vs[1] + hk * a.vs[2], ok, a.Dv, lane);
  af32x16_t ak[2][S::KO], av[S::VO];
#pragma unroll
  for (int d = 0; d < S::KO; ++d) { ak[0][d] = af32x16_t{0.0f}; ak[1][d] = af32x16_t{0.0f}; }
#pragma unroll
  for (int d = 0; d < S::VO; ++d) av[d] = af32x16_t{0.0f};
  const float c = a.scale * kLog2e, rscale = 1.0f / a.scale, lt = lam_top<T>(a.lam, hk, a.G, lane);
  const uint32_t t32 = a.t16 << 16;
  const uint64_t zseed = attn_seed(a.seed, a.seed_dev) + (uint64_t)(j >> 2);

  // tiles of a head from the first whose rows may see a key of the block
  const int first = MASK && a.causal ? max(0, jb - off) / N : 0, per = max(0, (a.Nq + N - 1) / N - first);
  const int all = per * a.G, begin = split * a.chunk, total = min(all, begin + a.chunk);
  if (split > 0 && begin >= all) return;
  const int st = SHARED ? threadIdx.x : lane;
  AttnStage<T, DH, DV, N, P::LT, P::PREF> sg;
  const uint32_t xrow = (uint32_t)(a.qs[1] * elem<T>::kBytes), yrow = (uint32_t)(a.gs[1] * elem<T>::kBytes);
  sg.init(st, xrow, (uint32_t)(a.qs[3] * elem<T>::kBytes), yrow, a.Dh, a.Dv);
  const int sr = st % N;
  float4 srow;
  float2 srowl = make_float2(0.0f, 0.0f);
  auto load = [&](int t, char* lds) {
    const int g = t / per, i0 = (first + t - g * per) * N, h = hk * a.G + g, left = a.Nq - i0;
    const char* xb = (const char*)a.q + (b * a.qs[0] + (int64_t)i0 * a.qs[1] + h * a.qs[2]) * elem<T>::kBytes;
    const char* yb = (const char*)a.go + (b * a.gs[0] + (int64_t)i0 * a.gs[1] + h * a.gs[2]) * elem<T>::kBytes;
    const uint64_t hid = left >= N ? 0ull : ~0ull << left;
    if constexpr (P::PREF) sg.load(xb, xrow, yb, yrow, hid, st);
    else sg.through(xb, xrow, yb, yrow, hid, lds, st);
    // (threads past the tile's rows repeat a row's: no divergent branch in the loop)
    const int64_t rid = ((int64_t)b * a.H + h) * a.Nq + i0 + min(sr, left - 1);
    srow = a.row[rid];
    if (fm) srowl = a.rowl[rid];
    const bool gone = sr >= left;                      // as a row that sees no key (row_probability)
    const float far = gone ? (fm ? 0.0f : -kNegInf) : 0.0f;
    srow.x = gone ? far : srow.x; srow.y = gone ? far : srow.y; srow.z = gone ? 0.0f : srow.z; srow.w = gone ? 0.0f : srow.w;
    srowl.x = gone ? -kNegInf : srowl.x; srowl.y = gone ? -kNegInf : srowl.y;
  };
  auto store = [&](char* at) {
    if constexpr (P::PREF) sg.store(at, st);
    reinterpret_cast<float4*>(at + S::xybytes(N))[sr] = srow;
    if (fm) reinterpret_cast<float2*>(at + S::xybytes(N) + 16 * N)[sr] = srowl;
  };
  char* const own = smem + (SHARED ? 0 : wk * S::bytes(N));
  int cur = 0;
  if (begin + wk < total) {
    load(begin + wk, own);
    store(own);
    tile_ready<SHARED>();
  }
  const float ls = lam_scale<T>(lt), ps = uniform(kProbScale<T> * ls);
#pragma unroll 1
  for (int t = begin + wk; t < total; t += P::WK) {
    const bool more = t + P::WK < total;
    if (P::PREF && more) load(t + P::WK, nullptr);
    const char* qt = SHARED ? smem + cur * S::bytes(N) : own;
    const char* gt = qt + S::xbytes(N);
    const float4* rows = reinterpret_cast<const float4*>(qt + S::xybytes(N));
    const float2* rowl = reinterpret_cast<const float2*>(rows + N);
    const int g = t / per, h = hk * a.G + g, i00 = (first + t - g * per) * N;
    const float lam = a.lam[h], lams = std::is_same<T, f16_t>::value ? uniform(lam * ls) : lam;
#pragma unroll 1
    for (int it0 = 0; it0 < N; it0 += 32) {
      const int i0 = i00 + it0;
      if (i0 >= a.Nq) break;
      af32x16_t x[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) x[m] = tile_dot<T, S::KB, S::LX, S::KEEP>(qt, it0, m * S::LX / 2, kf[m], lane);
      af32x16_t gm = {0.0f};
      if constexpr (PART != 2) gm = tile_dot<T, S::VB, S::LY, S::KEEP>(gt, it0, 0, vf, lane);
      if (MASK && a.causal) {
        const int lim = jc - off - i0 - 4 * (lane >> 5);                // rows before it do not see the key
        if (__any(lim > -4 * (lane >> 5))) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (8 * (e >> 2) + (e & 3) < lim) { x[0][e] = kNegInf; x[1][e] = kNegInf; }
        }
      }
      if (MODE == kAttnAny && a.mask_kind != 0) {
        const int64_t o = b * a.ms[0] + h * a.ms[1] + jc * a.ms[3];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t oi = o + min(i0 + tile_item(e, lane), a.Nq - 1) * a.ms[2];
          float bias;
          if (fm) bias = mask_raw(((const float*)a.mask)[oi], rscale);
          else bias = ((const uint8_t*)a.mask)[oi] ? kNegInf : 0.0f;
          x[0][e] = mask_add(x[0][e], bias);
          x[1][e] = mask_add(x[1][e], bias);
        }
      }
      const uint64_t zt = zseed + (uint64_t)((((int64_t)b * a.H + h) * a.Nq + i0 + 4 * (lane >> 5) + (lane & 3)) * a.n4);
      // 16 rows at a time: the matrix instructions of one half run beside the arithmetic of the other
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float pc[8], ds[2][8];
#pragma unroll
        for (int q = 2 * s; q < 2 * s + 2; ++q) {
          const int r0 = it0 + tile_item(4 * q, lane);
          uint32_t word[4];
          if (drop) quad_words(attn_mix(zt + (uint64_t)(8 * q * (int64_t)a.n4)), lane, word);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = 4 * q + e, k = n - 8 * s;
            const float4 rw = rows[r0 + e];
            const float2 rl = fm ? rowl[r0 + e] : make_float2(0.0f, 0.0f);
            const float p1 = row_probability(fm, x[0][n], c, rw.x, rl.x), a2 = row_probability(fm, x[1][n], c, rw.y, rl.y);
            const float p2 = lams * a2;
            float gn = gm[n], pn = fmaf(-lam, a2, p1);
            if (drop) {
              const bool keep = attn_keep(word[e], lane & 1, t32);
              gn = keep ? gn * a.up : 0.0f;
              pn = keep ? pn : 0.0f;
            }
            pc[k] = kProbScale<T> == 1.0f ? pn : pn * ps;
            ds[0][k] = p1 * (gn - rw.z);
            ds[1][k] = p2 * (rw.w - gn);
          }
        }
        if constexpr (PART != 1) {
          const typename M::frag fp = M::pack(pc);
#pragma unroll
          for (int d = 0; d < S::VO; ++d) av[d] = M::mul(M::template load_tr<S::LY>(gt, it0 + 16 * s, 0, d, lane), fp, av[d]);
        }
#pragma unroll
        for (int m = 0; m < (PART != 2 ? 2 : 0); ++m) {
          typename M::frag f, rest;
          M::split(ds[m], f, rest);
#pragma unroll
          for (int d = 0; d < S::KO; ++d) {
            const typename M::frag qf = M::template load_tr<S::LX>(qt, it0 + 16 * s, m * S::LX / 2, d, lane);
            ak[m][d] = M::mul(qf, f, ak[m][d]);
            if constexpr (M::SPLIT) ak[m][d] = M::mul(qf, rest, ak[m][d]);
          }
        }
      }
    }
    if (more) {
      if constexpr (SHARED) cur ^= 1;
      else tile_ready<false>();
      if constexpr (!P::PREF) load(t + P::WK, own);
      store(SHARED ? smem + cur * S::bytes(N) : own);
      tile_ready<SHARED>();
    }
  }
  if constexpr (!SHARED) {
    constexpr int NA = PART != 2 ? 2 * S::KO : 0, NB = NA + (PART != 1 ? S::VO : 0);
    af32x16_t* ptr[NB];
#pragma unroll
    for (int d = 0; d < NA / 2; ++d) { ptr[d] = &ak[0][d]; ptr[S::KO + d] = &ak[1][d]; }
#pragma unroll
    for (int d = 0; d < NB - NA; ++d) ptr[NA + d] = &av[d];
    join_waves<P::WK>(ptr, reinterpret_cast<float*>(smem), wk, lane);
    if (wk != 0) return;
  }
  if (!in) return;
  // (a hidden key's columns may hold anything: stored as zeros)
  constexpr int N0 = PART == 2 ? 2 * S::KO : 0, N1 = PART == 1 ? 2 * S::KO : 2 * S::KO + S::VO;
  if (all > a.chunk) {
    float* at = a.part + ((((int64_t)bh * ((a.Nk + 31) / 32) + jb / 32 + wq) * a.splits + split) * 64) * S::KFLOATS + lane * 4;
#pragma unroll
    for (int n = N0; n < N1; ++n) put_block(at + 1024 * n, n < 2 * S::KO ? ak[n / S::KO % 2][n % S::KO] : av[(n - 2 * S::KO) % S::VO], 256);
    return;
  }
#pragma unroll
  for (int n = N0; n < N1; ++n)
    store_gkv<T, S::KO>(a, b, hk, j, ok, n, n < 2 * S::KO ? ak[n / S::KO % 2][n % S::KO] : av[(n - 2 * S::KO) % S::VO], ls, lane);
}

// sums of the splits' gradients: one block an own tile of 32 rows (or keys) and block of 32 columns, one wave
template <typename T, int DH, int DV>
__global__ __launch_bounds__(64) void diff_attn_join_q_kernel(const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  RowWave w;
  const int tile = blockIdx.x / (2 * S::KO), n = blockIdx.x - tile * 2 * S::KO;
  w.init<1, 1, true>(a, tile);
  const int parts = ((rows_end(a, w.rb / a.own * a.own, a.own) + a.n - 1) / a.n + a.chunk - 1) / a.chunk;
  if (!w.ok || parts <= 1) return;
  const int64_t step = 64 * S::QFLOATS;
  const float* at = a.part + w.tile32(a) * a.splits * 64 * S::QFLOATS + w.lane * 4;
  if (n == 0) {
    float dl = 0.0f;
    for (int p = 0; p < parts; ++p) dl += at[p * step + 2048 * S::KO];
    dl = half_sum(dl);
    if (w.lane < 32) a.dlrow[w.rowid] = -dl;
  }
  if (a.gq != nullptr) store_gq<T, S::KO>(a, w, n, sum_block(at + 1024 * n, parts, step));
}
template <typename T, int DH, int DV>
__global__ __launch_bounds__(64) void diff_attn_join_kv_kernel(const DiffAttnArgs a) {
  using S = AttnTile<T, DH, DV>;
  constexpr int NB = 2 * S::KO + S::VO;
  const int tile = blockIdx.x / NB, n = blockIdx.x - tile * NB, lane = threadIdx.x;
  const int tiles = (a.Nk + 31) / 32, bh = tile / tiles, j = (tile - bh * tiles) * 32 + (lane & 31), b = bh / a.Hk, hk = bh - b * a.Hk;
  const int jb = (tile - bh * tiles) * 32 / a.own * a.own, first = a.causal ? max(0, jb - (a.Nk - a.Nq)) / a.n : 0;
  const int parts = (max(0, (a.Nq + a.n - 1) / a.n - first) * a.G + a.chunk - 1) / a.chunk;
  const float ls = lam_scale<T>(lam_top<T>(a.lam, hk, a.G, lane));        // (by all lanes, before some leave)
  if (j >= a.Nk || parts <= 1) return;
  const bool ok = !(a.kpm != nullptr && a.kpm[(int64_t)b * a.Nk + j]);
  const float* at = a.part + (int64_t)tile * a.splits * 64 * S::KFLOATS + lane * 4;
  store_gkv<T, S::KO>(a, b, hk, j, ok, n, sum_block(at + 1024 * n, parts, 64 * S::KFLOATS), ls, lane);
}

// ---- launch -----------------------------------------------------------------------------------------------------------------------
template <typename K>
static int attn_launch(K kernel, int64_t blocks, int threads, int lds, const DiffAttnArgs& args, hipStream_t st, const char* who) {
  DiffAttnArgs a = args;
  a.work = (int)blocks;
  blocks = (blocks + 7) / 8 * 8;                     // (xcd_tile)
  if (blocks >= (int64_t(1) << 31)) { set_error("%s: %ld blocks", who, (long)blocks); return UBV_ERR_UNSUPPORTED; }
  if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), (size_t)lds, st, a);
  UBV_CHECK_LAUNCH(who);
  return UBV_OK;
}

template <typename F> static int attn_mode(const DiffAttnArgs& a, F&& f) {
  if (a.mask_kind != 0 || (a.causal && a.t16 != 0)) return f(std::integral_constant<int, kAttnAny>{});
  if (a.causal) return f(std::integral_constant<int, kAttnCausal>{});
  if (a.t16 != 0) return f(std::integral_constant<int, kAttnDrop>{});
  return f(std::integral_constant<int, kAttnPlain>{});
}

// How a pass over `own` items a head against `staged` ones is cut into blocks.
//
// shared: a shared block does four private blocks' work in 4 `cost` times their time (it stages a tile once for 128 own items), but
// there are a quarter as many: with 256 CUs the rounds of blocks decide.  Measured at one block a CU (bf16, us, shared / private):
// 64 / 64 wide heads 80 / 121, 128 / 128 133 / 278; 32 / 64 at 10 000 x 10 000 and 4 heads (316 or 1252 blocks) 400 / 299.
// f32 at 8 x 8 heads, 900 x 900, grad_q: 64 / 64 386 / 476, 128 / 128 1119 / 2338, 128 / 256 1440 / 2593.  What the rule does not see
// yet: causal f32 heads up to 64 / 128 are slower shared (2 x 16 heads, 2048 causal, forward / grad_q / grad_k and grad_v: 32 / 64
// 405, 432, 674, private 283, 293, 385; 64 / 128 771, 851, 1474, private 634, 620, 862), and f32 128 / 128 at half a chip of wide
// tiles (4 heads, 4096 x 4096) slower private: forward 1706, shared 1527, grad_q 2554, 2050.
// splits: private blocks that share the staged items of one own tile, `chunk` staged tiles each, where own tiles alone leave the chip
// empty: up to twice as many waves as fill it (ragged batches and causal rows are unequal), at least four tiles for each wave.
// (Shared blocks that split a causal own tile into equal chunks fill the chip too, but lose to it what joining them costs: 64 / 128
// wide f16 heads, 2 x 2 shared by four each, 2047 causal, us: forward 109 + 14, private 125; grad_q 135 + 8, 126; grad_k / grad_v
// 182 + 8, 148 + 5.)
struct AttnCut {
  bool shared;
  int splits, chunk;
  AttnCut whole() const { return {shared, 1, 1 << 29}; }
};
// staged: items that an own tile meets at most, in `heads` heads with ends of their own
template <typename T, int DH, int DV>
static AttnCut attn_cut(const DiffAttnArgs& a, int64_t groups, int64_t own, int64_t staged, int heads, bool may_share) {
  using S = AttnTile<T, DH, DV>;
  const int64_t wide = groups * ((own + 127) / 128), narrow = groups * ((own + 31) / 32);
  const double cost = 4.0 * (DH <= 32 ? 0.8 : 0.65);
  const double ts = a.causal ? std::max(cost, cost * wide / 512.0) : cost * ((wide + 255) / 256);
  const double tp = a.causal ? std::max(1.0, narrow / 512.0) : (double)((narrow + 255) / 256);
  if (may_share && ts < tp) return AttnCut{true}.whole();
  const int64_t tiles = (staged + 31) / 32 * heads, waves = narrow * S::WK, fill = 1024 * S::MINW * 2;
  int64_t splits = waves * 2 >= fill && !a.causal ? 1 : (fill + waves - 1) / waves;
  splits = std::min<int64_t>({splits, tiles / S::WK / 4, kAttnSplits});
  if (splits <= 1) return AttnCut{false}.whole();
  return {false, (int)splits, (int)((tiles + splits - 1) / splits)};
}
template <typename T, int DH, int DV> static AttnCut attn_cut_fwd(const DiffAttnArgs& a) {
  return attn_cut<T, DH, (DV > 128 ? 128 : DV)>(a, (int64_t)a.B * a.Hk * (a.Dv > 128 ? 2 : 1), a.R, a.Nk, 1, true);
}
template <typename T, int DH, int DV> static AttnCut attn_cut_q(const DiffAttnArgs& a) {
  return attn_cut<T, DH, DV>(a, (int64_t)a.B * a.Hk, a.R, a.Nk, 1, true);
}
// (128 / 128 in one pass spills as a shared block: 357 us, private 277)
template <int DH, int DV> constexpr bool kAttnKvPrivate = DH == 128 && DV == 128;
template <typename T, int DH, int DV> static AttnCut attn_cut_kv(const DiffAttnArgs& a) {
  return attn_cut<T, DH, DV>(a, (int64_t)a.B * a.Hk, a.Nk, a.Nq, a.G, !kAttnKvPrivate<DH, DV>);
}

// bytes of the splits' sums
template <typename T, int DH, int DV> static int64_t attn_bytes_fwd(const DiffAttnArgs& a) {
  constexpr int DC = DV > 128 ? 128 : DV;
  const AttnCut c = attn_cut_fwd<T, DH, DV>(a);
  return c.splits <= 1 ? 0 : (int64_t)a.B * a.Hk * ((a.R + 31) / 32) * ((a.Dv + DC - 1) / DC) * c.splits * 64 * FwdState<T, DC>::FLOATS * 4;
}
template <typename T, int DH, int DV> static int64_t attn_bytes_bwd(const DiffAttnArgs& a) {
  using S = AttnTile<T, DH, DV>;
  const AttnCut q = attn_cut_q<T, DH, DV>(a), kv = attn_cut_kv<T, DH, DV>(a);
  const int64_t heads = (int64_t)a.B * a.Hk;
  const int64_t bq = q.splits <= 1 ? 0 : heads * ((a.R + 31) / 32) * q.splits * 64 * S::QFLOATS * 4;
  const int64_t bk = kv.splits <= 1 ? 0 : heads * ((a.Nk + 31) / 32) * kv.splits * 64 * S::KFLOATS * 4;
  return bq > bk ? bq : bk;
}

template <typename T, int DH, int DV>
static int attn_forward(DiffAttnArgs a, void* ws, int64_t ws_bytes, hipStream_t st) {
  // heads of 256: two blocks with 128 columns each (both compute the scores; one block's accumulators would not fit)
  constexpr int DC = DV > 128 ? 128 : DV;
  const int64_t heads = (int64_t)a.B * a.Hk;
  const char* who = "diff_attention_forward";
  AttnCut cut = attn_cut_fwd<T, DH, DV>(a);
  if (ws_bytes < attn_bytes_fwd<T, DH, DV>(a)) cut = cut.whole();
  a.splits = cut.splits; a.chunk = cut.chunk;
  a.part = (float*)ws;
  a.halves = (a.Dv + DC - 1) / DC;
  auto run = [&](auto shared) {
    constexpr bool SH = decltype(shared)::value;
    using P = AttnPlan<T, DH, DC, SH>;
    a.own = 32 * P::WQ; a.n = P::N;
    return attn_mode(a, [&](auto mode) {
      return attn_launch(diff_attn_fwd_kernel<T, DH, DC, SH, decltype(mode)::value>,
                         heads * ((a.R + 32 * P::WQ - 1) / (32 * P::WQ)) * a.halves * a.splits, P::NT, P::lds(FwdState<T, DC>::FLOATS), a, st, who);
    });
  };
  const int rc = cut.shared ? run(std::true_type{}) : run(std::false_type{});
  if (rc != UBV_OK || a.splits == 1) return rc;
  if (a.R < 32) hipLaunchKernelGGL((diff_attn_join_kernel<T, DC>), dim3((unsigned)(heads * a.R * a.halves)), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((diff_attn_join_rows_kernel<T, DC>), dim3((unsigned)(heads * ((a.R + 31) / 32) * a.halves * (DC / 32))), dim3(64), 0, st, a);
  UBV_CHECK_LAUNCH(who);
  return UBV_OK;
}

template <typename T, int DH, int DV>
static int attn_backward(DiffAttnArgs a, float* glam, int64_t part_bytes, hipStream_t st) {
  using S = AttnTile<T, DH, DV>;
  const int64_t heads = (int64_t)a.B * a.Hk, rows = (int64_t)a.B * a.H * a.Nq;
  const char* who = "diff_attention_backward";
  const bool room = part_bytes >= attn_bytes_bwd<T, DH, DV>(a);
  auto run = [&](auto shared, auto pass) {
    constexpr bool SH = decltype(shared)::value;
    constexpr int PASS = decltype(pass)::value;                 // 0 .. 2: grad_k / grad_v of that part, 3: grad_q
    using P = AttnPlan<T, DH, DV, SH>;
    a.own = 32 * P::WQ; a.n = P::N;
    const int64_t blocks = heads * (((PASS == 3 ? a.R : a.Nk) + 32 * P::WQ - 1) / (32 * P::WQ)) * a.splits;
    return attn_mode(a, [&](auto mode) {
      constexpr int MODE = decltype(mode)::value;
      if constexpr (PASS == 3)
        return attn_launch(diff_attn_bwd_q_kernel<T, DH, DV, SH, MODE>, blocks, P::NT, P::lds((2 * S::KO + 1) * 16), a, st, who);
      else
        return attn_launch(diff_attn_bwd_kv_kernel<T, DH, DV, SH, MODE, PASS>, blocks, P::NT, P::lds((2 * S::KO + S::VO) * 16), a, st, who);
    });
  };
  auto pass = [&](AttnCut cut, auto which) {
    if (!room) cut = cut.whole();
    a.splits = cut.splits; a.chunk = cut.chunk;
    if constexpr (decltype(which)::value == 3 || !kAttnKvPrivate<DH, DV>)
      if (cut.shared) return run(std::true_type{}, which);
    return run(std::false_type{}, which);
  };
  int rc = UBV_OK;
  if (a.gq != nullptr || glam != nullptr) {
    rc = pass(attn_cut_q<T, DH, DV>(a), std::integral_constant<int, 3>{});
    if (rc != UBV_OK) return rc;
    if (a.splits > 1) {
      hipLaunchKernelGGL((diff_attn_join_q_kernel<T, DH, DV>), dim3((unsigned)(heads * ((a.R + 31) / 32) * 2 * S::KO)), dim3(64), 0, st, a);
      UBV_CHECK_LAUNCH(who);
    }
    if (glam != nullptr) {
      hipLaunchKernelGGL(diff_attn_lam_kernel, dim3((unsigned)a.H), dim3(1024), 0, st, a.dlrow, glam, a.B, a.H, a.Nq);
      UBV_CHECK_LAUNCH(who);
    }
  } else {
    hipLaunchKernelGGL(diff_attn_del_kernel<T>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a);
    UBV_CHECK_LAUNCH(who);
  }
  if (a.gk == nullptr) return rc;
  const AttnCut cut = attn_cut_kv<T, DH, DV>(a);
  if constexpr (2 * DH + DV > 384) {
    rc = pass(cut, std::integral_constant<int, 1>{});
    if (rc == UBV_OK) rc = pass(cut, std::integral_constant<int, 2>{});
  } else {
    rc = pass(cut, std::integral_constant<int, 0>{});
  }
  if (rc != UBV_OK || a.splits == 1) return rc;
  hipLaunchKernelGGL((diff_attn_join_kv_kernel<T, DH, DV>), dim3((unsigned)(heads * ((a.Nk + 31) / 32) * (2 * S::KO + S::VO))), dim3(64), 0, st, a);
  UBV_CHECK_LAUNCH(who);
  return UBV_OK;
}

// the smallest pair of widths that holds the call's
#define UBV_ATTN_PAIRS(DO)                                                                    \
  if (a.Dh <= 16 && a.Dv <= 32) DO(16, 32)                                                    \
  if (a.Dh <= 32 && a.Dv <= 64) DO(32, 64)                                                    \
  if (a.Dh <= 64 && a.Dv <= 64) DO(64, 64)                                                    \
  if (a.Dh <= 64 && a.Dv <= 128) DO(64, 128)                                                  \
  if (a.Dh <= 128 && a.Dv <= 128) DO(128, 128)                                                \
  DO(128, 256)

int UBV_ATTN_NAME(forward)(const DiffAttnArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
#define UBV_DO(DH, DV) return attn_forward<UBV_ATTN_T, DH, DV>(a, ws, ws_bytes, st);
  UBV_ATTN_PAIRS(UBV_DO)
#undef UBV_DO
}

int UBV_ATTN_NAME(backward)(const DiffAttnArgs& a, float* glam, int64_t part_bytes, hipStream_t st) {
#define UBV_DO(DH, DV) return attn_backward<UBV_ATTN_T, DH, DV>(a, glam, part_bytes, st);
  UBV_ATTN_PAIRS(UBV_DO)
#undef UBV_DO
}

int64_t UBV_ATTN_NAME(bytes)(const DiffAttnArgs& a, bool backward) {
#define UBV_DO(DH, DV) return backward ? attn_bytes_bwd<UBV_ATTN_T, DH, DV>(a) : attn_bytes_fwd<UBV_ATTN_T, DH, DV>(a);
  UBV_ATTN_PAIRS(UBV_DO)
#undef UBV_DO
}

}  // namespace ubv
