// Matrix-product tiles shared by the encoder and softmax-loss operators (linear.hip, softmax_loss.hip, attention.hip):
// one code path for float, bf16 and fp16 operands with fp32 accumulation (gfx950).  Internal to the library.
//
// Fragments.  A wave multiplies 32x32 tiles; a lane's operand fragment is 16 bytes of ONE row: with r = lane & 31 and
// h = lane >> 5 the elements k = g + KPF * h + [0, KPF) of row r, where KPF = 16 / sizeof(T).  For 16-bit types that is one
// v_mfma_f32_32x32x16; for float it is four v_mfma_f32_32x32x2, whose two k-slots may name any pair of k as long as both
// operands agree.  So LDS images, loads and loops are the same bytes for every type.
//
// Accumulator: lane holds column (lane & 31) and rows 8 a + 4 h + c, register 4 a + c: four consecutive ROWS per quad.
// The row operand is therefore the one whose index is contiguous in the output (the weights of a linear layer): a quad is
// then 8 or 16 contiguous bytes of the output row.
#pragma once
#include "tile_pick.h"
#include "tt_common.h"

namespace ttm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <class T> struct Type;
template <> struct Type<float> {
  typedef f32x4 quad;
  static constexpr int KPF = 4;  // elements of a 16-byte fragment
};
template <> struct Type<__bf16> {
  typedef bf16x4 quad;
  static constexpr int KPF = 8;
};
template <> struct Type<_Float16> {
  typedef f16x4 quad;
  static constexpr int KPF = 8;
};

template <class T>
__device__ __forceinline__ void mma(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[s], fb[s], c, 0, 0, 0);
  } else if constexpr (__is_same(T, __bf16)) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// four floats -> four T, rounded to nearest even (one rounding)
template <class T>
__device__ __forceinline__ typename Type<T>::quad to_quad(f32x4 v) {
  return __builtin_convertvector(v, typename Type<T>::quad);
}
template <class T>
__device__ __forceinline__ f32x4 from_quad(typename Type<T>::quad v) {
  return __builtin_convertvector(v, f32x4);
}

// LDS images.  Every operand tile is kept as it lies in memory, in blocks of rows of 128 bytes: eight 16-byte chunks whose
// position is XORed with a function of the row.  A block is read two ways:
//   along its rows (row_frag: lanes = 16 consecutive rows, one chunk): a K-contiguous operand;
//   across them (col_frag: lanes = 32 consecutive columns, KPF rows each): a K-strided operand, transposed by the read itself —
//   16-bit by two ds_read_b64_tr_b16 (16 lanes hand in four rows of 32 bytes, each gets four rows of its column), float by
//   four ds_read_b32.
// The XOR reverses bits 1..3 of the row: 16 rows at one chunk lie in 16 different slots, and four rows at one 64-byte window
// in the four quarters of the banks: both reads are free of bank conflicts.
constexpr int kRowBytes = 128;
__device__ __forceinline__ int twist(int row) { return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1); }
__device__ __forceinline__ int swz(int row, int chunk) { return row * kRowBytes + (chunk ^ twist(row)) * 16; }

__device__ __forceinline__ u32x4 row_frag(const char* __restrict__ block, int row, int chunk) {
  return *reinterpret_cast<const u32x4*>(block + swz(row, chunk));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ u32x2 tr_read(const char* __restrict__ p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
}
// rows [k, k + KPF) of column (col0 + lane & 31), k = k0 + KPF * (lane >> 5);  k0 % (2 KPF) == 0, col0 % 32 == 0
template <class T>
__device__ __forceinline__ u32x4 col_frag(const char* __restrict__ block, int k0, int col0, int lane) {
  if constexpr (sizeof(T) == 4) {
    const int c = col0 + (lane & 31), k = k0 + 4 * (lane >> 5);
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(block + swz(k + j, c >> 2) + (c & 3) * 4);
    return v;
  } else {
    const int j = lane & 15;
    const int c = col0 + (lane & 16) + 4 * (j & 3), k = k0 + 8 * (lane >> 5) + (j >> 2);
    const int at = (c & 4) * 2;  // the second half of a 16-byte chunk
    const u32x2 lo = tr_read(block + swz(k, c >> 3) + at), hi = tr_read(block + swz(k + 4, c >> 3) + at);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

// Global memory to LDS without registers: each lane names its 16 bytes, a wave fills 1024 contiguous bytes (8 rows of a
// block).  The caller waits (stage_wait) before anyone reads.
typedef __attribute__((address_space(1))) const void gas_void;
typedef __attribute__((address_space(3))) void las_void;
__device__ __forceinline__ void lds_fill(const char* src, char* dst) {
  __builtin_amdgcn_global_load_lds((gas_void*)src, (las_void*)dst, 16, 0, 0);
}
// This wave's outstanding fills have landed and its LDS accesses are done; then the whole workgroup's.
__device__ __forceinline__ void stage_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// LDS as a wave's own scratch: what its lanes wrote is there for all of them
__device__ __forceinline__ void wave_lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---- a product's operand in global memory ------------------------------------------------------------------
// `p` is 16-byte aligned, `ld` a multiple of KPF elements, and so is the contiguous extent (callers pack what is not).
// K-contiguous (KS = false): element (row, k) at p[row * ld + k].  K-strided (KS = true): element (row, k) at p[k * ld + row].
struct Operand {
  const void* p;
  long long ld;
};

// A tile of an operand in LDS: K-contiguous one block of R rows (128 bytes of k each); K-strided BK rows in R * sizeof(T) / 128
// column blocks.  Either way R * 128 bytes, filled in groups of 8 rows x 128 bytes, one group per wave and instruction.
template <class T, bool KS, int R, int WAVES>
struct Tile {
  static constexpr int KPF = Type<T>::KPF, BK = kRowBytes / (int)sizeof(T), BYTES = R * kRowBytes;
  static constexpr int N = R / 8 / WAVES;  // groups per wave
  static_assert(R % (8 * WAVES) == 0 && R % BK == 0, "whole groups per wave, whole column blocks");
  uint32_t off[N];  // of this lane's 16 bytes of each group, from the tile's first element

  // r0: first row of the output side, r0 < rows: how many there are (K-strided: readable columns)
  __device__ __forceinline__ void init(const Operand& o, int r0, int rows, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = i * WAVES + wave, row = 8 * g + (lane >> 3);
      if constexpr (!KS) {
        const int ch = (lane & 7) ^ twist(row);
        off[i] = (uint32_t)(((long long)(min(r0 + row, rows - 1) - r0) * o.ld + ch * KPF) * (int)sizeof(T));
      } else {
        const int blk = row / BK, k = row % BK, ch = (lane & 7) ^ twist(k);
        off[i] = (uint32_t)((k * o.ld + min(r0 + blk * BK + ch * KPF, rows - KPF) - r0) * (int)sizeof(T));
      }
    }
  }
  static __device__ __forceinline__ const char* base(const Operand& o, int r0, int k0) {
    return static_cast<const char*>(o.p) + (KS ? k0 * o.ld + r0 : r0 * o.ld + k0) * (long long)sizeof(T);
  }
  __device__ __forceinline__ void fill(const char* __restrict__ src, char* __restrict__ tile, int wave) const {
#pragma unroll
    for (int i = 0; i < N; ++i) lds_fill(src + off[i], tile + (i * WAVES + wave) * 1024);
  }
  // the last, partial step of k: what lies at or behind kend arrives as zero
  __device__ __forceinline__ void fill_tail(const char* __restrict__ src, char* __restrict__ tile, int left, int wave, int lane) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = 8 * (i * WAVES + wave) + (lane >> 3);
      const int k = KS ? row % BK : ((lane & 7) ^ twist(row)) * KPF;
      u32x4 v = {0, 0, 0, 0};
      if (k < left) v = *reinterpret_cast<const u32x4*>(src + off[i]);
      *reinterpret_cast<u32x4*>(tile + (i * WAVES + wave) * 1024 + lane * 16) = v;
    }
  }
  // fragment of rows [row0, row0 + 32) of the output side, group g of the step's k
  static __device__ __forceinline__ u32x4 get(const char* __restrict__ tile, int row0, int g, int lane) {
    if constexpr (!KS) return row_frag(tile, row0 + (lane & 31), 2 * g + (lane >> 5));
    else return col_frag<T>(tile + row0 / BK * (BK * kRowBytes), g * 2 * KPF, row0 % BK, lane);
  }
};

// Tile coordinates of workgroup `id` of `total`: workgroups go round the eight XCDs, so each XCD is given one contiguous
// eighth of the tiles, whose operand panels then meet in its own L2.  A label for placement only; any mapping is right.
__device__ __forceinline__ int xcd_tile(int id, int total) {
  const int q = total >> 3, r = total & 7, x = id & 7;
  return x * q + min(x, r) + (id >> 3);
}

constexpr int kBand = 4;
// Row and column of tile t of a grid of gm x gn: bands of four rows, column by column, so that the tiles in flight on an XCD
// share both operands' panels (32 tiles of one row would share one; bf16 8192 cubed, 128-wide tiles: 1236 -> 1112 us).
__device__ __forceinline__ void tile_at(int t, int gm, int gn, int& m, int& n) {
  const int band = t / (kBand * gn), first = band * kBand, rows = min(kBand, gm - first), in = t - band * kBand * gn;
  n = in / rows;
  m = first + in - n * rows;
}

struct Shape {
  int M, N, K;      // output [M, N] (N contiguous), contraction K.  A K-contiguous operand is readable, and zero, up to the
                    // next multiple of KPF behind K; a K-strided one has K rows, readable to the next multiple of KPF columns
  int kper;         // k of one split (a multiple of BK unless there is one split)
};

// A workgroup's tile: BM x BN outputs, WM x WN waves of MJ x NI accumulators each; two LDS buffers of BYTES.
template <int BM_, int BN_, int WM_, int WN_>
struct Block {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int MJ = BM / 32 / WM, NI = BN / 32 / WN, BYTES = (BM + BN) * kRowBytes;
  f32x16 acc[NI][MJ];
  int lane, wave, r, h, wm, wn;

  __device__ __forceinline__ Block() {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    r = lane & 31;
    h = lane >> 5;
    wm = wave % WM;
    wn = wave / WM;
  }

  // acc[i][j]: output columns n0 + 32 (wn * NI + i) + row, output rows m0 + 32 (wm * MJ + j) + (lane & 31).
  // X: output rows (M), Y: output columns (N).  One step ahead: the next step's tiles stream into the other buffer under
  // this step's matrix instructions; one barrier a step.  LDS may be reused after the caller's next barrier.
  // float: every other step goes to a second set of accumulators, which halves the length of the chains of additions.
  template <class T, bool XKS, bool YKS>
  __device__ __forceinline__ void product(char* __restrict__ b0, char* __restrict__ b1, const Operand& X, const Operand& Y,
                                          const Shape& s, int m0, int n0, int kbeg, int kend) {
    using TX = Tile<T, XKS, BM, WAVES>;
    using TY = Tile<T, YKS, BN, WAVES>;
    constexpr int BK = TX::BK;
    constexpr bool TWO = sizeof(T) == 4;
    f32x16 acc2[TWO ? NI : 1][TWO ? MJ : 1];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          acc[i][j][e] = 0.f;
          if constexpr (TWO) acc2[i][j][e] = 0.f;
        }
    if (kbeg >= kend) return;
    constexpr int KPF = Type<T>::KPF;
    // a padded contiguous extent bounds what a column clamp may touch
    const int xr = XKS ? (s.M + KPF - 1) / KPF * KPF : s.M, yr = YKS ? (s.N + KPF - 1) / KPF * KPF : s.N;
    TX tx;
    TY ty;
    tx.init(X, m0, xr, wave, lane);
    ty.init(Y, n0, yr, wave, lane);
    const char* xs = TX::base(X, m0, kbeg);
    const char* ys = TY::base(Y, n0, kbeg);
    const long long xstep = (XKS ? X.ld * BK : BK) * (long long)sizeof(T), ystep = (YKS ? Y.ld * BK : BK) * (long long)sizeof(T);
    const int steps = (kend - kbeg + BK - 1) / BK, left = kend - kbeg - (steps - 1) * BK;
    auto issue = [&](int t, char* __restrict__ b) {
      if (t + 1 < steps || left == BK) {
        tx.fill(xs, b, wave);
        ty.fill(ys, b + BM * kRowBytes, wave);
        xs += xstep;
        ys += ystep;
      } else {
        tx.fill_tail(xs, b, left, wave, lane);
        ty.fill_tail(ys, b + BM * kRowBytes, left, wave, lane);
      }
    };
    auto step = [&](int t, char* __restrict__ cur, char* __restrict__ nxt, auto& c) {
      stage_wait();
      if (t + 1 < steps) issue(t + 1, nxt);
      // the next group's fragments are asked for before this group's products
      u32x4 fy[2][NI], fx[2][MJ];
      auto get = [&](int g) {
#pragma unroll
        for (int i = 0; i < NI; ++i) fy[g & 1][i] = TY::get(cur + BM * kRowBytes, (wn * NI + i) * 32, g, lane);
#pragma unroll
        for (int j = 0; j < MJ; ++j) fx[g & 1][j] = TX::get(cur, (wm * MJ + j) * 32, g, lane);
      };
      get(0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g < 3) get(g + 1);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int j = 0; j < MJ; ++j) mma<T>(c[i][j], fy[g & 1][i], fx[g & 1][j]);
      }
    };
    issue(0, b0);
    for (int t = 0; t < steps; t += 2) {
      step(t, b0, b1, acc);
      if (t + 1 < steps) {
        if constexpr (TWO) step(t + 1, b1, b0, acc2);
        else step(t + 1, b1, b0, acc);
      }
    }
    if constexpr (TWO) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) acc[i][j] += acc2[i][j];
    }
  }

  // Calls fn(m, n, quad) for every quad of four consecutive output columns this lane holds.
  template <class F>
  __device__ __forceinline__ void for_quads(int m0, int n0, F&& fn) {
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x4 v = {acc[i][j][4 * a], acc[i][j][4 * a + 1], acc[i][j][4 * a + 2], acc[i][j][4 * a + 3]};
          fn(m0 + (wm * MJ + j) * 32 + r, n0 + (wn * NI + i) * 32 + 8 * a + 4 * h, v);
        }
  }

  // Rows of the output instead: the accumulators of 32 rows at a time go through the wave's own part of LDS and come back as
  // KPF consecutive columns per lane, so that 16 lanes read and write 256 consecutive bytes of a row (a quad per lane and row
  // touched 16 bytes of 32 rows at a time).  fn(j, step, m, n, v): v holds KPF / 4 quads; n does not depend on j, nor, where
  // 64 lanes are whole rows, on the step.
  // The 16-byte chunk of a row is XORed with the row: no bank conflicts either way.  pre(j): before the rows of j.
  template <class T>
  struct Rows {
    static constexpr int W = NI * 32, Q = Type<T>::KPF / 4, LPR = W / Type<T>::KPF, STEPS = LPR / 2;
    static constexpr bool WHOLE = 64 % LPR == 0;  // a lane keeps its columns
  };
  template <class T>
  __device__ __forceinline__ int chunk_at(int step) const { return ((Rows<T>::WHOLE ? 0 : step * 64) + lane) % Rows<T>::LPR; }
  template <class T>
  __device__ __forceinline__ int row_in(int step) const {
    return Rows<T>::WHOLE ? step * (64 / Rows<T>::LPR) + lane / Rows<T>::LPR : (step * 64 + lane) / Rows<T>::LPR;
  }
  template <class T>
  __device__ __forceinline__ int row_col(int n0, int step) const { return n0 + wn * Rows<T>::W + chunk_at<T>(step) * Type<T>::KPF; }
  template <class T>
  __device__ __forceinline__ int row_at(int m0, int j, int step) const { return m0 + (wm * MJ + j) * 32 + row_in<T>(step); }
  template <class T, class P, class F>
  __device__ __forceinline__ void for_rows(char* __restrict__ b0, char* __restrict__ b1, int m0, int n0, P&& pre, F&& fn) {
    using R = Rows<T>;
    constexpr int AREA = 32 * R::W * 4, PER = BYTES / AREA;
    static_assert(PER * 2 >= WAVES, "an area per wave");
    __syncthreads();  // everyone is done with the operands
    char* const area = wave < PER ? b0 + wave * AREA : b1 + (wave - PER) * AREA;
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      pre(j);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x4 v = {acc[i][j][4 * a], acc[i][j][4 * a + 1], acc[i][j][4 * a + 2], acc[i][j][4 * a + 3]};
          *reinterpret_cast<f32x4*>(area + r * (R::W * 4) + (((i * 8 + 2 * a + h) ^ (r & 7)) * 16)) = v;
        }
      wave_lds_sync();
#pragma unroll
      for (int s = 0; s < R::STEPS; ++s) {
        const int row = row_in<T>(s);
        f32x4 v[R::Q];
#pragma unroll
        for (int q = 0; q < R::Q; ++q)
          v[q] = *reinterpret_cast<const f32x4*>(area + row * (R::W * 4) + (((chunk_at<T>(s) * R::Q + q) ^ (row & 7)) * 16));
        fn(j, s, row_at<T>(m0, j, s), row_col<T>(n0, s), v);
      }
      wave_lds_sync();
    }
  }
};
using Small = Block<64, 64, 2, 2>;
using Mid = Block<128, 128, 2, 2>;
using Large = Block<256, 256, 4, 2>;
using Three = Block<256, 192, 4, 2>;  // gradients of 384 columns: two of these, where 256 leave a quarter empty

// one row's quad at columns [n, n + 4) of a row-major matrix; `vec`: whole quads are in range and aligned
template <class T>
__device__ __forceinline__ void store_quad(T* __restrict__ p, long long ld, int m, int n, int N, bool vec, f32x4 v) {
  const typename Type<T>::quad q = to_quad<T>(v);
  T* __restrict__ d = p + m * ld + n;
  if (vec) {
    if (n < N) *reinterpret_cast<typename Type<T>::quad*>(d) = q;
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < N) d[c] = q[c];
  }
}
template <class T>
__device__ __forceinline__ f32x4 load_quad(const T* __restrict__ p, long long ld, int m, int n, int N, bool vec) {
  const T* __restrict__ d = p + m * ld + n;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    if (n < N) v = from_quad<T>(*reinterpret_cast<const typename Type<T>::quad*>(d));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < N) v[c] = (float)d[c];
  }
  return v;
}

// KPF consecutive columns (16 bytes) of a row
template <class T>
struct Chunk {
  static constexpr int Q = Type<T>::KPF / 4;
  typename Type<T>::quad q[Q];
  __device__ __forceinline__ void load(const T* __restrict__ p) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
    __builtin_memcpy(q, &v, 16);
  }
  __device__ __forceinline__ void store(T* __restrict__ p) const {
    u32x4 v;
    __builtin_memcpy(&v, q, 16);
    *reinterpret_cast<u32x4*>(p) = v;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < Q; ++i) q[i] = typename Type<T>::quad(0);
  }
};

// ---- host side ----------------------------------------------------------------------------------------------
inline long long pad_to(long long n, int m) { return (n + m - 1) / m * m; }
inline int dtype_bytes(int dtype) { return dtype == TT_F32 ? 4 : 2; }
// scales and caps of scores that are taken (false for NaN)
inline bool tt_scale_ok(float s) { return s >= 1e-15f && s <= 1e15f; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Can a [rows, cols] matrix of row stride ld be read in 16-byte chunks as it is?
inline bool packed_ok(const void* p, long long ld, long long cols, int dtype) {
  const int kpf = 16 / dtype_bytes(dtype);
  // (the last bound keeps a tile's 32-bit offsets in range)
  return tt_aligned16(p) && ld % kpf == 0 && cols % kpf == 0 && ld < (1 << 22);
}
// bytes of its packed copy (row stride padded to 16 bytes, the padding zero), 0 if it needs none
inline size_t pack_bytes(const void* p, long long ld, long long rows, long long cols, int dtype) {
  if (packed_ok(p, ld, cols, dtype)) return 0;
  return align256((size_t)rows * (size_t)pad_to(cols, 16 / dtype_bytes(dtype)) * dtype_bytes(dtype));
}

// f(block) with the block shape of a tile edge that pick_tile gave for T
template <class T, class F>
int with_block(int edge, F&& f) {
  if constexpr (sizeof(T) == 2)
    if (edge == 256) return f(static_cast<Large*>(nullptr));
  return edge == 64 ? f(static_cast<Small*>(nullptr)) : f(static_cast<Mid*>(nullptr));
}

}  // namespace ttm

// The gradient products of linear.hip and softmax_loss.hip: P = X Y with a K-strided Y [K, N] and X K-contiguous (xks = 0:
// [M, K]) or K-strided (xks = 1: [K, M]).
//   out  != null: out[m, n] = T(alpha * (*alpha_dev) * P)    (alpha_dev may be null; one split)
//   slab != null: slab[z][m, n] = P of split z (accumulate = 0), or slab[m, n] += P (accumulate = 1, one split)
struct GradProduct {
  ttm::Operand X, Y;
  int M, N, K, xks, nsplit;
  void* out;
  long long ldo;
  float* slab;
  int accumulate;
  float alpha;
  const float* alpha_dev;
};
int tt_launch_grad_product(const GradProduct& g, int dtype, hipStream_t st);
// out[i] = T(alpha * (*alpha_dev) * sum_z slab[z][i]), z in order, for n elements of a [n / N, N] matrix of row stride ldo
int tt_launch_slab_sum(const float* slab, int nsplit, long long n, void* out, int dtype, float alpha, const float* alpha_dev,
                       hipStream_t st);
// splits of a [M, N] gradient product of contraction K
int tt_grad_splits(long long M, long long N, long long K, int dtype);

// packs a [rows, cols] matrix (row stride ld elements of `width` bytes) to row stride `ldp`, zeros behind cols (linear.hip)
int tt_launch_pack(const void* src, long long ld, void* dst, long long ldp, long long rows, long long cols, int width,
                   hipStream_t st);
