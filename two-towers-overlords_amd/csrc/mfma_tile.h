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

// LDS image of an operand tile: rows of 128 bytes (BK = 128 / sizeof(T) consecutive k), eight 16-byte chunks whose position
// is XORed with a function of the row.  Reads (lanes = consecutive rows, one chunk) meet 16 different slots per 16 rows;
// so do the transposing writes of stage_ks (lanes = every fourth row, one chunk): conflict-free both ways.
constexpr int kRowBytes = 128;
__device__ __forceinline__ int swz(int row, int chunk) { return row * kRowBytes + ((chunk ^ ((row >> 1) ^ (row >> 4))) & 7) * 16; }

__device__ __forceinline__ u32x4 frag(const char* __restrict__ tile, int row, int chunk) {
  return *reinterpret_cast<const u32x4*>(tile + swz(row, chunk));
}

// Eight 16-bit rows x four columns (or four float rows x four columns), one 8- / 16-byte load per row, to four 16-byte
// chunks of consecutive k: the transposition of a K-strided operand on its way into LDS.  16-bit: two v_perm_b32 make the
// (k, k+1) pairs of two columns, the rest is register naming.
template <class T> struct KsUnit;
template <> struct KsUnit<float> {
  f32x4 v[4];
  __device__ __forceinline__ u32x4 column(int c) const {
    f32x4 o = {v[0][c], v[1][c], v[2][c], v[3][c]};
    return __builtin_bit_cast(u32x4, o);
  }
};
struct KsUnit16 {
  u32x2 v[8];
  __device__ __forceinline__ u32x4 column(int c) const {
    const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;  // high / low halves of (row k + 1, row k)
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = __builtin_amdgcn_perm(v[2 * j + 1][c >> 1], v[2 * j][c >> 1], sel);
    return o;
  }
};
template <> struct KsUnit<__bf16> : KsUnit16 {};
template <> struct KsUnit<_Float16> : KsUnit16 {};

// ---- a product's operand in global memory ------------------------------------------------------------------
// `p` is 16-byte aligned, `ld` a multiple of KPF elements, and so is the contiguous extent (callers pack what is not).
// K-contiguous (KS = false): element (row, k) at p[row * ld + k].  K-strided (KS = true): element (row, k) at p[k * ld + row].
struct Operand {
  const void* p;
  long long ld;
};

// One operand's staging registers for a tile of R rows x BK, 256 threads.
template <class T, bool KS, int R>
struct Stage {
  static constexpr int KPF = Type<T>::KPF, BK = kRowBytes / (int)sizeof(T);
  static constexpr int kChunks = R * 8 / 256;                       // KS = false: 16-byte chunks per thread
  static constexpr int kUnits = 8 * (R / 4), kPer = (kUnits + 255) / 256;  // KS = true: transposing units per thread
  u32x4 c[KS ? 1 : kChunks];
  KsUnit<T> u[KS ? kPer : 1];

  __device__ __forceinline__ void load(const Operand& o, int r0, int rows, int k0, int kend, int tid) {
    const T* __restrict__ p = static_cast<const T*>(o.p);
    if constexpr (!KS) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int f = tid + i * 256, row = f >> 3, ch = f & 7;
        const int gr = min(r0 + row, rows - 1), gk = k0 + ch * KPF;  // rows past the end: any row, their results are not stored
        const u32x4 v = *reinterpret_cast<const u32x4*>(p + gr * o.ld + min(gk, (kend - 1) / KPF * KPF));
        c[i] = gk < kend ? v : u32x4{0, 0, 0, 0};
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int f = tid + i * 256;
        if (kUnits % 256 != 0 && f >= kUnits) break;
        const int kg = f / (R / 4), cq = f % (R / 4);
        const int gr = min(r0 + 4 * cq, rows - 4);
#pragma unroll
        for (int j = 0; j < KPF; ++j) {
          const int gk = k0 + kg * KPF + j;
          using V = decltype(u[i].v[0] + u[i].v[0]);
          const V v = *reinterpret_cast<const V*>(p + min(gk, kend - 1) * o.ld + gr);
          u[i].v[j] = gk < kend ? v : V(0);
        }
      }
    }
  }
  __device__ __forceinline__ void store(char* __restrict__ tile, int tid) const {
    if constexpr (!KS) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int f = tid + i * 256;
        *reinterpret_cast<u32x4*>(tile + swz(f >> 3, f & 7)) = c[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int f = tid + i * 256;
        if (kUnits % 256 != 0 && f >= kUnits) break;
        const int kg = f / (R / 4), cq = f % (R / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4*>(tile + swz(4 * cq + j, kg)) = u[i].column(j);
      }
    }
  }
};

// Tile coordinates of workgroup `id` of `total`: workgroups go round the eight XCDs, so each XCD is given one contiguous
// eighth of the tiles, whose operand panels then meet in its own L2.  A label for placement only; any mapping is right.
__device__ __forceinline__ int xcd_tile(int id, int total) {
  const int q = total >> 3, r = total & 7, x = id & 7;
  return x * q + min(x, r) + (id >> 3);
}

struct Shape {
  int M, N, K;      // output [M, N] (N contiguous), contraction K.  A K-contiguous operand is readable, and zero, up to the
                    // next multiple of KPF behind K; a K-strided one has K rows, readable to the next multiple of KPF columns
  int kper;         // k of one split (a multiple of BK unless there is one split)
};

// The product of one BM x BN tile: acc[i][j] is the 32x32 tile of output columns n0 + 32 (wn * NI + i) + ..., output rows
// m0 + 32 (wm * MJ + j) + ...  256 threads, waves 2 x 2.  `lds` holds 2 * (BM + BN) * 128 bytes.
// X: output rows (M), Y: output columns (N).
template <class T, bool XKS, bool YKS, int BM, int BN>
__device__ __forceinline__ void tile_product(f32x16 (&acc)[BN / 64][BM / 64], char* __restrict__ lds, const Operand& X,
                                             const Operand& Y, const Shape& s, int m0, int n0, int kbeg, int kend) {
  constexpr int BK = kRowBytes / (int)sizeof(T);
  constexpr int NI = BN / 64, MJ = BM / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = lane & 31, h = lane >> 5, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  if (kbeg >= kend) return;
  char* const xt[2] = {lds, lds + BM * kRowBytes};
  char* const yt[2] = {lds + 2 * BM * kRowBytes, lds + (2 * BM + BN) * kRowBytes};
  Stage<T, XKS, BM> sx;
  Stage<T, YKS, BN> sy;
  // a padded contiguous extent bounds what a row clamp may touch
  const int xr = XKS ? (s.M + Type<T>::KPF - 1) / Type<T>::KPF * Type<T>::KPF : s.M;
  const int yr = YKS ? (s.N + Type<T>::KPF - 1) / Type<T>::KPF * Type<T>::KPF : s.N;
  sx.load(X, m0, xr, kbeg, kend, tid);
  sy.load(Y, n0, yr, kbeg, kend, tid);
  sx.store(xt[0], tid);
  sy.store(yt[0], tid);
  __syncthreads();
  int b = 0;
  for (int k = kbeg; k < kend; k += BK, b ^= 1) {
    const bool more = k + BK < kend;
    if (more) {
      sx.load(X, m0, xr, k + BK, kend, tid);
      sy.load(Y, n0, yr, k + BK, kend, tid);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x4 fy[NI], fx[MJ];
#pragma unroll
      for (int i = 0; i < NI; ++i) fy[i] = frag(yt[b], (wn * NI + i) * 32 + r, 2 * g + h);
#pragma unroll
      for (int j = 0; j < MJ; ++j) fx[j] = frag(xt[b], (wm * MJ + j) * 32 + r, 2 * g + h);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) mma<T>(acc[i][j], fy[i], fx[j]);
    }
    if (more) {
      sx.store(xt[b ^ 1], tid);
      sy.store(yt[b ^ 1], tid);
    }
    __syncthreads();
  }
}

// Calls fn(m, n, quad) for every quad of four consecutive output columns this lane holds, tile by tile.
template <int BM, int BN, class F>
__device__ __forceinline__ void for_quads(f32x16 (&acc)[BN / 64][BM / 64], int m0, int n0, F&& fn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h = lane >> 5, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int j = 0; j < BM / 64; ++j)
#pragma unroll
    for (int i = 0; i < BN / 64; ++i)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 v = {acc[i][j][4 * a], acc[i][j][4 * a + 1], acc[i][j][4 * a + 2], acc[i][j][4 * a + 3]};
        fn(m0 + (wm * (BM / 64) + j) * 32 + r, n0 + (wn * (BN / 64) + i) * 32 + 8 * a + 4 * h, v);
      }
}

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

// ---- host side ----------------------------------------------------------------------------------------------
inline long long pad_to(long long n, int m) { return (n + m - 1) / m * m; }
inline int dtype_bytes(int dtype) { return dtype == TT_F32 ? 4 : 2; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Can a [rows, cols] matrix of row stride ld be read in 16-byte chunks as it is?
inline bool packed_ok(const void* p, long long ld, long long cols, int dtype) {
  const int kpf = 16 / dtype_bytes(dtype);
  return tt_aligned16(p) && ld % kpf == 0 && cols % kpf == 0;
}
// bytes of its packed copy (row stride padded to 16 bytes, the padding zero), 0 if it needs none
inline size_t pack_bytes(const void* p, long long ld, long long rows, long long cols, int dtype) {
  if (packed_ok(p, ld, cols, dtype)) return 0;
  return align256((size_t)rows * (size_t)pad_to(cols, 16 / dtype_bytes(dtype)) * dtype_bytes(dtype));
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
int tt_grad_splits(long long M, long long N, long long K);

// packs a [rows, cols] matrix (row stride ld elements of `width` bytes) to row stride `ldp`, zeros behind cols (linear.hip)
int tt_launch_pack(const void* src, long long ld, void* dst, long long ldp, long long rows, long long cols, int width,
                   hipStream_t st);
