// linear_act — y = act(x W^T + b) + r with one epilogue, and its gradients.
//
//   forward   z = x W^T + b (fp32), y = act(z) + r rounded once; z is kept (rounded to the type) for the backward pass
//   backward  dz = dy act'(z), db = column sums of dz       one pass over dy and z (db before dz is rounded)
//             dx = dz W                                     K-strided W, transposed on its way into LDS
//             dW = dz^T x                                   both operands K-strided, contraction over the rows split
//
// 2 M N K operations each product; bound by the matrix units from a few hundred rows on, by the epilogue's bytes at small K.
//
// 16-bit types round z where it is kept (in fp32 twice the bytes, written and read) and dz where
// it becomes the products' operand (matrix instructions take no wider one beside 16 bits): the gradients of 16384 x 1024 -> 4096 in
// bf16 are 2.4e-3 of their size from exact, their own rounding is 1.7e-3 of it.
//
// Replaces the nn.Linear (+ activation, + residual add) calls of the frozen encoder of backend/model.py:51-52.
#include <type_traits>
#include "mfma_tile.h"

using namespace ttm;

namespace {

constexpr float kRsqrt2 = 0.70710678118654752f, kRsqrt2Pi = 0.39894228040143268f;
constexpr float kGeluC = 0.79788456080286536f, kGeluA = 0.044715f;

// Phi(z) = erfc(-z / sqrt 2) / 2 and e = exp(-z^2 / 2), which gelu's derivative needs as well.  erfc(a) = t Q(t) exp(-a^2) with
// t = 1 / (1 + p a), a = |z| / sqrt 2, no cancellation on the negative side, where gelu's values are small: Q's error has to be
// small relative to erfc, not only absolutely.  Q is a Chebyshev fit to exp(a^2) erfc(a) / t on 0 <= a <= 10.  16-bit results: p =
// 0.48, degree 6, absolute error of Phi 1.5e-7, relative 2e-5 down to the smallest normal float (z = -13), of which the rounding of
// exp's argument is half; a 200th of bf16's rounding, a 24th of fp16's.  float: p = 0.5, degree 8 (relative error 4e-8).  erff cost
// a quarter of the float epilogue's time.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float a = fabsf(z) * kRsqrt2;
  e = __builtin_amdgcn_exp2f(-1.4426950408889634f * (a * a));
  float q, t;
  if constexpr (FAST) {
    t = __builtin_amdgcn_rcpf(fmaf(0.48f, a, 1.f));
    q = fmaf(t, 0.08723334223031998f, -0.39258500933647156f);
    q = fmaf(t, q, 0.5168355703353882f);
    q = fmaf(t, q, -0.05077535659074783f);
    q = fmaf(t, q, 0.30745595693588257f);
    q = fmaf(t, q, 0.26038721203804016f);
    q = fmaf(t, q, 0.2714482247829437f);
  } else {
    t = __builtin_amdgcn_rcpf(fmaf(0.5f, a, 1.f));
    q = fmaf(t, -0.05906921625137329f, 0.2845761775970459f);
    q = fmaf(t, q, -0.48720231652259827f);
    q = fmaf(t, q, 0.27806979417800903f);
    q = fmaf(t, q, -0.02662738598883152f);
    q = fmaf(t, q, 0.2026875615119934f);
    q = fmaf(t, q, 0.24310359358787537f);
    q = fmaf(t, q, 0.2823753356933594f);
    q = fmaf(t, q, 0.28208640217781067f);
  }
  const float half = 0.5f * (t * q) * e;
  return z > 0.f ? 1.f - half : half;
}
template <bool FAST>
__device__ __forceinline__ float exp_(float x) {
  return FAST ? __builtin_amdgcn_exp2f(1.4426950408889634f * x) : expf(x);
}
template <bool FAST>
__device__ __forceinline__ float inv_(float x) {
  return FAST ? __builtin_amdgcn_rcpf(x) : 1.f / x;
}

template <int ACT, bool FAST>
__device__ __forceinline__ float act_(float z) {
  if constexpr (ACT == TT_ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == TT_ACT_GELU) {
    float e;
    const float y = z * normal_cdf<FAST>(z, e);
    return z < -40.f ? 0.f : y;  // -inf * 0
  }
  if constexpr (ACT == TT_ACT_GELU_TANH) {  // z / (1 + exp(-2u)) = 0.5 z (1 + tanh u)
    const float u = kGeluC * z * fmaf(kGeluA * z, z, 1.f);
    return z * inv_<FAST>(1.f + exp_<FAST>(-2.f * u));
  }
  if constexpr (ACT == TT_ACT_SILU) return z * inv_<FAST>(1.f + exp_<FAST>(-z));
  return z;
}
// act'(z).  Far out the derivatives are their limits 0 and 1, where z times an exponential could be inf * 0; NaN stays NaN.
template <int ACT, bool FAST>
__device__ __forceinline__ float dact_(float z) {
  if constexpr (ACT == TT_ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if constexpr (ACT == TT_ACT_NONE) return 1.f;
  z = z > 40.f ? 40.f : (z < -40.f ? -40.f : z);
  if constexpr (ACT == TT_ACT_GELU) {
    float e;
    const float p = normal_cdf<FAST>(z, e);
    return fmaf(z * kRsqrt2Pi, e, p);
  }
  if constexpr (ACT == TT_ACT_GELU_TANH) {
    const float u = kGeluC * z * fmaf(kGeluA * z, z, 1.f);
    const float s = inv_<FAST>(1.f + exp_<FAST>(-2.f * u));  // (1 + tanh u) / 2;  1 - tanh^2 = 4 s (1 - s)
    return s + z * 2.f * s * (1.f - s) * kGeluC * fmaf(3.f * kGeluA * z, z, 1.f);
  }
  const float s = inv_<FAST>(1.f + exp_<FAST>(-z));
  return s * fmaf(z, 1.f - s, 1.f);
}

template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {  // uniform
    case TT_ACT_RELU: f(std::integral_constant<int, TT_ACT_RELU>{}); break;
    case TT_ACT_GELU: f(std::integral_constant<int, TT_ACT_GELU>{}); break;
    case TT_ACT_GELU_TANH: f(std::integral_constant<int, TT_ACT_GELU_TANH>{}); break;
    case TT_ACT_SILU: f(std::integral_constant<int, TT_ACT_SILU>{}); break;
    default: f(std::integral_constant<int, TT_ACT_NONE>{}); break;
  }
}

struct FwdArgs {
  Operand X, W;
  Shape s;
  const void *bias, *res;
  void *y, *z;
  long long ldr, ldy;
  int act, vec, gm, gn;  // tiles along M and N
};

// The pre-activation as it is kept: a positive z below fp16's range must not become 0, relu'(z) is 1 there.
template <class T>
__device__ __forceinline__ f32x4 kept(f32x4 v, int act) {
  if (__is_same(T, _Float16) && act == TT_ACT_RELU) {
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = v[c] > 0.f ? fmaxf(v[c], 5.9604645e-8f) : v[c];
  }
  return v;
}

// whole 16-byte chunks, aligned
template <class T, int ACT, class B>
__device__ __forceinline__ void epilogue(B& blk, const FwdArgs& a, char* __restrict__ b0, char* __restrict__ b1, int m0, int n0) {
  using R = typename B::template Rows<T>;
  static_assert(R::WHOLE, "a lane's bias");
  const int n = blk.template row_col<T>(n0, 0), M = a.s.M;
  const bool col = n < a.s.N;
  const T* __restrict__ res = static_cast<const T*>(a.res);
  Chunk<T> bias;
  bias.zero();
  if (a.bias && col) bias.load(static_cast<const T*>(a.bias) + n);
  Chunk<T> rq[R::STEPS];
  blk.template for_rows<T>(
      b0, b1, m0, n0,
      [&](int j) {  // the residual of 32 rows at once
        if (!res) return;
#pragma unroll
        for (int s = 0; s < R::STEPS; ++s) {
          const int m = blk.template row_at<T>(m0, j, s);
          rq[s].zero();
          if (m < M && col) rq[s].load(res + m * a.ldr + n);
        }
      },
      [&](int j, int s, int m, int, f32x4 (&v)[R::Q]) {
        const bool in = m < M && col;
        Chunk<T> z, y;
#pragma unroll
        for (int q = 0; q < R::Q; ++q) {
          v[q] += from_quad<T>(bias.q[q]);
          z.q[q] = to_quad<T>(kept<T>(v[q], ACT));
#pragma unroll
          for (int c = 0; c < 4; ++c) v[q][c] = act_<ACT, sizeof(T) == 2>(v[q][c]);
          if (res) v[q] += from_quad<T>(rq[s].q[q]);
          y.q[q] = to_quad<T>(v[q]);
        }
        if (a.z && in) z.store(static_cast<T*>(a.z) + (long long)m * a.s.N + n);
        if (in) y.store(static_cast<T*>(a.y) + m * a.ldy + n);
      });
}

// float 35841 x 384 -> 1536 with gelu: 383 us, 110 TFLOP/s (the library's product alone reaches 133 on large ones).  bf16 16384 x 1024
// -> 4096 with gelu, residual and kept z: 222 us, 128 of them the product at 1070 TFLOP/s, the rest the epilogue's 400 MB, which
// nothing overlaps (two 128-wide workgroups per compute unit do, at a lower rate: equal; a persistent loop spilled: slower).
// bf16 35841 x 1536 -> 384 with residual: 58 us, 843 tiles of 128 are 1.65 rounds; floor 33 by bytes.
template <class T, class B>
__global__ __launch_bounds__(B::THREADS) __attribute__((amdgpu_waves_per_eu(2))) void linear_fwd_kernel(FwdArgs a) {
  __shared__ __align__(16) char b0[B::BYTES];
  __shared__ __align__(16) char b1[B::BYTES];
  int m0, n0;
  tile_at(xcd_tile(blockIdx.x, gridDim.x), a.gm, a.gn, m0, n0);
  m0 *= B::BM;
  n0 *= B::BN;
  B blk;
  blk.template product<T, false, false>(b0, b1, a.X, a.W, a.s, m0, n0, 0, a.s.K);
  if (!a.vec) {  // columns or strides that are not whole chunks: element by element
    T* __restrict__ z = static_cast<T*>(a.z);
    blk.for_quads(m0, n0, [&](int m, int n, f32x4 v) {
      if (m >= a.s.M || n >= a.s.N) return;
      if (a.bias) v += load_quad<T>(static_cast<const T*>(a.bias), 0, 0, n, a.s.N, false);
      if (z) store_quad<T>(z, a.s.N, m, n, a.s.N, false, kept<T>(v, a.act));
      with_act(a.act, [&](auto tag) {
        for (int c = 0; c < 4; ++c) v[c] = act_<decltype(tag)::value, sizeof(T) == 2>(v[c]);
      });
      if (a.res) v += load_quad<T>(static_cast<const T*>(a.res), a.ldr, m, n, a.s.N, false);
      store_quad<T>(static_cast<T*>(a.y), a.ldy, m, n, a.s.N, false, v);
    });
    return;
  }
  with_act(a.act, [&](auto tag) { epilogue<T, decltype(tag)::value>(blk, a, b0, b1, m0, n0); });
}

// Few rows (a query's tokens): a tile of 64 x 64 leaves most of the chip idle and walks K alone.  Here a workgroup forms 32 x 32
// outputs with eight waves, each on every eighth 32-byte pair of chunks of K, its operands straight from memory into registers
// (up to kFewAhead groups in flight), and the waves' sums meet in LDS, added in wave order.  Weight reads' latency bounds it:
// float 11 x 384 -> 1536 with gelu 6.0 us, 2.4 MB.
constexpr int kFewWaves = 8, kFewAhead = 6;
template <class T>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_kernel(FwdArgs a) {
  constexpr int KPF = Type<T>::KPF;
  __shared__ __align__(16) float red[kFewWaves][32][36];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
  const int m0 = blockIdx.x / a.gn * 32, n0 = blockIdx.x % a.gn * 32, M = a.s.M, N = a.s.N, K = a.s.K;
  const T* __restrict__ x = static_cast<const T*>(a.X.p) + min(m0 + r, M - 1) * a.X.ld + h * KPF;
  const T* __restrict__ w = static_cast<const T*>(a.W.p) + min(n0 + r, N - 1) * a.W.ld + h * KPF;
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  for (int k0 = wave * 2 * KPF; k0 < K; k0 += kFewAhead * kFewWaves * 2 * KPF) {
    u32x4 fx[kFewAhead], fw[kFewAhead];
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int k = k0 + i * kFewWaves * 2 * KPF;
      fx[i] = fw[i] = u32x4{0, 0, 0, 0};
      if (k + h * KPF < K) {  // a chunk that starts inside K is readable, and zero behind it
        fx[i] = *reinterpret_cast<const u32x4*>(x + k);
        fw[i] = *reinterpret_cast<const u32x4*>(w + k);
      }
    }
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i)
      if (k0 + i * kFewWaves * 2 * KPF < K) mma<T>(acc, fw[i], fx[i]);  // uniform
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 v = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    *reinterpret_cast<f32x4*>(&red[wave][r][8 * q + 4 * h]) = v;
  }
  __syncthreads();
  const int row = threadIdx.x >> 4, c = (threadIdx.x & 15) * 2, m = m0 + row;  // two columns per thread
  if (m >= M) return;
  float z[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) {
    z[0] += red[i][row][c];
    z[1] += red[i][row][c + 1];
  }
  with_act(a.act, [&](auto tag) {
    constexpr int ACT = decltype(tag)::value;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = n0 + c + e;
      if (n >= N) break;
      if (a.bias) z[e] += (float)static_cast<const T*>(a.bias)[n];
      if (a.z) static_cast<T*>(a.z)[(long long)m * N + n] = (T)kept<T>(f32x4{z[e], 0.f, 0.f, 0.f}, ACT)[0];
      float y = act_<ACT, sizeof(T) == 2>(z[e]);
      if (a.res) y += (float)static_cast<const T*>(a.res)[m * a.ldr + n];
      static_cast<T*>(a.y)[m * a.ldy + n] = (T)y;
    }
  });
}

// dz = dy act'(z) (written when dz != null, row stride ldz) and, per block of rows, the column sums of dz.  Memory-bound: bf16 16384
// x 4096 with gelu 83 us, 4.9 TB/s of a large copy's 5.1.
// 256 threads = 64 chunks of KPF columns x 4 rows; grid (ceil(N / (64 KPF)), row blocks).
struct DzArgs {
  const void *dy, *z;
  void* dz;
  float* part;  // [gridDim.y, N] or null
  long long lddy, ldz;
  int M, N, rows, act, vec;
};
template <class T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* __restrict__ p, long long ld, int m, int n, int N, bool vec) {
  Chunk<T> c;
  if (vec) {
    c.load(p + m * ld + n);
  } else {
#pragma unroll
    for (int i = 0; i < Type<T>::KPF; ++i) c.q[i >> 2][i & 3] = n + i < N ? p[m * ld + n + i] : (T)0.f;
  }
  return c;
}
template <class T>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs a) {
  constexpr int Q = Chunk<T>::Q, KPF = Type<T>::KPF;
  __shared__ f32x4 red[4][64][Q];
  const int q = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = (blockIdx.x * 64 + q) * KPF;
  const int m1 = min(a.M, (int)(blockIdx.y + 1) * a.rows);
  const T* __restrict__ dy = static_cast<const T*>(a.dy);
  const T* __restrict__ z = static_cast<const T*>(a.z);
  T* __restrict__ dz = static_cast<T*>(a.dz);
  f32x4 sum[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool vec = a.vec;
  if (n < a.N) {
    with_act(a.act, [&](auto tag) {
      constexpr int ACT = decltype(tag)::value;
#pragma unroll 2
      for (int m = blockIdx.y * a.rows + w; m < m1; m += 4) {
        Chunk<T> c = load_chunk<T>(dy, a.lddy, m, n, a.N, vec), zc = c;
        if constexpr (ACT != TT_ACT_NONE) zc = load_chunk<T>(z, a.N, m, n, a.N, vec);
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          f32x4 v = from_quad<T>(c.q[i]);
          if constexpr (ACT != TT_ACT_NONE) {
            const f32x4 zz = from_quad<T>(zc.q[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= dact_<ACT, sizeof(T) == 2>(zz[e]);
          }
          sum[i] += v;
          c.q[i] = to_quad<T>(v);
        }
        if (dz) c.store(dz + m * a.ldz + n);  // ldz covers whole chunks; columns behind N get 0 * act'(0)
      }
    });
  }
  if (!a.part) return;
#pragma unroll
  for (int i = 0; i < Q; ++i) red[w][q][i] = sum[i];
  __syncthreads();
  if (w == 0 && n < a.N) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const f32x4 s = (red[0][q][i] + red[1][q][i]) + (red[2][q][i] + red[3][q][i]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + 4 * i + e < a.N) a.part[(long long)blockIdx.y * a.N + n + 4 * i + e] = s[e];
    }
  }
}

template <class T>
__global__ __launch_bounds__(256) void slab_sum_kernel(const float* __restrict__ slab, int ns, long long n, T* __restrict__ out,
                                                       float alpha, const float* __restrict__ alpha_dev) {
  if (alpha_dev) alpha *= *alpha_dev;
  const long long stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    float v = 0.f;
    for (int z = 0; z < ns; ++z) v += slab[z * n + i];
    out[i] = (T)(v * alpha);
  }
}

__global__ __launch_bounds__(256) void pack_kernel(const char* __restrict__ src, long long ld, char* __restrict__ dst, long long ldp,
                                                   long long rows, long long cols, int width) {
  const long long n = rows * ldp, stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const long long r = i / ldp, c = i - r * ldp;
    if (width == 4)
      reinterpret_cast<float*>(dst)[i] = c < cols ? reinterpret_cast<const float*>(src)[r * ld + c] : 0.f;
    else
      reinterpret_cast<uint16_t*>(dst)[i] = c < cols ? reinterpret_cast<const uint16_t*>(src)[r * ld + c] : (uint16_t)0;
  }
}

// P = X Y, or its parts along K (slabs, added in order by slab_sum: the same inputs give the same bits).  Bound by the matrix
// units: bf16 dx of 16384 x 1024 from 4096 136 us, 1010 TFLOP/s; dw of it in two parts 155 us, 890; dx and dw of 8192 x 30522
// logit gradients, 384 wide, 201 and 207 us, 950 and 930.  Results leave through LDS as whole rows (16-byte stores of a lane's own
// columns: linear's training pass 727 us, 598 like this).
struct GradArgs {
  GradProduct g;
  Shape s;
  int gm, gn, vec;
};
template <class T, bool XKS, class B>
__global__ __launch_bounds__(B::THREADS) __attribute__((amdgpu_waves_per_eu(2))) void grad_product_kernel(GradArgs a) {
  __shared__ __align__(16) char b0[B::BYTES];
  __shared__ __align__(16) char b1[B::BYTES];
  const int tiles = a.gm * a.gn;
  const int id = xcd_tile(blockIdx.x, gridDim.x);
  const int z = id / tiles, t = id - z * tiles;
  int m0, n0;
  tile_at(t, a.gm, a.gn, m0, n0);
  m0 *= B::BM;
  n0 *= B::BN;
  B blk;
  const int kbeg = z * a.s.kper;
  blk.template product<T, XKS, true>(b0, b1, a.g.X, a.g.Y, a.s, m0, n0, kbeg, min(a.s.K, kbeg + a.s.kper));
  const int M = a.s.M, N = a.s.N;
  const bool vec = a.vec;
  const float alpha = a.g.alpha_dev ? a.g.alpha * *a.g.alpha_dev : a.g.alpha;
  if (a.g.slab) {
    float* __restrict__ c = a.g.slab + (long long)z * M * N;
    const bool more = a.g.accumulate;
    if (!vec) {
      blk.for_quads(m0, n0, [&](int m, int n, f32x4 v) {
        if (m >= M) return;
        if (more) v += load_quad<float>(c, N, m, n, N, false);
        store_quad<float>(c, N, m, n, N, false, v);
      });
      return;
    }
    using R = typename B::template Rows<float>;
    f32x4 old[R::STEPS];
    blk.template for_rows<float>(
        b0, b1, m0, n0,
        [&](int j) {
          if (!more) return;
#pragma unroll
          for (int s = 0; s < R::STEPS; ++s) {
            const int m = blk.template row_at<float>(m0, j, s), n = blk.template row_col<float>(n0, s);
            if (m < M && n < N) old[s] = *reinterpret_cast<const f32x4*>(c + (long long)m * N + n);
          }
        },
        [&](int j, int s, int m, int n, f32x4 (&v)[R::Q]) {
          if (more) v[0] += old[s];
          if (m < M && n < N) *reinterpret_cast<f32x4*>(c + (long long)m * N + n) = v[0];
        });
    return;
  }
  T* __restrict__ c = static_cast<T*>(a.g.out);
  const long long ldo = a.g.ldo;
  if (!vec) {
    blk.for_quads(m0, n0, [&](int m, int n, f32x4 v) {
      if (m < M) store_quad<T>(c, ldo, m, n, N, false, v * alpha);
    });
    return;
  }
  using R = typename B::template Rows<T>;
  blk.template for_rows<T>(
      b0, b1, m0, n0, [](int) {},
      [&](int j, int s, int m, int n, f32x4 (&v)[R::Q]) {
        Chunk<T> o;
#pragma unroll
        for (int q = 0; q < R::Q; ++q) o.q[q] = to_quad<T>(v[q] * alpha);
        if (m < M && n < N) o.store(c + m * ldo + n);
      });
}

template <class F>
int with_type(int dtype, F&& f) {
  switch (dtype) {
    case TT_F32: return f(float{});
    case TT_BF16: return f(__bf16{});
    case TT_F16: return f(_Float16{});
    default: return TT_ERR_BAD_DTYPE;
  }
}
// 2^22 columns: 256 packed rows are within a tile's 32-bit offsets
bool shape_ok(int64_t M, int N, int K) { return M >= 0 && M <= 1LL << 30 && N >= 1 && N <= 1 << 22 && K >= 1 && K <= 1 << 22; }
bool known_dtype(int d) { return d == TT_F32 || d == TT_BF16 || d == TT_F16; }
// rows of 16-byte chunks
bool chunk_ok(const void* p, long long ld, int width) { return !p || (tt_aligned16(p) && ld % (16 / width) == 0); }

}  // namespace

int tt_launch_pack(const void* src, long long ld, void* dst, long long ldp, long long rows, long long cols, int width, hipStream_t st) {
  const long long n = rows * ldp;
  if (n == 0) return TT_OK;
  const unsigned g = (unsigned)(n / 1024 + 1 < 8192 ? n / 1024 + 1 : 8192);
  hipLaunchKernelGGL(pack_kernel, dim3(g), dim3(256), 0, st, (const char*)src, ld, (char*)dst, ldp, rows, cols, width);
  TT_CHECK_LAUNCH();
  return TT_OK;
}

int tt_launch_slab_sum(const float* slab, int ns, long long n, void* out, int dtype, float alpha, const float* alpha_dev, hipStream_t st) {
  if (n == 0) return TT_OK;
  const unsigned g = (unsigned)(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096);
  return with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL(slab_sum_kernel<T>, dim3(g), dim3(256), 0, st, slab, ns, n, (T*)out, alpha, alpha_dev);
    TT_CHECK_LAUNCH();
    return (int)TT_OK;
  });
}

// the least estimated time: dx of 8192 x 30522 bf16 logits, 384 wide, by "two workgroups per compute unit" (three parts of 576
// tiles) 352 us, by this 265 with 128-wide tiles (five parts), 201 with 256 x 192 (four, one round)
int tt_grad_splits(long long M, long long N, long long K, int dtype) {
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= 32 && (s == 1 || K / s >= 512); ++s) {  // at least eight 16-bit steps of K each
    double cost;
    pick_tile(M, N, s, dtype, true, &cost);
    // seconds: the slowest compute unit's product; the parts written and read once
    double t = cost * (2. * K / s) / (dtype == TT_F32 ? 5.2e11 : 4.4e12);
    if (s > 1) t += s * 8. * M * N / 4e12 + 4e-6;
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

int tt_launch_grad_product(const GradProduct& g, int dtype, hipStream_t st) {
  GradArgs a{};
  a.g = g;
  const int bk = kRowBytes / dtype_bytes(dtype);
  a.s = Shape{g.M, g.N, g.K, (int)(pad_to((g.K + g.nsplit - 1) / g.nsplit, bk))};
  a.vec = g.slab ? g.N % 4 == 0 && tt_aligned16(g.slab) : chunk_ok(g.out, g.ldo, dtype_bytes(dtype)) && g.N % (16 / dtype_bytes(dtype)) == 0;
  const int b = pick_tile(g.M, g.N, g.nsplit, dtype, true), bm = b == 192 ? 256 : b;
  a.gm = (g.M + bm - 1) / bm;
  a.gn = (g.N + b - 1) / b;
  const long long grid = (long long)a.gm * a.gn * g.nsplit;
  if (grid == 0) return TT_OK;
  TT_REQUIRE(grid <= 0x7fffffffLL, TT_ERR_BAD_SHAPE);
  return with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    auto go = [&](auto* shape) {
      using B = std::remove_pointer_t<decltype(shape)>;
      if (g.xks) hipLaunchKernelGGL((grad_product_kernel<T, true, B>), dim3((unsigned)grid), dim3(B::THREADS), 0, st, a);
      else hipLaunchKernelGGL((grad_product_kernel<T, false, B>), dim3((unsigned)grid), dim3(B::THREADS), 0, st, a);
      TT_CHECK_LAUNCH();
      return (int)TT_OK;
    };
    if constexpr (sizeof(T) == 2)
      if (b == 192) return go(static_cast<Three*>(nullptr));
    return with_block<T>(b, go);
  });
}

extern "C" size_t tt_linear_act_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int N, int K,
                                                int dtype) {
  if (!known_dtype(dtype) || !shape_ok(M, N, K)) return 0;
  return pack_bytes(x, ldx, M, K, dtype) + pack_bytes(w, ldw, N, K, dtype);
}

extern "C" int tt_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                             int64_t ldr, void* y, int64_t ldy, void* preact, int64_t M, int N, int K, int dtype, int act,
                             void* workspace, size_t workspace_bytes, tt_stream_t stream) {
  TT_REQUIRE(known_dtype(dtype), TT_ERR_BAD_DTYPE);
  TT_REQUIRE(act >= TT_ACT_NONE && act <= TT_ACT_SILU, TT_ERR_UNSUPPORTED);
  TT_REQUIRE(shape_ok(M, N, K) && ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), TT_ERR_BAD_SHAPE);
  if (M == 0) return TT_OK;
  TT_REQUIRE(x && w && y, TT_ERR_NULL_POINTER);
  const size_t need = tt_linear_act_workspace_bytes(x, ldx, w, ldw, M, N, K, dtype);
  TT_REQUIRE(need == 0 || workspace, TT_ERR_NULL_POINTER);
  TT_REQUIRE(workspace_bytes >= need, TT_ERR_WORKSPACE);
  TT_REQUIRE(need == 0 || tt_aligned16(workspace), TT_ERR_ALIGNMENT);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int width = dtype_bytes(dtype);
  char* ws = static_cast<char*>(workspace);
  const long long ldp = pad_to(K, 16 / width);
  FwdArgs a{};
  a.X = Operand{x, ldx};
  a.W = Operand{w, ldw};
  if (size_t n = pack_bytes(x, ldx, M, K, dtype)) {
    int rc = tt_launch_pack(x, ldx, ws, ldp, M, K, width, st);
    if (rc != TT_OK) return rc;
    a.X = Operand{ws, ldp};
    ws += n;
  }
  if (pack_bytes(w, ldw, N, K, dtype)) {
    int rc = tt_launch_pack(w, ldw, ws, ldp, N, K, width, st);
    if (rc != TT_OK) return rc;
    a.W = Operand{ws, ldp};
  }
  a.s = Shape{(int)M, N, K, K};
  a.bias = bias; a.res = residual; a.y = y; a.z = preact; a.ldr = ldr; a.ldy = ldy; a.act = act;
  a.vec = N % (16 / width) == 0 && chunk_ok(bias, 0, width) && chunk_ok(residual, ldr, width) && chunk_ok(y, ldy, width) && chunk_ok(preact, N, width);
  // one round of 32 x 32 workgroups: measured against 64-wide tiles, K = 384 / 1536, N = 1536 / 384, gelu: 11 rows float 11.0 ->
  // 5.5 us / 30.3 -> 14.6, bf16 4.5 -> 3.6 / 8.6 -> 6.3; at two rounds (N = 1536, 256 rows) 11.6 against 11.2, bf16 4.8 against 5.5
  if (((M + 31) / 32) * ((N + 31) / 32) <= 256) {
    a.gm = (int)((M + 31) / 32);
    a.gn = (N + 31) / 32;
    return with_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      hipLaunchKernelGGL(linear_few_kernel<T>, dim3((unsigned)(a.gm * a.gn)), dim3(64 * kFewWaves), 0, st, a);
      TT_CHECK_LAUNCH();
      return (int)TT_OK;
    });
  }
  const int b = pick_tile(M, N, 1, dtype);
  a.gm = (int)((M + b - 1) / b);
  a.gn = (N + b - 1) / b;
  const long long grid = (long long)a.gm * a.gn;
  TT_REQUIRE(grid <= 0x7fffffffLL, TT_ERR_BAD_SHAPE);
  return with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_block<T>(b, [&](auto* shape) {
      using B = std::remove_pointer_t<decltype(shape)>;
      hipLaunchKernelGGL((linear_fwd_kernel<T, B>), dim3((unsigned)grid), dim3(B::THREADS), 0, st, a);
      TT_CHECK_LAUNCH();
      return (int)TT_OK;
    });
  });
}

namespace {
struct BwdPlan {
  bool own_dz;        // dz is written to the workspace (an activation, or a dy that cannot be read in 16-byte chunks)
  long long ldz;
  int splits, row_blocks, rows;
  size_t dz, x, w, slab, part, total;
};
BwdPlan bwd_plan(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int N, int K,
                 int dtype, int act, bool need_dx, bool need_dw) {
  BwdPlan p{};
  const int width = dtype_bytes(dtype);
  p.own_dz = act != TT_ACT_NONE || !packed_ok(dy, lddy, N, dtype);
  p.ldz = p.own_dz ? pad_to(N, 16 / width) : lddy;
  p.splits = need_dw ? tt_grad_splits(N, K, M, dtype) : 1;
  const long long gx = (N + 1024 / width - 1) / (1024 / width);
  long long rb = (1024 + gx - 1) / gx;
  if (rb > (M + 15) / 16) rb = (M + 15) / 16;
  if (rb < 1) rb = 1;
  p.rows = (int)((M + rb - 1) / rb);
  if (p.rows < 1) p.rows = 1;
  p.row_blocks = (int)((M + p.rows - 1) / p.rows);
  if (p.row_blocks < 1) p.row_blocks = 1;
  p.dz = p.own_dz && (need_dx || need_dw) ? align256((size_t)M * p.ldz * width) : 0;
  p.x = need_dw ? pack_bytes(x, ldx, M, K, dtype) : 0;
  p.w = need_dx ? pack_bytes(w, ldw, N, K, dtype) : 0;
  p.slab = p.splits > 1 ? align256((size_t)p.splits * N * K * 4) : 0;
  p.part = align256((size_t)p.row_blocks * N * 4);
  p.total = p.dz + p.x + p.w + p.slab + p.part;
  return p;
}
}  // namespace

extern "C" size_t tt_linear_act_bwd_workspace_bytes(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w,
                                                    int64_t ldw, int64_t M, int N, int K, int dtype, int act) {
  if (!known_dtype(dtype) || !shape_ok(M, N, K)) return 0;
  return bwd_plan(dy, lddy, x, ldx, w, ldw, M, N, K, dtype, act, w != nullptr, x != nullptr).total;
}

extern "C" int tt_linear_act_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                 const void* preact, void* dx, void* dw, void* dbias, int64_t M, int N, int K, int dtype, int act,
                                 void* workspace, size_t workspace_bytes, tt_stream_t stream) {
  TT_REQUIRE(known_dtype(dtype), TT_ERR_BAD_DTYPE);
  TT_REQUIRE(act >= TT_ACT_NONE && act <= TT_ACT_SILU, TT_ERR_UNSUPPORTED);
  TT_REQUIRE(shape_ok(M, N, K) && lddy >= N && ldx >= K && ldw >= K, TT_ERR_BAD_SHAPE);
  TT_REQUIRE(workspace, TT_ERR_NULL_POINTER);
  TT_REQUIRE(M == 0 || (dy && (!dx || w) && (!dw || x) && (act == TT_ACT_NONE || preact)), TT_ERR_NULL_POINTER);
  TT_REQUIRE(tt_aligned16(workspace), TT_ERR_ALIGNMENT);
  const BwdPlan p = bwd_plan(dy, lddy, x, ldx, w, ldw, M, N, K, dtype, act, dx != nullptr, dw != nullptr);
  TT_REQUIRE(workspace_bytes >= p.total, TT_ERR_WORKSPACE);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int width = dtype_bytes(dtype);
  int rc;
  if (M == 0) {  // empty sums
    if (dw && (rc = tt_launch_slab_sum(nullptr, 0, (long long)N * K, dw, dtype, 0.f, nullptr, st)) != TT_OK) return rc;
    if (dbias && (rc = tt_launch_slab_sum(nullptr, 0, N, dbias, dtype, 0.f, nullptr, st)) != TT_OK) return rc;
    return TT_OK;
  }
  char* ws = static_cast<char*>(workspace);
  char* dz = ws;              ws += p.dz;
  char* xp = ws;              ws += p.x;
  char* wp = ws;              ws += p.w;
  float* slab = (float*)ws;   ws += p.slab;
  float* part = (float*)ws;
  Operand Z{dy, lddy}, X{x, ldx}, W{w, ldw};
  const bool products = dx || dw;
  const bool write_dz = p.own_dz && products;
  if (write_dz || dbias) {
    DzArgs a{};
    a.dy = dy; a.z = preact; a.dz = write_dz ? dz : nullptr; a.part = dbias ? part : nullptr;
    a.lddy = lddy; a.ldz = p.ldz; a.M = (int)M; a.N = N; a.rows = p.rows; a.act = act;
    a.vec = N % (16 / width) == 0 && chunk_ok(dy, lddy, width) && chunk_ok(act == TT_ACT_NONE ? nullptr : preact, N, width);
    rc = with_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      hipLaunchKernelGGL(linear_dz_kernel<T>, dim3((N + 1024 / width - 1) / (1024 / width), p.row_blocks), dim3(256), 0, st, a);
      TT_CHECK_LAUNCH();
      return (int)TT_OK;
    });
    if (rc != TT_OK) return rc;
    if (dbias && (rc = tt_launch_slab_sum(part, p.row_blocks, N, dbias, dtype, 1.f, nullptr, st)) != TT_OK) return rc;
  }
  if (write_dz) Z = Operand{dz, p.ldz};
  if (dx) {
    if (p.w) {
      rc = tt_launch_pack(w, ldw, wp, pad_to(K, 16 / width), N, K, width, st);
      if (rc != TT_OK) return rc;
      W = Operand{wp, pad_to(K, 16 / width)};
    }
    GradProduct g{};
    g.X = Z; g.Y = W; g.M = (int)M; g.N = K; g.K = N; g.xks = 0; g.nsplit = 1; g.out = dx; g.ldo = K; g.alpha = 1.f;
    rc = tt_launch_grad_product(g, dtype, st);
    if (rc != TT_OK) return rc;
  }
  if (dw) {
    if (p.x) {
      rc = tt_launch_pack(x, ldx, xp, pad_to(K, 16 / width), M, K, width, st);
      if (rc != TT_OK) return rc;
      X = Operand{xp, pad_to(K, 16 / width)};
    }
    GradProduct g{};
    g.X = Z; g.Y = X; g.M = N; g.N = K; g.K = (int)M; g.xks = 1; g.nsplit = p.splits; g.alpha = 1.f;
    if (p.splits > 1) g.slab = slab; else { g.out = dw; g.ldo = K; }
    rc = tt_launch_grad_product(g, dtype, st);
    if (rc != TT_OK) return rc;
    if (p.splits > 1) return tt_launch_slab_sum(slab, p.splits, (long long)N * K, dw, dtype, 1.f, nullptr, st);
  }
  return TT_OK;
}
