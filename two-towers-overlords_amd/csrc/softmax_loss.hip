// softmax_loss — cross entropy over a large set of candidates without keeping the logits, and its gradients.
//
//   l_ij = scale x_i.w_j,  lse_i = log sum_j exp l_ij,  loss_i = lse_i - l_i,target
//   G_ij = c_i (exp(l_ij - lse_i) - [j = target_i]),  dx = scale G w,  dw = scale G^T x
//
// A target that is nearly certain has G = c (p - 1), of which fp32's lse leaves few digits (float, logits up to 20: 5e-6 of dx), so
// where a piece holds whole rows (float always) the target's entry is minus the sum of the row's others, in 16-bit types if the
// target's p is above 1/4.  Elsewhere an entry within twice lse's rounding of 0 is 0.
//
// Forward: the product's epilogue leaves each row's maximum and sum of a tile's candidates (fp32, base 2); a second launch
// joins them.  Backward: G is recomputed from x, w and lse into the workspace piece by piece.  16-bit types take pieces of the
// candidates (dw of a piece is final, dx is summed in fp32 over the pieces), float pieces of the rows (the other way round).
// 8 N V D operations instead of 6 with stored logits.
//
// G is rounded to the operands' type (it feeds matrix instructions).  float takes c as it is; 16-bit types take c / max|c|, so that
// the rounding of a mean's 1 / N is not in every target's entry (bf16: up to 2^-8 of all of dx), fp16 times 2^14, which keeps its
// precision down to 2^-28 of the largest.  The products' epilogues take the factor out again.
//
// The candidates of the same group as a row (cand_ids[j] == row_ids[i], j not the target) are left out of its sum.  A row without a
// target keeps candidate 0: its lse is defined, and nothing but lse depends on it.
#include <type_traits>
#include "mfma_tile.h"

using namespace ttm;

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.9259629911e-8f;  // log2 e = the sum
constexpr float kF16Up = 16384.f;

struct Args {
  Operand X, W;
  Shape s;               // M rows, N candidates (all of them, or a piece), K features
  const long long *target, *rid, *cid;
  long long ignore;
  int v0, V, gm, gn;     // first candidate of the piece; candidates in all; tiles along the rows and the candidates
  float scale2;          // scale * log2 e
  float2* part;          // [gn, M] (maximum, sum) of a tile's candidates
  float* others;         // backward, where a piece holds whole rows: [row_parts, M] sums of G's entries, the target's left out
  int* near;             // 16-bit: [M] is the target's p large?
  float scale;
  float* tlogit;         // [M] the target's x.w
  const float *lse, *coef, *cmax;  // backward
  void* G;
  long long ldg;
};

// Is candidate j left out of the row's sum (its own group, or behind the last)?
__device__ __forceinline__ bool left_out(const Args& a, int j, long long t, long long rid) {
  bool out = j >= a.V;
  if (a.rid) out |= (a.cid[min(j, a.V - 1)] == rid) & (j != t);
  return out;
}

// A lane holds 16 NI candidates of MJ rows: maximum and sum are in-lane, one exchange, then the waves' through LDS.  Six K-steps at 384
// features against an epilogue of an exponential per logit, which nothing overlaps: bf16 8192 x 30522 246 us, 780 TFLOP/s; 203
// rows x 250000 62 us, 192 MB of candidates at 3.1 TB/s (a tile is 256 rows, 203 in use).
template <class T, class B>
__global__ __launch_bounds__(B::THREADS) __attribute__((amdgpu_waves_per_eu(2))) void softmax_lse_kernel(Args a) {
  __shared__ __align__(16) char b0[B::BYTES];
  __shared__ __align__(16) char b1[B::BYTES];
  constexpr int NI = B::NI, MJ = B::MJ;
  int tm, tn;
  tile_at(xcd_tile(blockIdx.x, gridDim.x), a.gm, a.gn, tm, tn);
  const int m0 = tm * B::BM, n0 = tn * B::BN;
  B blk;
  blk.template product<T, false, false>(b0, b1, a.X, a.W, a.s, m0, n0, 0, a.s.K);
  auto& acc = blk.acc;
  const int r = blk.r, h = blk.h, wm = blk.wm, wn = blk.wn;
  __syncthreads();
  float2* red = reinterpret_cast<float2*>(b0);  // [WN][BM]
  const int nw = n0 + wn * NI * 32;             // the wave's first candidate
  const bool plain = !a.rid && nw + NI * 32 <= a.V;
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int ml = (wm * MJ + j) * 32 + r, m = m0 + ml;
    const bool in = m < a.s.M;
    const long long t = in ? a.target[m] : -1;
    const long long at = t - nw;
    if (__any(at >= 0 && at < NI * 32)) {  // some row's target is among these candidates
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (at == i * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) a.tlogit[m] = acc[i][j][e];
    }
    if (!plain) {
      const long long rid = in && a.rid ? a.rid[m] : 0, keep = t == a.ignore ? 0 : t;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (left_out(a, nw + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3), keep, rid)) acc[i][j][e] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[i][j][e]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale2;
    const float base = mx == -INFINITY ? 0.f : -mx;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) part[e & 3] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], a.scale2, base));
    float sum = (part[0] + part[1]) + (part[2] + part[3]);
    sum += __shfl_xor(sum, 32, 64);
    if (h == 0) red[wn * B::BM + ml] = make_float2(mx, sum);
  }
  __syncthreads();
  for (int ml = threadIdx.x; ml < B::BM && m0 + ml < a.s.M; ml += B::THREADS) {
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < B::WN; ++k) mx = fmaxf(mx, red[k * B::BM + ml].x);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < B::WN; ++k) sum = fmaf(red[k * B::BM + ml].y, __builtin_amdgcn_exp2f(red[k * B::BM + ml].x - base), sum);
    a.part[(long long)tn * a.s.M + m0 + ml] = make_float2(mx, sum);
  }
}

// joins the tiles' (maximum, sum) of each row: ROWS rows x 256 / ROWS lanes per workgroup, tiles in a fixed order
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float mx = fmaxf(a.x, b.x), base = mx == -INFINITY ? 0.f : mx;
  // a NaN sum is carried on
  return make_float2(mx, a.y * __builtin_amdgcn_exp2f(a.x - base) + b.y * __builtin_amdgcn_exp2f(b.x - base));
}
template <int ROWS>
__global__ __launch_bounds__(256) void softmax_join_kernel(const float2* __restrict__ part, const float* __restrict__ tlogit,
                                                           const long long* __restrict__ target, long long ignore, int M, int V,
                                                           int gn, float scale2, float* __restrict__ loss, float* __restrict__ lse) {
  constexpr int LANES = 256 / ROWS;
  __shared__ float2 red[256];
  const int rl = threadIdx.x % ROWS, q = threadIdx.x / ROWS, m = blockIdx.x * ROWS + rl;
  float mx = -INFINITY, sum = 0.f;
  if (m < M) {
    for (int t = q; t < gn; t += LANES) {
      const float2 p = part[(long long)t * M + m];
      if (p.x > mx) {
        sum = fmaf(sum, __builtin_amdgcn_exp2f(mx - p.x), p.y);
        mx = p.x;
      } else if (p.y != 0.f) {
        sum = fmaf(p.y, p.x == mx ? 1.f : __builtin_amdgcn_exp2f(p.x - mx), sum);  // also carries a NaN on
      }
    }
  }
  red[threadIdx.x] = make_float2(mx, sum);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (q < o) red[threadIdx.x] = join(red[threadIdx.x], red[threadIdx.x + o * ROWS]);
  }
  if (q != 0 || m >= M) return;
  mx = red[rl].x;
  sum = red[rl].y;
  const float base = mx == -INFINITY ? 0.f : mx;
  // in 64 bits, a row each: a row whose target is nearly certain has a loss far below its lse's rounding
  const double l = log2((double)sum), ln2 = 0.6931471805599453094;
  lse[m] = mx == -INFINITY && sum == 0.f ? -INFINITY : (float)((base + l) * ln2);
  const long long t = target[m];
  if (t >= 0 && t < V && sum > 0.f && sum == __builtin_amdgcn_exp2f(fmaf(tlogit[m], scale2, -base))) {  // the target's term is the whole sum
    loss[m] = 0.f;
    return;
  }
  loss[m] = t == ignore ? 0.f : (t < 0 || t >= V ? NAN : (float)(((double)base - (double)tlogit[m] * scale2 + l) * ln2));
}

// G of a piece of the candidates, [M, ldg] in T; columns behind the last candidate are zero.  The logits' product again, then 500 MB of
// G at 8192 x 30522 bf16: 375 us (product and exponentials 246, the rest the stores, through LDS as whole rows).  Keeping the
// logits instead would write and read them once more and need N V elements.
template <class T, class B>
__global__ __launch_bounds__(B::THREADS) __attribute__((amdgpu_waves_per_eu(2))) void softmax_grad_kernel(Args a) {
  __shared__ __align__(16) char b0[B::BYTES];
  __shared__ __align__(16) char b1[B::BYTES];
  int tm, tn;
  tile_at(xcd_tile(blockIdx.x, gridDim.x), a.gm, a.gn, tm, tn);
  const int m0 = tm * B::BM, n0 = tn * B::BN;
  B blk;
  blk.template product<T, false, false>(b0, b1, a.X, a.W, a.s, m0, n0, 0, a.s.K);
  T* __restrict__ G = static_cast<T*>(a.G);
  // what a row's coefficient is scaled by in G; the products' alpha takes 16-bit types' out again, and has float's already
  const float up = sizeof(T) == 4 ? a.scale : (__is_same(T, _Float16) ? kF16Up : 1.f) / *a.cmax;
  using R = typename B::template Rows<T>;
  blk.template for_rows<T>(
      b0, b1, m0, n0, [](int) {},
      [&](int j, int s, int m, int nl, f32x4 (&v)[R::Q]) {
        if (m >= a.s.M || nl >= a.ldg) return;  // whole rows of lanes; behind ldg whole waves, whose part of `others` is no row_part
        const long long t = a.target[m];
        // the target's entry comes from the others: always in float, for a likely target in 16-bit types
        const bool sums = sizeof(T) == 4 || (a.near && a.near[m]);
        const float lse = a.lse[m], c = t == a.ignore ? 0.f : (t < 0 || t >= a.V ? NAN : a.coef[m] * up);
        // lse in base 2 as two floats; the second one scales the row
        const float lse2 = lse * kLog2e, cp = c * __builtin_amdgcn_exp2f(-fmaf(lse, kLog2e, -lse2) - lse * kLog2eLow);
        const int n = a.v0 + nl;
#pragma unroll
        for (int q = 0; q < R::Q; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[q][e] = cp * __builtin_amdgcn_exp2f(fmaf(v[q][e], a.scale2, -lse2));
        if (t >= n && t < n + 4 * R::Q) {
          const float least = fabsf(c) * fmaf(1.1920929e-7f, fabsf(lse), 2.3841858e-7f);
#pragma unroll
          for (int q = 0; q < R::Q; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + 4 * q + e == t) {
                const float d = v[q][e] - c;  // a target that is the row's only candidate has 0
                v[q][e] = sums || fabsf(d) <= least ? 0.f : d;
              }
        }
        const bool off = t == a.ignore;
        if (off || a.rid || n + 4 * R::Q > a.V) {
          const long long rid = a.rid ? a.rid[m] : 0;
#pragma unroll
          for (int q = 0; q < R::Q; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = (off | left_out(a, n + 4 * q + e, t, rid)) ? 0.f : v[q][e];
        }
        if (sizeof(T) == 4 || __any(sums)) {
          float sum = (v[0][0] + v[0][1]) + (v[0][2] + v[0][3]);
          if constexpr (R::Q == 2) sum += (v[1][0] + v[1][1]) + (v[1][2] + v[1][3]);
#pragma unroll
          for (int o = R::LPR / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
          if (blk.lane % R::LPR == 0) a.others[(long long)(tn * B::WN + blk.wn) * a.s.M + m] = sum;
        }
        Chunk<T> g;
#pragma unroll
        for (int q = 0; q < R::Q; ++q) g.q[q] = to_quad<T>(v[q]);
        g.store(G + m * a.ldg + nl);
      });
}

// near[m]: is the target's p above 1/4?  A wave per row.  (With every row's sums the training pass of 8192 x 30522 bf16 took 1074 us,
// without 993.)
template <class T>
__global__ __launch_bounds__(256) void softmax_near_kernel(Args a, int* __restrict__ near) {
  const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (m >= a.s.M) return;
  const long long t = a.target[m];
  float dot = 0.f;
  if (t >= 0 && t < a.V) {
    const T* __restrict__ x = static_cast<const T*>(a.X.p) + m * a.X.ld;
    const T* __restrict__ w = static_cast<const T*>(a.W.p) + t * a.W.ld;
    for (int k = lane * Type<T>::KPF; k < a.s.K; k += 64 * Type<T>::KPF) {  // zeros behind K
      Chunk<T> u, v;
      u.load(x + k);
      v.load(w + k);
#pragma unroll
      for (int q = 0; q < Chunk<T>::Q; ++q) {
        const f32x4 y = from_quad<T>(u.q[q]) * from_quad<T>(v.q[q]);
        dot += (y[0] + y[1]) + (y[2] + y[3]);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
  if (lane == 0) near[m] = fmaf(dot, a.scale2, -a.lse[m] * kLog2e) > -2.f;
}

// G's target entries, minus the sum of the row's others; 16 rows x 16 lanes per workgroup, parts in a fixed order
template <class T>
__global__ __launch_bounds__(256) void softmax_target_kernel(const float* __restrict__ others, const long long* __restrict__ target,
                                                             const int* __restrict__ near, long long ignore, int M, int V, int parts,
                                                             T* __restrict__ G, long long ldg) {
  __shared__ float red[16][17];
  const int rl = threadIdx.x & 15, q = threadIdx.x >> 4, m = blockIdx.x * 16 + rl;
  float sum = 0.f;
  if (m < M && (!near || near[m]))
    for (int t = q; t < parts; t += 16) sum += others[(long long)t * M + m];
  red[rl][q] = sum;
  __syncthreads();
  if (q != 0 || m >= M) return;
  const long long t = target[m];
  if (t == ignore || t < 0 || t >= V || (near && !near[m])) return;
  sum = 0.f;
  for (int i = 0; i < 16; ++i) sum += red[rl][i];
  G[m * ldg + t] = (T)-sum;
}

// cmax[0] = max |coef| over the rows that have a target (1 if that is infinite, at least 10^-30), cmax[1] = cmax[0] / up
__global__ __launch_bounds__(1024) void softmax_cmax_kernel(const float* __restrict__ coef, const long long* __restrict__ target,
                                                            long long ignore, int M, float up, float* __restrict__ cmax) {
  __shared__ float red[16];
  float v = 0.f;
  for (int m = threadIdx.x; m < M; m += 1024)
    if (target[m] != ignore) v = fmaxf(v, fabsf(coef[m]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) v = fmaxf(v, red[i]);
  v = v == INFINITY ? 1.f : fmaxf(v, 1e-30f);  // 1 / v times 2^14 is finite
  cmax[0] = v;
  cmax[1] = v / up;
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

struct Plan {
  int gn, fwd_tile;
  long long piece, rows;  // candidates (a multiple of 128) and rows of a piece of G
  int pieces, blocks;     // pieces of the candidates, pieces of the rows (one of them is 1)
  int sx, sw;             // splits of the two gradient products
  size_t x, w, part, tlogit, cmax, G, others, near, dx, dw, fwd, bwd;
};
constexpr long long kPieceBytes = 512LL << 20;  // of G; 8192 rows x 30522 bf16 candidates: 64 MB 1421 us, 128 1279, 256 1272, 512 1217
Plan plan(const void* x, long long ldx, const void* w, long long ldw, long long M, int V, int D, int dtype) {
  Plan p{};
  const int width = dtype_bytes(dtype);
  p.fwd_tile = pick_tile(M, V, 1, dtype);
  p.gn = (V + p.fwd_tile - 1) / p.fwd_tile;
  p.x = pack_bytes(x, ldx, M, D, dtype);
  p.w = pack_bytes(w, ldw, V, D, dtype);
  p.part = align256((size_t)p.gn * M * sizeof(float2));
  p.tlogit = align256((size_t)M * 4);
  p.fwd = p.x + p.w + p.part + p.tlogit;
  const long long vp = pad_to(V, 128);
  p.piece = vp;
  p.rows = M;
  p.pieces = p.blocks = 1;
  if (dtype == TT_F32) {
    const long long cap = kPieceBytes / (vp * width) / 128 * 128, reach = (1LL << 32) / (vp * width);  // a tile's 32-bit offsets
    const long long most = cap >= 128 ? cap : (reach < 128 ? reach : 128);
    p.blocks = (int)((M + most - 1) / most);
    p.rows = (M + p.blocks - 1) / p.blocks;
    if (most >= 128) p.rows = pad_to(p.rows, 128);
    if (p.rows > M) p.rows = M;
    p.blocks = (int)((M + p.rows - 1) / p.rows);
  } else {
    const long long cap = kPieceBytes / (M * width) / 128 * 128, most = cap < 1024 ? 1024 : cap;
    p.pieces = (int)((vp + most - 1) / most);
    p.piece = pad_to((vp + p.pieces - 1) / p.pieces, 128);
    p.pieces = (int)((vp + p.piece - 1) / p.piece);
  }
  // whole rows of G: sums of a row's parts, as many as any tile shape has
  if (p.pieces == 1) p.others = align256((size_t)((vp + 63) / 64) * 2 * p.rows * 4);
  if (p.pieces == 1 && dtype != TT_F32) p.near = align256((size_t)p.rows * 4);
  p.sx = tt_grad_splits(p.rows, D, p.piece, dtype);
  p.sw = p.blocks > 1 ? 1 : tt_grad_splits(p.piece, D, M, dtype);  // several blocks of rows add up in dw itself
  p.cmax = 256;
  p.G = align256((size_t)p.rows * p.piece * width);
  p.dx = p.pieces > 1 || p.sx > 1 ? align256((size_t)p.sx * p.rows * D * 4) : 0;
  p.dw = p.sw > 1 ? align256((size_t)p.sw * p.piece * D * 4) : 0;
  p.bwd = p.x + p.w + p.cmax + p.G + p.others + p.near + p.dx + p.dw;
  return p;
}

int check(int64_t ldx, int64_t ldw, int64_t N, int V, int D, int dtype, float scale) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16, TT_ERR_BAD_DTYPE);
  // 2^28 candidates: two rows of float G are within a tile's 32-bit offsets; 2^22 features: 256 packed rows are
  TT_REQUIRE(N >= 0 && N <= 1LL << 30 && V >= 1 && V <= 1 << 28 && D >= 1 && D <= 1 << 22 && ldx >= D && ldw >= D && tt_scale_ok(scale),
             TT_ERR_BAD_SHAPE);
  return TT_OK;
}

int operand(Operand& o, const void* p, long long ld, long long rows, int D, int dtype, size_t bytes, char* ws, hipStream_t st) {
  o = Operand{p, ld};
  if (!bytes) return TT_OK;
  const long long ldp = pad_to(D, 16 / dtype_bytes(dtype));
  o = Operand{ws, ldp};
  return tt_launch_pack(p, ld, ws, ldp, rows, D, dtype_bytes(dtype), st);
}

}  // namespace

extern "C" size_t tt_softmax_loss_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int V, int D,
                                                  int dtype) {
  if (check(ldx, ldw, N, V, D, dtype, 1.f) != TT_OK || N == 0) return 0;
  return plan(x, ldx, w, ldw, N, V, D, dtype).fwd;
}
extern "C" size_t tt_softmax_loss_bwd_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int V, int D,
                                                      int dtype) {
  if (check(ldx, ldw, N, V, D, dtype, 1.f) != TT_OK || N == 0) return 0;
  return plan(x, ldx, w, ldw, N, V, D, dtype).bwd;
}

extern "C" int tt_softmax_loss(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target, const int64_t* row_ids,
                               const int64_t* cand_ids, int64_t N, int V, int D, int dtype, float scale, int64_t ignore_index,
                               float* loss, float* lse, void* workspace, size_t workspace_bytes, tt_stream_t stream) {
  int rc = check(ldx, ldw, N, V, D, dtype, scale);
  if (rc != TT_OK) return rc;
  TT_REQUIRE((row_ids == nullptr) == (cand_ids == nullptr), TT_ERR_NULL_POINTER);
  if (N == 0) return TT_OK;
  TT_REQUIRE(x && w && target && loss && lse && workspace, TT_ERR_NULL_POINTER);
  const Plan p = plan(x, ldx, w, ldw, N, V, D, dtype);
  TT_REQUIRE(workspace_bytes >= p.fwd, TT_ERR_WORKSPACE);
  TT_REQUIRE(tt_aligned16(workspace), TT_ERR_ALIGNMENT);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  Args a{};
  if ((rc = operand(a.X, x, ldx, N, D, dtype, p.x, ws, st)) != TT_OK) return rc;
  ws += p.x;
  if ((rc = operand(a.W, w, ldw, V, D, dtype, p.w, ws, st)) != TT_OK) return rc;
  ws += p.w;
  a.part = (float2*)ws;    ws += p.part;
  a.tlogit = (float*)ws;
  a.s = Shape{(int)N, V, D, D};
  a.target = (const long long*)target; a.rid = (const long long*)row_ids; a.cid = (const long long*)cand_ids;
  a.ignore = ignore_index; a.V = V; a.gn = p.gn; a.scale2 = scale * kLog2e;
  const int b = p.fwd_tile;
  a.gm = (int)((N + b - 1) / b);
  const long long grid = (long long)a.gm * p.gn;
  TT_REQUIRE(grid <= 0x7fffffffLL, TT_ERR_BAD_SHAPE);
  rc = with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_block<T>(b, [&](auto* shape) {
      using B = std::remove_pointer_t<decltype(shape)>;
      hipLaunchKernelGGL((softmax_lse_kernel<T, B>), dim3((unsigned)grid), dim3(B::THREADS), 0, st, a);
      TT_CHECK_LAUNCH();
      return (int)TT_OK;
    });
  });
  if (rc != TT_OK) return rc;
  const bool few = N <= 2048 && p.gn > 64;  // 203 rows x 977 tiles: 24 us with 16 rows per workgroup, the pass 85 -> 67 with two
  const int per = few ? 2 : 16;
  hipLaunchKernelGGL(few ? softmax_join_kernel<2> : softmax_join_kernel<16>, dim3((unsigned)((N + per - 1) / per)), dim3(256), 0, st,
                     a.part, a.tlogit, a.target, a.ignore, (int)N, V, p.gn, a.scale2, loss, lse);
  TT_CHECK_LAUNCH();
  return TT_OK;
}

extern "C" int tt_softmax_loss_bwd(const float* row_coef, const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target,
                                   const int64_t* row_ids, const int64_t* cand_ids, const float* lse, int64_t N, int V, int D,
                                   int dtype, float scale, int64_t ignore_index, void* dx, void* dw, void* workspace,
                                   size_t workspace_bytes, tt_stream_t stream) {
  int rc = check(ldx, ldw, N, V, D, dtype, scale);
  if (rc != TT_OK) return rc;
  TT_REQUIRE((row_ids == nullptr) == (cand_ids == nullptr), TT_ERR_NULL_POINTER);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (N == 0) return dw ? tt_launch_slab_sum(nullptr, 0, (long long)V * D, dw, dtype, 0.f, nullptr, st) : (int)TT_OK;
  TT_REQUIRE(row_coef && x && w && target && lse && workspace, TT_ERR_NULL_POINTER);
  const Plan p = plan(x, ldx, w, ldw, N, V, D, dtype);
  TT_REQUIRE(workspace_bytes >= p.bwd, TT_ERR_WORKSPACE);
  TT_REQUIRE(tt_aligned16(workspace), TT_ERR_ALIGNMENT);
  if (!dx && !dw) return TT_OK;
  const int width = dtype_bytes(dtype);
  char* ws = static_cast<char*>(workspace);
  Args a{};
  if ((rc = operand(a.X, x, ldx, N, D, dtype, p.x, ws, st)) != TT_OK) return rc;
  ws += p.x;
  Operand W;
  if ((rc = operand(W, w, ldw, V, D, dtype, p.w, ws, st)) != TT_OK) return rc;
  ws += p.w;
  float* cmax = (float*)ws;   ws += p.cmax;
  a.G = ws;                   ws += p.G;
  a.others = p.others ? (float*)ws : nullptr;
  ws += p.others;
  a.near = p.near ? (int*)ws : nullptr;
  ws += p.near;
  float* dxs = (float*)ws;    ws += p.dx;
  float* dws = (float*)ws;
  const float* alpha_dev = nullptr;
  if (dtype != TT_F32) {
    hipLaunchKernelGGL(softmax_cmax_kernel, dim3(1), dim3(1024), 0, st, row_coef, (const long long*)target, (long long)ignore_index,
                       (int)N, dtype == TT_F16 ? kF16Up : 1.f, cmax);
    TT_CHECK_LAUNCH();
    alpha_dev = cmax + 1;
  }
  const float alpha = dtype == TT_F32 ? 1.f : scale;
  a.cid = (const long long*)cand_ids;
  a.ignore = ignore_index; a.V = V; a.scale = scale; a.scale2 = scale * kLog2e; a.cmax = cmax; a.ldg = p.piece;
  const Operand X = a.X;
  for (int i = 0; i < p.pieces * p.blocks; ++i) {
    const long long v0 = p.pieces > 1 ? i * p.piece : 0, r0 = p.blocks > 1 ? i * p.rows : 0;
    const int vc = (int)(V - v0 < p.piece ? V - v0 : p.piece), rows = (int)(N - r0 < p.rows ? N - r0 : p.rows);
    a.v0 = (int)v0;
    a.W = Operand{static_cast<const char*>(W.p) + v0 * W.ld * width, W.ld};
    a.X = Operand{static_cast<const char*>(X.p) + r0 * X.ld * width, X.ld};
    a.target = (const long long*)target + r0;
    a.rid = row_ids ? (const long long*)row_ids + r0 : nullptr;
    a.lse = lse + r0;
    a.coef = row_coef + r0;
    a.s = Shape{rows, vc, D, D};
    const int b = pick_tile(rows, vc, 1, dtype);
    a.gn = (vc + b - 1) / b;  // every tile starts at a candidate of the piece; the last one zero-fills behind it
    a.gm = (rows + b - 1) / b;
    const long long grid = (long long)a.gm * a.gn;
    TT_REQUIRE(grid <= 0x7fffffffLL, TT_ERR_BAD_SHAPE);
    rc = with_type(dtype, [&](auto tag) {
      using T = decltype(tag);
      if (a.near) {
        hipLaunchKernelGGL(softmax_near_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, a.near);
        TT_CHECK_LAUNCH();
      }
      return with_block<T>(b, [&](auto* shape) {
        using B = std::remove_pointer_t<decltype(shape)>;
        hipLaunchKernelGGL((softmax_grad_kernel<T, B>), dim3((unsigned)grid), dim3(B::THREADS), 0, st, a);
        TT_CHECK_LAUNCH();
        if (a.others) {
          static_assert(B::WN == 2 && B::NI * 64 == B::BN && 128 % (B::NI * 32) == 0, "row_parts");
          hipLaunchKernelGGL(softmax_target_kernel<T>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a.others, a.target, a.near, a.ignore,
                             rows, V, row_parts(B::BN, a.gn, a.ldg), (T*)a.G, a.ldg);
          TT_CHECK_LAUNCH();
        }
        return (int)TT_OK;
      });
    });
    if (rc != TT_OK) return rc;
    if (dx) {
      GradProduct g{};
      g.X = Operand{a.G, p.piece}; g.Y = a.W; g.M = rows; g.N = D; g.K = vc; g.xks = 0; g.nsplit = p.sx;
      g.alpha = alpha; g.alpha_dev = alpha_dev;
      char* out = static_cast<char*>(dx) + r0 * D * width;
      if (p.dx) { g.slab = dxs; g.accumulate = v0 > 0; } else { g.out = out; g.ldo = D; }
      if ((rc = tt_launch_grad_product(g, dtype, st)) != TT_OK) return rc;
      if (p.dx && v0 + p.piece >= V &&
          (rc = tt_launch_slab_sum(dxs, p.sx, (long long)rows * D, out, dtype, alpha, alpha_dev, st)) != TT_OK)
        return rc;
    }
    if (dw) {
      GradProduct g{};
      g.X = Operand{a.G, p.piece}; g.Y = a.X; g.M = vc; g.N = D; g.K = rows; g.xks = 1; g.nsplit = p.sw;
      g.alpha = alpha; g.alpha_dev = alpha_dev;
      char* out = static_cast<char*>(dw) + v0 * D * width;
      if (p.blocks > 1) { g.slab = (float*)dw; g.accumulate = i > 0; }
      else if (p.sw > 1) g.slab = dws; else { g.out = out; g.ldo = D; }
      if ((rc = tt_launch_grad_product(g, dtype, st)) != TT_OK) return rc;
      if (p.sw > 1 && (rc = tt_launch_slab_sum(dws, p.sw, (long long)vc * D, out, dtype, alpha, alpha_dev, st)) != TT_OK) return rc;
    }
  }
  return TT_OK;
}
