// packed_attention — attention inside documents that are packed back to back, and its gradients.
//
//   s_ij = cap tanh(scale q_i.k_j / cap) - slope |i - j|,  p = softmax_j over the keys query i sees,  o_i = sum_j p_ij v_j
//   sees: same document, key mask set, and "causal" j <= i / "prefix" j <= i or j < prefix[document]
//
// One pass over the keys with a running maximum and sum (fp32, base 2); no score leaves the registers.
//
// Layout.  A wave owns 32 queries (the accumulator's columns, one per lane & 31) and walks tiles of 128 / sizeof(T) keys.  It
// forms S^T = K Q^T, so a lane holds scores of ONE query: a row maximum is an in-lane maximum and one exchange with lane ^ 32,
// and running maximum, sum and rescaling are one register per lane.  O^T = V^T P^T takes P^T straight from the score registers:
// the K rows are read from LDS in an order (`fold`) that puts eight consecutive keys into a 16-bit lane's fragment (float:
// four, in place).  V lies in LDS as in memory and is read across its rows (ds_read_b64_tr_b16).  The backward pass does the same from both sides: one kernel owns
// queries (dq, and delta = dO.O), one owns keys (dk, dv); each recomputes S.  No atomics: results do not depend on the order.
//
// Which document a workgroup works on: document b gets floor(cu[b] / BM) + b as its first tile, which leaves every document
// at least as many tiles as it has blocks of BM rows; a workgroup finds its document with a 64-wide search in cu.  So the
// grid follows from T and the number of documents alone, and no length has to be known on the host.  Rows behind the last
// document form a last "document" that is only zero-filled.
#include <type_traits>
#include "mfma_tile.h"

using namespace ttm;

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Args {
  const void *q, *k, *v, *o, *dout;
  long long qt, qh, kt, kh, vt, vh, ot, oh, dot, doh;  // element strides per token and head
  void *out, *dq, *dk, *dv;
  long long dqt, dqh, dkt, dkh, dvt, dvh;
  float *lse, *delta;                                   // [H, T]
  const int *cu, *prefix;
  const float* slopes;
  const unsigned char* keep;
  int T, docs, H, Hkv, Dh, causal, spread, sorted;
  float scale, cap;
};

// Head and tile slot of this workgroup.  Short documents: consecutive slots, all heads of each, on one XCD, whose L2 then holds
// the rows they share.  Long ones (spread): neighbours go round the XCDs, which evens out documents of different lengths and
// the triangle of a causal mask; `last_first`: the tiles with the longest rows of keys first.
__device__ __forceinline__ void place(const Args& a, int heads, bool last_first, int& head, int& slot) {
  int id = blockIdx.x;
  if (!a.spread) id = xcd_tile(id, gridDim.x);
  else if (last_first && !a.sorted) id = gridDim.x - 1 - id;
  head = id % heads;
  slot = id / heads;
}

struct Where {
  int doc, start, len, tile;
  bool tail;
};

// the document and tile of workgroup slot t (see above); every lane gets the same answer
__device__ __forceinline__ Where locate(const int* __restrict__ cu, int docs, int T, int t, int bm) {
  const int lane = threadIdx.x & 63;
  auto at = [&](int b) { return min(max(cu[b], 0), T); };
  int lo = 0, cnt = docs + 1;
  while (cnt > 1) {
    const int step = (cnt + 63) >> 6, b = lo + lane * step;
    const bool in = b < lo + cnt;
    const unsigned long long m = __ballot(in && at(in ? b : lo) / bm + (in ? b : lo) <= t);
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    const int end = lo + cnt;
    lo += k * step;
    cnt = min(step, end - lo);
  }
  Where w;
  w.doc = __builtin_amdgcn_readfirstlane(lo);
  w.start = at(w.doc);
  w.tail = w.doc == docs;
  const int e = w.tail ? T : max(at(w.doc + 1), w.start);
  w.len = e - w.start;
  w.tile = t - (w.start / bm + w.doc);
  return w;
}

// The same with the tiles sorted by their place in their document, for at most 64 documents: the longest rows of a triangle
// first, whatever the documents' lengths.  last_first: the last tiles (they see the most keys), else the first ones (their keys
// are seen by the most queries).  Lane b holds document b's tile count; a ballot counts the documents that reach a tile.
__device__ __forceinline__ Where locate_sorted(const int* __restrict__ cu, int docs, int T, int rank, int bm, bool last_first) {
  const int lane = threadIdx.x & 63;
  auto at = [&](int b) { return min(max(cu[b], 0), T); };
  const int s = lane < docs ? at(lane) : 0, e = lane < docs ? max(at(lane + 1), s) : 0, tiles = (e - s + bm - 1) / bm;
  int top = tiles;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
  top = __builtin_amdgcn_readfirstlane(top);
  Where w;
  w.tail = false;
  for (int i = 0; i < top; ++i) {
    const int k = last_first ? top - 1 - i : i;
    unsigned long long m = __ballot(tiles > k);
    const int n = __builtin_popcountll(m);
    if (rank >= n) {
      rank -= n;
      continue;
    }
    while (rank-- > 0) m &= m - 1;
    w.doc = __builtin_ctzll(m);
    w.start = __builtin_amdgcn_readlane(s, w.doc);
    w.len = __builtin_amdgcn_readlane(e, w.doc) - w.start;
    w.tile = k;
    return w;
  }
  w.tail = true;
  w.doc = docs;
  w.start = at(docs);
  w.len = T - w.start;
  w.tile = rank;
  return w;
}

// row of the K (or Q) image that feeds accumulator row r of a 32-row tile: 16-bit operands swap bits 2 and 3, so that
// accumulator registers 8 g .. 8 g + 7 of lane half h are rows 16 g + 8 h + [0, 8) — a fragment's order
template <class T>
__device__ __forceinline__ int fold(int r) {
  return sizeof(T) == 2 ? ((r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1)) : r;
}
// row (within the 32) that accumulator register i of lane half h holds after fold
template <class T>
__device__ __forceinline__ constexpr int row_of(int i, int h) {
  return sizeof(T) == 2 ? 16 * (i >> 3) + 8 * h + (i & 7) : 8 * (i >> 2) + 4 * h + (i & 3);
}
// fragment g of a folded 32-row accumulator, rounded to T (16-bit: 2 fragments of 8; float: 4 of 4)
template <class T>
__device__ __forceinline__ u32x4 acc_frag(const f32x16& s, int g) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 v = {s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
    return __builtin_bit_cast(u32x4, v);
  } else {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    typedef T t8 __attribute__((ext_vector_type(8)));
    f32x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s[8 * g + i];
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, t8));
  }
}

template <class T, int DP>
struct Dim {
  static constexpr int KPF = Type<T>::KPF;
  static constexpr int TILE = kRowBytes / (int)sizeof(T);     // rows of a tile: 64 (16-bit) or 32 (float)
  static constexpr int SUB = TILE / 32;                       // accumulator tiles of a tile
  static constexpr int PER = 4 / SUB;                         // fragments of an accumulator tile, as the second product's operand
  static constexpr int CH = DP / KPF;                         // 16-byte chunks of a row
  static constexpr int G = CH / 2;                            // matrix instructions' groups along the head
  static constexpr int DT = DP / 32;                          // accumulator tiles along the head
  static constexpr int PITCH = CH < 8 ? CH * 16 : kRowBytes;  // bytes of a row in a block; a block is 128 bytes wide, or the head
  static constexpr int CPB = PITCH / 16;
  static constexpr int BYTES = TILE * CH * 16;                // of a tile's image
  static constexpr int RPG = 1024 / PITCH;                    // rows that a wave fills with one instruction
  static constexpr int GROUPS = BYTES / 1024;
};

__device__ __constant__ uint32_t kZeros[4] = {0, 0, 0, 0};  // what a lane reads for a row that is not there

// The image of a tile of TILE rows of one head, as it lies in memory: read along the rows (the first products) and across
// them (the second ones).  64-byte rows are twisted by bits 2..3 of the row, which has the same effect as `twist`.
template <class T, int DP>
struct Image {
  using D = Dim<T, DP>;
  static __device__ __forceinline__ int tw(int row) { return D::CPB == 8 ? twist(row) : (row >> 2) & 3; }
  static __device__ __forceinline__ const char* at(const char* img, int row, int chunk) {
    return img + (chunk / D::CPB) * (D::TILE * D::PITCH) + row * D::PITCH + ((chunk % D::CPB) ^ tw(row)) * 16;
  }
  static __device__ __forceinline__ u32x4 row(const char* img, int r, int chunk) { return *reinterpret_cast<const u32x4*>(at(img, r, chunk)); }
  // rows [2 KPF g + KPF h, + KPF) of column 32 t + (lane & 31)
  static __device__ __forceinline__ u32x4 col(const char* img, int g, int t, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      const int c = 32 * t + (lane & 31);
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(at(img, 8 * g + 4 * h + j, c >> 2) + (c & 3) * 4);
      return v;
    } else {
      const int j = lane & 15, c = 32 * t + (lane & 16) + 4 * (j & 3), k = 16 * g + 8 * h + (j >> 2), half = (c & 4) * 2;
      const u32x2 lo = tr_read(at(img, k, c >> 3) + half), hi = tr_read(at(img, k + 4, c >> 3) + half);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }
};

// Fills images of tiles of one head.  Rows whose bit of `vis` is clear (behind the document's end, or taken out by the key
// mask) and columns behind the head arrive as zeros: 0 * NaN must not reach a sum.
template <class T, int DP, int WAVES>
struct Filler {
  using D = Dim<T, DP>;
  static constexpr int N = (D::GROUPS + WAVES - 1) / WAVES;
  const char* p;      // the head's rows from the document's start
  long long ld;       // bytes between rows
  bool whole;         // the head fills its padded width

  __device__ __forceinline__ void init(const void* base, long long token_stride, int Dh) {
    p = static_cast<const char*>(base);
    ld = token_stride * (long long)sizeof(T);
    whole = Dh == DP;
  }
  __device__ __forceinline__ void operator()(char* __restrict__ img, int r0, unsigned long long vis, int Dh, int wave, int lane) const {
    const char* __restrict__ src = p + r0 * ld;
    const bool all = whole && vis == (D::TILE == 64 ? ~0ull : 0xffffffffull);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = i * WAVES + wave;
      if (D::GROUPS % WAVES != 0 && g >= D::GROUPS) break;
      const int lin = g * D::RPG + lane / D::CPB, blk = lin / D::TILE, row = lin % D::TILE;
      const int ch = blk * D::CPB + ((lane % D::CPB) ^ Image<T, DP>::tw(row));
      const char* s = src + (uint32_t)(row * (uint32_t)ld) + ch * 16;
      if (!all && !(((vis >> row) & 1) && ch * D::KPF < Dh)) s = reinterpret_cast<const char*>(kZeros);
      lds_fill(s, img + g * 1024);
    }
  }
};

// Which of the tile's rows [r0, r0 + TILE) hold keys: the document's length and the key mask, whose bytes (`kb`, one per
// lane) were asked for a tile earlier.
template <class T>
__device__ __forceinline__ unsigned long long visible(int r0, int len, bool masked, unsigned kb, int lane) {
  constexpr int TILE = kRowBytes / (int)sizeof(T);
  if (masked) return __ballot(lane < TILE && r0 + lane < len && kb != 0);
  const int n = len - r0;
  return n >= TILE ? (TILE == 64 ? ~0ull : 0xffffffffull) : (n <= 0 ? 0ull : (1ull << n) - 1);
}
// this lane's 16 rows of accumulator tile t, as bits row_of(e, 0): `vis` and, where the query sees only the first `seen` rows, those
template <class T>
__device__ __forceinline__ uint32_t lane_bits(unsigned long long vis, int t, int seen, int h) {
  uint32_t w = (uint32_t)(vis >> (32 * t));
  const int n = seen - 32 * t;
  w &= n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
  return w >> ((sizeof(T) == 2 ? 8 : 4) * h);
}

// this lane's fragments of ONE row (its column of the accumulator): chunks 2 g + h
template <class T, int DP>
__device__ __forceinline__ void load_own(u32x4* __restrict__ f, const T* __restrict__ p, bool ok, int Dh, int h) {
#pragma unroll
  for (int g = 0; g < Dim<T, DP>::G; ++g) {
    const int d = (2 * g + h) * Type<T>::KPF;
    f[g] = u32x4{0, 0, 0, 0};
    if (ok && d < Dh) f[g] = *reinterpret_cast<const u32x4*>(p + d);
  }
}

// Scores from raw products, in units in which p = exp2(s * c - ...): raw products where there is no cap (c = scale log2 e, the
// bias's slope divided by the scale), natural units behind a cap.  By value: references kept these in scratch memory.
struct Units {
  float c, slope;
};
__device__ __forceinline__ Units units(const Args& a, int head) {
  Units u;
  const float slope = a.slopes ? a.slopes[head] : 0.f;
  u.c = a.cap > 0.f ? kLog2e : a.scale * kLog2e;
  u.slope = a.cap > 0.f ? slope : slope / a.scale;
  return u;
}
// cap tanh(s scale / cap).  16-bit operands: where no score of the tile is beyond 0.35 cap, the series to x^9 (the next term is
// below 10^-7; not where the cap is so small that the factors of its powers leave fp32: 0 times them would be NaN); else 1 - 2 / (1 + exp 2x), good to 2^-22 absolute and +-1 far out.  float: the accurate function.
template <class T>
__device__ __forceinline__ f32x16 capped(f32x16 s, const Args& a) {
  if (!(a.cap > 0.f)) return s;
  const float r = a.scale / a.cap;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = a.cap * tanhf(s[i] * r);
    return s;
  }
  float top = 0.35f / 4096.f;  // no series from r = 4096 on.  (As a condition of its own it moved scores to scratch memory)
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[i]));
  if (!__any(top * r > 0.35f)) {
    const float r2 = r * r, k9 = 62.f / 2835.f * r2 * r2 * r2 * r2 * a.scale, k7 = -17.f / 315.f * r2 * r2 * r2 * a.scale,
                k5 = 2.f / 15.f * r2 * r2 * a.scale, k3 = -1.f / 3.f * r2 * a.scale;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float u = s[i] * s[i];
      s[i] *= fmaf(u, fmaf(u, fmaf(u, fmaf(u, k9, k7), k5), k3), a.scale);
    }
  } else {
    const float e2 = 2.f * kLog2e * r;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i] = fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[i] * e2)), a.cap);
  }
  return s;
}
// The distance bias of accumulator tile t, -slope |at - row| with row = 32 t + row_of(e, 0) and `at` the lane's own position
// less the tile's (and the lane half's rows).  side > 0 / < 0: the whole tile lies on one side of the wave's own positions, and
// the bias is linear: the part that depends on the row is added here, the lane's own part (`own`) is left to the exponent.
struct Bias {
  float slope, at, own;
  int side;
};
template <class T, bool PLAIN>
__device__ __forceinline__ Bias bias_of(const Args& a, const Units& u, int first, int pos, int r0, int h) {  // first: the wave's first position
  Bias b{u.slope, 0.f, 0.f, 2};
  if (!PLAIN && a.slopes) {
    b.at = (float)(pos - r0 - (sizeof(T) == 2 ? 8 : 4) * h);  // exact: positions are below 2^24 apart
    b.side = first >= r0 + kRowBytes / (int)sizeof(T) - 1 ? 1 : (first + 31 <= r0 ? -1 : 0);
    if (b.side) b.own = -(float)b.side * b.slope * b.at;
  }
  return b;
}
template <class T>
__device__ __forceinline__ f32x16 biased(f32x16 s, const Bias& b, int t) {
  if (b.side == 2) return s;
  if (b.side) {
    const float k = b.side > 0 ? b.slope : -b.slope;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fmaf(k, (float)(32 * t + row_of<T>(i, 0)), s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fmaf(-b.slope, fabsf(b.at - (float)(32 * t + row_of<T>(i, 0))), s[i]);
  }
  return s;
}
// x where bit `bit` of w is set, else `other` (two instructions, no condition code)
__device__ __forceinline__ float pick(uint32_t w, int bit, float x, float other) {
  const int m = (int)(w << (31 - bit)) >> 31;
  return __builtin_bit_cast(float, (__builtin_bit_cast(int, x) & m) | (__builtin_bit_cast(int, other) & ~m));
}
// d x capped score / d (scale q.k) = x (1 - (score / cap)^2)
__device__ __forceinline__ f32x16 through_cap(f32x16 x, f32x16 s, const Args& a) {
  if (a.cap > 0.f) {
    const float r = 1.f / a.cap;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float t = s[i] * r;
      x[i] *= fmaf(-t, t, 1.f);
    }
  }
  return x;
}

// The document's first query sees one key: its p is 1 and its dS exactly 0, which dP less delta, rounded apart, would miss.
__device__ __forceinline__ bool first_alone(const Args& a, int prefix, int len) {
  return len == 1 || ((a.causal || a.prefix) && prefix <= 1);
}

// number of keys (from the document's start) that some query of [i0, i1) sees, and the first from which masking is needed
__device__ __forceinline__ int key_end(const Args& a, int prefix, int i1, int len) {
  if (!a.causal && !a.prefix) return len;
  return min(len, max(i1, prefix));
}

// ------------------------------------------------------------------------------------------------ forward
// K and V tiles stream into one pair of LDS images while the other is in use: one barrier a tile.  A row's sum and output are
// rescaled only when its maximum has grown by 2^8 (the probabilities stay below 2^8, fp32 sums do not mind).
// P is rounded to the type for P V (a matrix instruction takes no wider operand beside V): bf16 o is 1.9e-3 of its size from exact,
// its own rounding 1.7e-3.
// Bound by vector arithmetic where there are a cap and a bias (5 documents of 1001-4096 tokens, heads of 64, bf16, prefix and key
// mask: 198 us, vector instructions in all of a busy compute unit's cycles), by it and by waits at heads of 32 (256 of 8-512, bf16,
// bias: 133 us, vector 76 %, 47 % of the waves' time waiting) and 128 (16 of 700-2048, 16 heads on 4, causal, fp16: 215 us, 640
// TFLOP/s, vector 37 %, matrix 31 %), by bytes and half-filled workgroups for short documents (512 of 12-128, 12 heads of 32, float:
// 97 us, floor 45 by bytes).
template <class T, int DP, int WAVES, bool PLAIN>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(DP == 32 ? 4 : DP == 64 ? 3 : 2))) void attention_fwd_kernel(Args a) {
  using D = Dim<T, DP>;
  constexpr int BM = 32 * WAVES;
  __shared__ __align__(16) char k0img[D::BYTES];
  __shared__ __align__(16) char v0img[D::BYTES];
  __shared__ __align__(16) char k1img[D::BYTES];
  __shared__ __align__(16) char v1img[D::BYTES];
  int head, slot;
  place(a, a.H, true, head, slot);
  const Where w = a.sorted ? locate_sorted(a.cu, a.docs, a.T, slot, BM, true) : locate(a.cu, a.docs, a.T, slot, BM);
  const int i0 = w.tile * BM;
  if (i0 < 0 || i0 >= w.len) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int i = i0 + wave * 32 + r;  // this lane's query, counted in its document
  const bool live = i < w.len;
  const long long tok = w.start + i;
  T* __restrict__ out = static_cast<T*>(a.out) + tok * a.ot + (long long)head * a.oh;
  if (w.tail) {
    if (live) {
      for (int d = h * (DP / 2); d < min(a.Dh, (h + 1) * (DP / 2)); ++d) out[d] = (T)0.f;
      if (h == 0) a.lse[(long long)head * a.T + tok] = -INFINITY;
    }
    return;
  }
  const int kvh = head / (a.H / a.Hkv);
  const T* __restrict__ kp = static_cast<const T*>(a.k) + w.start * a.kt + kvh * a.kh;
  const T* __restrict__ vp = static_cast<const T*>(a.v) + w.start * a.vt + kvh * a.vh;
  const unsigned char* __restrict__ keep = a.keep ? a.keep + w.start : nullptr;
  const int prefix = a.prefix ? min(max(a.prefix[w.doc], 0), w.len) : 0;
  const bool limited = a.causal || a.prefix;
  const int kend = key_end(a, prefix, min(i0 + BM, w.len), w.len);
  const int wend = key_end(a, prefix, min(i0 + wave * 32 + 32, w.len), w.len);  // this wave's own end
  const int seen = limited ? max(i + 1, prefix) : w.len;                       // this query's
  const Units un = units(a, head);
  const float c = un.c;

  u32x4 qf[D::G];
  load_own<T, DP>(qf, static_cast<const T*>(a.q) + tok * a.qt + head * a.qh, live, a.Dh, h);
  f32x16 o[D::DT];
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  Filler<T, DP, WAVES> fk, fv;
  fk.init(kp, a.kt, a.Dh);
  fv.init(vp, a.vt, a.Dh);
  auto mask_byte = [&](int r0) -> unsigned { return keep && lane < D::TILE && r0 + lane < w.len ? keep[r0 + lane] : 0u; };
  unsigned kb = mask_byte(0);
  unsigned long long vis = visible<T>(0, w.len, keep, kb, lane);
  fk(k0img, 0, vis, a.Dh, wave, lane);
  fv(v0img, 0, vis, a.Dh, wave, lane);
  kb = mask_byte(D::TILE);
  const float jump = 8.f / c;  // a row's maximum is followed once it is 2^8 behind: sums stay exact enough, rescaling is rare

  auto tile = [&](int k0, const char* __restrict__ kimg, const char* __restrict__ vimg, char* __restrict__ kn, char* __restrict__ vn) {
    stage_wait();
    const unsigned long long now = vis;
    if (k0 + D::TILE < kend) {
      vis = visible<T>(k0 + D::TILE, w.len, keep, kb, lane);
      fk(kn, k0 + D::TILE, vis, a.Dh, wave, lane);
      fv(vn, k0 + D::TILE, vis, a.Dh, wave, lane);
      kb = mask_byte(k0 + 2 * D::TILE);
    }
    if (k0 >= wend || i0 + wave * 32 >= w.len) return;
    f32x16 s[D::SUB];
    const int rem = wend - k0;
    const bool masked = now != (D::TILE == 64 ? ~0ull : 0xffffffffull) ||
                        (limited && k0 + D::TILE > i0 + wave * 32 + 1 && k0 + D::TILE > prefix);
    const Bias bias = bias_of<T, PLAIN>(a, un, i0 + wave * 32, i, k0, h);
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < D::SUB; ++t) {
      f32x16 acc;
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = 0.f;
      if (32 * t < rem) {  // uniform: not the half of a tile that nobody here sees
#pragma unroll
        for (int g = 0; g < D::G; ++g) mma<T>(acc, Image<T, DP>::row(kimg, 32 * t + fold<T>(r), 2 * g + h), qf[g]);
        if constexpr (!PLAIN) acc = biased<T>(capped<T>(acc, a), bias, t);
        if (masked) {
          const uint32_t bits = lane_bits<T>(now, t, seen - k0, h);
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = pick(bits, row_of<T>(e, 0), acc[e], -INFINITY);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[e]);
      }
      s[t] = acc;
    }
    mx += bias.own;  // the lane halves' own parts differ by their rows
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__any(mx > m + jump || m == -INFINITY)) {
      mx = fmaxf(mx, m);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mx) * c);
      l *= f;
#pragma unroll
      for (int t = 0; t < D::DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] *= f;
      m = mx;
    }
    const float mc = fmaf(bias.own, c, m == -INFINITY ? 0.f : -m * c);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < D::SUB; ++t) {
      if (32 * t >= rem) break;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, mc));
        sum[e & 3] += s[t][e];
      }
#pragma unroll
      for (int g = 0; g < D::PER; ++g) {
        const u32x4 pf = acc_frag<T>(s[t], g);
#pragma unroll
        for (int u = 0; u < D::DT; ++u) mma<T>(o[u], Image<T, DP>::col(vimg, t * D::PER + g, u, lane), pf);
      }
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  for (int k0 = 0; k0 < kend; k0 += 2 * D::TILE) {
    tile(k0, k0img, v0img, k1img, v1img);
    if (k0 + D::TILE < kend) tile(k0 + D::TILE, k1img, v1img, k0img, v0img);
  }
  l += __shfl_xor(l, 32, 64);
  if (!live) return;
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * t + 8 * q + 4 * h;
      const f32x4 v = {o[t][4 * q] * inv, o[t][4 * q + 1] * inv, o[t][4 * q + 2] * inv, o[t][4 * q + 3] * inv};
      if (d < a.Dh) *reinterpret_cast<typename Type<T>::quad*>(out + d) = to_quad<T>(v);
    }
  if (h == 0) a.lse[(long long)head * a.T + tok] = l == 0.f ? -INFINITY : (m * c + __builtin_amdgcn_logf(l)) * kLn2;
}

// ------------------------------------------------------------------------------------------------ dq, delta
// dS = P (dO V^T - delta) d,  dq_i = scale sum_j dS_ij k_j,  delta_i = dO_i . o_i
// dS rounded to 16 bits would cost as much again as dq's own rounding: its product takes dS in two parts (bf16, 256 documents of
// 8-512 tokens, 12 heads of 32, distance bias: this kernel 181 -> 220 us, dq's error 1.5 -> 1.2 roundings; fp16, 16 of 700-2048,
// 16 heads of 128: both passes 1140 -> 1176 us, 1.5 -> 1.2).  Where one tile holds all keys, delta is formed from P and dP before
// dS: with a few keys dS is a small difference, and o's rounding in dO.o was 2 to 3 roundings of dq.
// 10 operations per pair and head element against the forward's 4, 16 exponentials per lane and 32 keys as there: bound by vector
// arithmetic at heads of 32 (209 us, 76 % of a busy compute unit's cycles); at 128 matrix (44 %) and vector instructions (39 %) take
// turns with waits (16 documents of 700-2048, fp16, causal: 333 us, 620 TFLOP/s).
template <class T, int DP, int WAVES, bool PLAIN>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(DP == 32 ? 3 : DP == 64 || sizeof(T) == 2 ? 2 : 1))) void attention_dq_kernel(Args a) {
  using D = Dim<T, DP>;
  constexpr int BM = 32 * WAVES;
  __shared__ __align__(16) char k0img[D::BYTES];
  __shared__ __align__(16) char v0img[D::BYTES];
  __shared__ __align__(16) char k1img[D::BYTES];
  __shared__ __align__(16) char v1img[D::BYTES];
  int head, slot;
  place(a, a.H, true, head, slot);
  const Where w = a.sorted ? locate_sorted(a.cu, a.docs, a.T, slot, BM, true) : locate(a.cu, a.docs, a.T, slot, BM);
  const int i0 = w.tile * BM;
  if (i0 < 0 || i0 >= w.len) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int i = i0 + wave * 32 + r;
  const bool live = i < w.len;
  const long long tok = w.start + i;
  T* __restrict__ dq = static_cast<T*>(a.dq) + tok * a.dqt + (long long)head * a.dqh;
  if (w.tail) {
    if (live)
      for (int d = h * (DP / 2); d < min(a.Dh, (h + 1) * (DP / 2)); ++d) dq[d] = (T)0.f;
    return;
  }
  const int kvh = head / (a.H / a.Hkv);
  const T* __restrict__ kp = static_cast<const T*>(a.k) + w.start * a.kt + kvh * a.kh;
  const T* __restrict__ vp = static_cast<const T*>(a.v) + w.start * a.vt + kvh * a.vh;
  const unsigned char* __restrict__ keep = a.keep ? a.keep + w.start : nullptr;
  const int prefix = a.prefix ? min(max(a.prefix[w.doc], 0), w.len) : 0;
  const bool limited = a.causal || a.prefix;
  const int kend = key_end(a, prefix, min(i0 + BM, w.len), w.len);
  const int wend = key_end(a, prefix, min(i0 + wave * 32 + 32, w.len), w.len);
  const int seen = limited ? max(i + 1, prefix) : w.len;
  const Units un = units(a, head);
  const float c = un.c;

  u32x4 qf[D::G], df[D::G];
  load_own<T, DP>(qf, static_cast<const T*>(a.q) + tok * a.qt + head * a.qh, live, a.Dh, h);
  load_own<T, DP>(df, static_cast<const T*>(a.dout) + tok * a.dot + head * a.doh, live, a.Dh, h);
  float delta = 0.f, lse2 = INFINITY;  // an infinite normaliser: p = 0
  {
    u32x4 of[D::G];
    load_own<T, DP>(of, static_cast<const T*>(a.o) + tok * a.ot + head * a.oh, live, a.Dh, h);
    typedef T tv __attribute__((ext_vector_type(Type<T>::KPF)));
#pragma unroll
    for (int g = 0; g < D::G; ++g) {
      const tv x = __builtin_bit_cast(tv, of[g]), y = __builtin_bit_cast(tv, df[g]);
#pragma unroll
      for (int e = 0; e < Type<T>::KPF; ++e) delta = fmaf((float)x[e], (float)y[e], delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (live) {
      const float t = a.lse[(long long)head * a.T + tok];
      if (t != -INFINITY && !(i == 0 && first_alone(a, prefix, w.len))) lse2 = t * kLog2e;
    }
  }
  float rest[4] = {0.f, 0.f, 0.f, 0.f};  // sum_j p_ij (dp_ij - delta): what the rounding of o left out of delta (sum_j p_ij = 1)
  f32x16 acc[D::DT];
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;

  Filler<T, DP, WAVES> fk, fv;
  fk.init(kp, a.kt, a.Dh);
  fv.init(vp, a.vt, a.Dh);
  auto mask_byte = [&](int r0) -> unsigned { return keep && lane < D::TILE && r0 + lane < w.len ? keep[r0 + lane] : 0u; };
  unsigned kb = mask_byte(0);
  unsigned long long vis = visible<T>(0, w.len, keep, kb, lane);
  fk(k0img, 0, vis, a.Dh, wave, lane);
  fv(v0img, 0, vis, a.Dh, wave, lane);
  kb = mask_byte(D::TILE);

  auto tile = [&](int k0, const char* __restrict__ kimg, const char* __restrict__ vimg, char* __restrict__ kn, char* __restrict__ vn, auto first) {
    stage_wait();
    const unsigned long long now = vis;
    if (k0 + D::TILE < kend) {
      vis = visible<T>(k0 + D::TILE, w.len, keep, kb, lane);
      fk(kn, k0 + D::TILE, vis, a.Dh, wave, lane);
      fv(vn, k0 + D::TILE, vis, a.Dh, wave, lane);
      kb = mask_byte(k0 + 2 * D::TILE);
    }
    if (k0 >= wend || i0 + wave * 32 >= w.len) return;
    const bool masked = now != (D::TILE == 64 ? ~0ull : 0xffffffffull) ||
                        (limited && k0 + D::TILE > i0 + wave * 32 + 1 && k0 + D::TILE > prefix);
    const int rem = wend - k0;
    const Bias bias = bias_of<T, PLAIN>(a, un, i0 + wave * 32, i, k0, h);
    const float off = fmaf(bias.own, c, -lse2);
    f32x16 s, sc;
    auto scores = [&](int t) {  // s = P (dO V^T - delta), sc = the capped scores
      f32x16 dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
      for (int g = 0; g < D::G; ++g) {
        mma<T>(s, Image<T, DP>::row(kimg, 32 * t + fold<T>(r), 2 * g + h), qf[g]);
        mma<T>(dp, Image<T, DP>::row(vimg, 32 * t + fold<T>(r), 2 * g + h), df[g]);
      }
      if constexpr (!PLAIN) {
        sc = capped<T>(s, a);
        s = biased<T>(sc, bias, t);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, off)) * (dp[e] - delta);
      if (masked) {
        const uint32_t bits = lane_bits<T>(now, t, seen - k0, h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = pick(bits, row_of<T>(e, 0), s[e], 0.f);
      }
    };
    if constexpr (decltype(first)::value && sizeof(T) == 2) {
      if (kend <= D::TILE && k0 == 0) {  // all keys are here: delta without o's rounding first, few keys' dS cancel in it
        float sum = 0.f;
        for (int t = 0; t < D::SUB && 32 * t < rem; ++t) {
          scores(t);
#pragma unroll
          for (int e = 0; e < 16; ++e) sum += s[e];
        }
        delta += sum + __shfl_xor(sum, 32, 64);
      }
    }
#pragma unroll
    for (int t = 0; t < D::SUB; ++t) {
      if (32 * t >= rem) break;
      scores(t);
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 16; ++e) rest[e & 3] += s[e];
      }
      if constexpr (!PLAIN) s = through_cap(s, sc, a);
#pragma unroll
      for (int g = 0; g < D::PER; ++g) {
        const u32x4 f = acc_frag<T>(s, g);
#pragma unroll
        for (int u = 0; u < D::DT; ++u) mma<T>(acc[u], Image<T, DP>::col(kimg, t * D::PER + g, u, lane), f);
        if constexpr (sizeof(T) == 2) {  // what the type's bits left of dS
          typedef T t8 __attribute__((ext_vector_type(8)));
          const t8 hi = __builtin_bit_cast(t8, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[8 * g + e] -= (float)hi[e];
          const u32x4 lo = acc_frag<T>(s, g);
#pragma unroll
          for (int u = 0; u < D::DT; ++u) mma<T>(acc[u], Image<T, DP>::col(kimg, t * D::PER + g, u, lane), lo);
        }
      }
    }
  };
  for (int k0 = 0; k0 < kend; k0 += 2 * D::TILE) {
    tile(k0, k0img, v0img, k1img, v1img, std::true_type{});
    if (k0 + D::TILE < kend) tile(k0 + D::TILE, k1img, v1img, k0img, v0img, std::false_type{});
  }
  if constexpr (sizeof(T) == 2) {  // the keys' kernel runs next and takes the better delta
    float r = (rest[0] + rest[1]) + (rest[2] + rest[3]);
    r += __shfl_xor(r, 32, 64);
    delta += r;
  }
  if (live && h == 0) a.delta[(long long)head * a.T + tok] = delta;
  if (!live) return;
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * t + 8 * q + 4 * h;
      const f32x4 v = {acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]};
      if (d < a.Dh) *reinterpret_cast<typename Type<T>::quad*>(dq + d) = to_quad<T>(v * a.scale);
    }
}

// ------------------------------------------------------------------------------------------------ dk, dv
// A wave owns 32 keys (columns) and walks the queries, for every query head that shares the key head:
// dv_j = sum_i p_ij dO_i,  dk_j = scale sum_i dS_ij q_i
// P and dS are rounded to the type once, where dq takes dS in two parts (that would be half as many products again): dk and dv are 2.4e-3
// (bf16) and 3.0e-4 (fp16) of their size from exact, their own rounding is 1.7e-3 and 2.1e-4 of it.
// 8 operations per pair and head element.  256 documents of 8-512 tokens, 12 heads of 32, bf16: 260 us; waits bound it (46 % of the
// waves' time at two waves per SIMD; vector instructions fill 43 % of a busy compute unit's cycles, the statistics, here per
// accumulator row, are 16 reads of lse and delta).  16 of 700-2048, 16 heads of 128 on 4, fp16: 627 us, 440 TFLOP/s: two accumulators
// of the head's width and two operands take 392 registers, one wave per SIMD (vector 22 %, matrix 29 %).
template <class T, int DP, int WAVES, bool PLAIN>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(DP == 32 || (DP == 64 && sizeof(T) == 2) ? 2 : 1))) void attention_dkv_kernel(Args a) {
  using D = Dim<T, DP>;
  constexpr int BM = 32 * WAVES;
  __shared__ __align__(16) char q0img[D::BYTES];
  __shared__ __align__(16) char d0img[D::BYTES];
  __shared__ __align__(16) char q1img[D::BYTES];
  __shared__ __align__(16) char d1img[D::BYTES];
  __shared__ __align__(16) float stat0[2 * D::TILE];
  __shared__ __align__(16) float stat1[2 * D::TILE];
  int kvh, slot;
  place(a, a.Hkv, false, kvh, slot);
  const Where w = a.sorted ? locate_sorted(a.cu, a.docs, a.T, slot, BM, false) : locate(a.cu, a.docs, a.T, slot, BM);
  const int j0 = w.tile * BM;
  if (j0 < 0 || j0 >= w.len) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int j = j0 + wave * 32 + r;  // this lane's key
  const bool in = j < w.len;
  const long long tok = w.start + j;
  T* __restrict__ dk = static_cast<T*>(a.dk) + tok * a.dkt + (long long)kvh * a.dkh;
  T* __restrict__ dv = static_cast<T*>(a.dv) + tok * a.dvt + (long long)kvh * a.dvh;
  if (w.tail) {
    if (in)
      for (int d = h * (DP / 2); d < min(a.Dh, (h + 1) * (DP / 2)); ++d) dk[d] = dv[d] = (T)0.f;
    return;
  }
  const bool live = in && (!a.keep || a.keep[tok] != 0);
  const int rep = a.H / a.Hkv;
  const int prefix = a.prefix ? min(max(a.prefix[w.doc], 0), w.len) : 0;
  const bool limited = a.causal || a.prefix;
  // queries from `first` on see this key; the workgroup starts at its own earliest
  const int first = !limited || j < prefix ? 0 : j;
  const int wfirst = !limited || j0 + wave * 32 < prefix ? 0 : j0 + wave * 32;
  const int bfirst = (!limited || j0 < prefix ? 0 : j0) / D::TILE * D::TILE;
  const float c = units(a, 0).c;
  const bool lone = j0 + wave * 32 == 0 && first_alone(a, prefix, w.len);

  u32x4 kf[D::G], vf[D::G];
  load_own<T, DP>(kf, static_cast<const T*>(a.k) + tok * a.kt + kvh * a.kh, live, a.Dh, h);
  load_own<T, DP>(vf, static_cast<const T*>(a.v) + tok * a.vt + kvh * a.vh, live, a.Dh, h);
  f32x16 ak[D::DT], av[D::DT];
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) ak[t][e] = av[t][e] = 0.f;

  // tiles of queries, head after head of the group: one pipeline
  const int per = bfirst < w.len ? (w.len - bfirst + D::TILE - 1) / D::TILE : 0, total = per * rep;
  const char* const qb = static_cast<const char*>(a.q) + (w.start * a.qt + (long long)kvh * rep * a.qh) * (long long)sizeof(T);
  const char* const db = static_cast<const char*>(a.dout) + (w.start * a.dot + (long long)kvh * rep * a.doh) * (long long)sizeof(T);
  float st[2];  // lse and delta of query (tid) of the tile being filled
  auto issue = [&](int n, char* __restrict__ qi, char* __restrict__ di) {
    const int hq = n / per, q0 = bfirst + (n - hq * per) * D::TILE;
    const unsigned long long vis = visible<T>(q0, w.len, false, 0, lane);
    Filler<T, DP, WAVES> f;
    f.init(qb + hq * a.qh * (long long)sizeof(T), a.qt, a.Dh);
    f(qi, q0, vis, a.Dh, wave, lane);
    f.init(db + hq * a.doh * (long long)sizeof(T), a.dot, a.Dh);
    f(di, q0, vis, a.Dh, wave, lane);
    st[0] = -INFINITY;
    st[1] = 0.f;
    if (tid < D::TILE && q0 + tid < w.len) {
      const long long at = (long long)(kvh * rep + hq) * a.T + w.start + q0 + tid;
      st[0] = a.lse[at];
      st[1] = a.delta[at];
    }
  };
  auto put = [&](float* __restrict__ s) {  // before the barrier that publishes the tile
    if (tid < D::TILE) {
      s[tid] = st[0] == -INFINITY ? INFINITY : st[0] * kLog2e;  // a row that sees nothing, or none: p = 0
      s[D::TILE + tid] = st[1];
    }
  };
  auto tile = [&](int n, const char* __restrict__ qimg, const char* __restrict__ dimg, float* __restrict__ stat,
                  char* __restrict__ qn, char* __restrict__ dn) {
    put(stat);
    stage_wait();
    if (n + 1 < total) issue(n + 1, qn, dn);
    const int hq = n / per, q0 = bfirst + (n - hq * per) * D::TILE;
    if (q0 + D::TILE <= wfirst || j0 + wave * 32 >= w.len) return;
    const Bias bias = bias_of<T, PLAIN>(a, units(a, kvh * rep + hq), j0 + wave * 32, j, q0, h);
    const float off = bias.own * c;
    const bool masked = limited && q0 < j0 + wave * 32 + 31 && j0 + wave * 32 + 31 >= prefix;
#pragma unroll
    for (int t = 0; t < D::SUB; ++t) {
      if (q0 + 32 * t >= w.len) break;
      f32x16 s, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
      for (int g = 0; g < D::G; ++g) {
        mma<T>(s, Image<T, DP>::row(qimg, 32 * t + fold<T>(r), 2 * g + h), kf[g]);
        mma<T>(dp, Image<T, DP>::row(dimg, 32 * t + fold<T>(r), 2 * g + h), vf[g]);
      }
      f32x16 sc;
      if constexpr (!PLAIN) {
        sc = capped<T>(s, a);
        s = biased<T>(sc, bias, t);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // four rows' lse and delta at a time
        const f32x4 ls = *reinterpret_cast<const f32x4*>(stat + 32 * t + row_of<T>(4 * q, h));
        const f32x4 de = *reinterpret_cast<const f32x4*>(stat + D::TILE + 32 * t + row_of<T>(4 * q, h));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 4 * q + i;
          s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, PLAIN ? -ls[i] : off - ls[i]));
          dp[e] = s[e] * (dp[e] - de[i]);
        }
      }
      if (lone && q0 + 32 * t == 0) dp[0] = lane == 0 ? 0.f : dp[0];
      if constexpr (!PLAIN) dp = through_cap(dp, sc, a);
      if (masked) {
        const uint32_t bits = ~lane_bits<T>(~0ull, t, first - q0, h);  // queries from `first` on
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = pick(bits, row_of<T>(e, 0), s[e], 0.f);
          dp[e] = pick(bits, row_of<T>(e, 0), dp[e], 0.f);
        }
      }
#pragma unroll
      for (int g = 0; g < D::PER; ++g) {
        const u32x4 pf = acc_frag<T>(s, g), sf = acc_frag<T>(dp, g);
#pragma unroll
        for (int u = 0; u < D::DT; ++u) {
          mma<T>(av[u], Image<T, DP>::col(dimg, t * D::PER + g, u, lane), pf);
          mma<T>(ak[u], Image<T, DP>::col(qimg, t * D::PER + g, u, lane), sf);
        }
      }
    }
  };
  if (total > 0) issue(0, q0img, d0img);
  for (int n = 0; n < total; n += 2) {
    tile(n, q0img, d0img, stat0, q1img, d1img);
    if (n + 1 < total) tile(n + 1, q1img, d1img, stat1, q0img, d0img);
  }
  if (!in) return;
#pragma unroll
  for (int t = 0; t < D::DT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * t + 8 * q + 4 * h;
      f32x4 x = {ak[t][4 * q], ak[t][4 * q + 1], ak[t][4 * q + 2], ak[t][4 * q + 3]};
      f32x4 y = {av[t][4 * q], av[t][4 * q + 1], av[t][4 * q + 2], av[t][4 * q + 3]};
      x *= a.scale;
      if (!live) x = y = f32x4{0.f, 0.f, 0.f, 0.f};  // a key nobody sees
      if (d < a.Dh) {
        *reinterpret_cast<typename Type<T>::quad*>(dk + d) = to_quad<T>(x);
        *reinterpret_cast<typename Type<T>::quad*>(dv + d) = to_quad<T>(y);
      }
    }
}

// PLAIN: neither cap nor bias, the encoder's own case: fewer registers and branches
template <class T, int DP, int WAVES, bool PLAIN>
int launch(const Args& a, bool backward, hipStream_t st) {
  const long long slots = (long long)a.T / (32 * WAVES) + a.docs + 1;
  TT_REQUIRE(slots * a.H <= 0x7fffffffLL, TT_ERR_BAD_SHAPE);
  const dim3 gq((unsigned)(slots * a.H)), gk((unsigned)(slots * a.Hkv)), bl(64 * WAVES);
  if (!backward) {
    hipLaunchKernelGGL((attention_fwd_kernel<T, DP, WAVES, PLAIN>), gq, bl, 0, st, a);
  } else {
    hipLaunchKernelGGL((attention_dq_kernel<T, DP, WAVES, PLAIN>), gq, bl, 0, st, a);
    TT_CHECK_LAUNCH();
    hipLaunchKernelGGL((attention_dkv_kernel<T, DP, WAVES, PLAIN>), gk, bl, 0, st, a);
  }
  TT_CHECK_LAUNCH();
  return TT_OK;
}

// workgroups of 128 rows where the documents are long enough to fill them, of 64 rows for short ones
// (documents of 700-2048 / 12-128 tokens: 1217 / 113 us with 128 rows, 1561 / 104 with 64)
int pick_waves(long long T, int docs) { return T >= 128LL * docs ? 4 : 2; }

template <class F>
int with_shape(int dtype, int Dh, F&& f) {
  auto dim = [&](auto t) {
    if (Dh <= 32) return f(t, std::integral_constant<int, 32>{});
    if (Dh <= 64) return f(t, std::integral_constant<int, 64>{});
    return f(t, std::integral_constant<int, 128>{});
  };
  switch (dtype) {
    case TT_F32: return dim(float{});
    case TT_BF16: return dim(__bf16{});
    case TT_F16: return dim(_Float16{});
    default: return (int)TT_ERR_BAD_DTYPE;
  }
}

bool view_ok(const tt_head_view& v, int width, bool required) {
  if (!v.data) return !required;
  const int kpf = 16 / width;
  // (the last bound keeps a tile's 32-bit offsets in range)
  return tt_aligned16(v.data) && v.token_stride % kpf == 0 && v.head_stride % kpf == 0 && v.token_stride >= 0 &&
         v.token_stride < (1 << 22);
}

int check(const tt_attention_args* p) {
  TT_REQUIRE(p, TT_ERR_NULL_POINTER);
  TT_REQUIRE(p->dtype == TT_F32 || p->dtype == TT_BF16 || p->dtype == TT_F16, TT_ERR_BAD_DTYPE);
  TT_REQUIRE(p->T >= 0 && p->T <= 1LL << 30 && p->docs >= 1 && p->heads >= 1 && p->kv_heads >= 1 &&
                 p->heads % p->kv_heads == 0 && p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0,
             TT_ERR_BAD_SHAPE);
  // (within these bounds quotients and products of scale, cap and a score stay in fp32's range)
  TT_REQUIRE(tt_scale_ok(p->scale) && (p->softcap == 0.f || tt_scale_ok(p->softcap)), TT_ERR_BAD_SHAPE);
  TT_REQUIRE(!(p->causal && p->prefix), TT_ERR_UNSUPPORTED);
  return TT_OK;
}
Args make_args(const tt_attention_args* p) {
  Args a{};
  a.q = p->q.data; a.qt = p->q.token_stride; a.qh = p->q.head_stride;
  a.k = p->k.data; a.kt = p->k.token_stride; a.kh = p->k.head_stride;
  a.v = p->v.data; a.vt = p->v.token_stride; a.vh = p->v.head_stride;
  a.o = a.out = p->out.data; a.ot = p->out.token_stride; a.oh = p->out.head_stride;
  a.dout = p->dout.data; a.dot = p->dout.token_stride; a.doh = p->dout.head_stride;
  a.dq = p->dq.data; a.dqt = p->dq.token_stride; a.dqh = p->dq.head_stride;
  a.dk = p->dk.data; a.dkt = p->dk.token_stride; a.dkh = p->dk.head_stride;
  a.dv = p->dv.data; a.dvt = p->dv.token_stride; a.dvh = p->dv.head_stride;
  a.lse = p->lse; a.delta = p->delta; a.cu = p->cu_seqlens; a.prefix = p->prefix; a.slopes = p->slopes; a.keep = p->key_mask;
  a.T = (int)p->T; a.docs = p->docs; a.H = p->heads; a.Hkv = p->kv_heads; a.Dh = p->head_dim; a.causal = p->causal;
  a.scale = p->scale; a.cap = p->softcap;
  // spread / sorted against XCD-contiguous order: 5 documents of 1001-4096 tokens with prefixes 340 -> 243 -> 198 us, 16 causal ones
  // of 700-2048 (both directions) 1306 -> 1217 -> 1159; 512 documents of 12-128 tokens 104 contiguous, 108 spread
  a.spread = p->T >= 256LL * p->docs;
  a.sorted = a.spread && p->docs <= 64 && (p->causal || p->prefix);
  return a;
}

int run(const tt_attention_args* p, bool backward, hipStream_t st) {
  const Args a = make_args(p);
  const int waves = pick_waves(p->T, p->docs);
  const bool plain = !(a.cap > 0.f) && !a.slopes;
  return with_shape(p->dtype, p->head_dim, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (plain) return waves == 4 ? launch<T, DP, 4, true>(a, backward, st) : launch<T, DP, 2, true>(a, backward, st);
    return waves == 4 ? launch<T, DP, 4, false>(a, backward, st) : launch<T, DP, 2, false>(a, backward, st);
  });
}

}  // namespace

extern "C" int tt_packed_attention(const tt_attention_args* p, tt_stream_t stream) {
  int rc = check(p);
  if (rc != TT_OK) return rc;
  if (p->T == 0) return TT_OK;
  TT_REQUIRE(p->q.data && p->k.data && p->v.data && p->out.data && p->lse && p->cu_seqlens, TT_ERR_NULL_POINTER);
  const int width = dtype_bytes(p->dtype);
  TT_REQUIRE(view_ok(p->q, width, true) && view_ok(p->k, width, true) && view_ok(p->v, width, true) && view_ok(p->out, width, true),
             TT_ERR_ALIGNMENT);
  return run(p, false, static_cast<hipStream_t>(stream));
}

extern "C" int tt_packed_attention_bwd(const tt_attention_args* p, tt_stream_t stream) {
  int rc = check(p);
  if (rc != TT_OK) return rc;
  if (p->T == 0) return TT_OK;
  TT_REQUIRE(p->q.data && p->k.data && p->v.data && p->out.data && p->dout.data && p->dq.data && p->dk.data && p->dv.data && p->lse &&
                 p->delta && p->cu_seqlens,
             TT_ERR_NULL_POINTER);
  const int width = dtype_bytes(p->dtype);
  TT_REQUIRE(view_ok(p->q, width, true) && view_ok(p->k, width, true) && view_ok(p->v, width, true) &&
                 view_ok(p->out, width, true) && view_ok(p->dout, width, true) && view_ok(p->dq, width, true) &&
                 view_ok(p->dk, width, true) && view_ok(p->dv, width, true),
             TT_ERR_ALIGNMENT);
  return run(p, true, static_cast<hipStream_t>(stream));
}
