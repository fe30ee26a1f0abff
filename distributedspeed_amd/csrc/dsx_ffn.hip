// dsx_ffn.hip -- the gated feed-forward block and its gradients (see
// include/dsx.h).
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T      (M tokens, D wide, F inner)
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Forward is two launches: the first computes both projections in one tile
// (half its columns from Wg, half from Wu, so a lane holds g and u of the same
// element) and writes h; the second is the product with Wd. Backward is three:
// dh with the gradients of g and u as its epilogue, dx as one sum over 2F, and
// the three weight gradients as one launch.
//
// What the backward's epilogue needs of the forward is not g and u but the two
// factors u act'(g) and act(g), from the fp32 sums: dg and du are then products
// with no activation to evaluate. A factor is kept as the upper 24 bits of its
// fp32 value (16 bits and 8 bits in separate planes): kept in bf16 they would
// add a rounding to both gradients as large as the one of dg and du to 16
// bits, which the matrix instruction's types do demand. h, dg and du are
// rounded to the inputs' type once (up to three tokens: k_few and WeightGrad).
//
// Operands whose rows are not whole 16-byte chunks are copied first to rows
// that are, where that pays (kRealignTokens).
//
// With few tokens there are fewer tiles than CUs while the weights' bytes
// bound the time: the sum over k is split over blocks, each writing fp32
// partial sums, and a second launch adds them in order and applies the
// epilogue.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "dsx.h"
#include "dsx_gemm.h"
#include "dsx_internal.h"

namespace {

using namespace dsxg;
using dsxi::as_stream;
using dsxi::ceil_div;
using dsxi::fail;
using dsxi::launch_status;
using dsxi::round_up;

// ---- activations -----------------------------------------------------------

struct ActValue {
  float f, d;  // value and derivative
};

__device__ inline ActValue activate(int act, float g) {
  ActValue r;
  if (act == DSX_ACT_SILU) {
    const float s = 1.0f / (1.0f + __expf(-g));
    r.f = g * s;
    r.d = s * (1.0f + g * (1.0f - s));
  } else if (act == DSX_ACT_GELU) {
    const float phi = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    r.f = g * phi;
    r.d = phi + g * 0.39894228040143268f * __expf(-0.5f * g * g);
  } else if (act == DSX_ACT_GELU_TANH) {
    const float k = 0.79788456080286536f, c = 0.044715f;
    const float t = tanhf(k * (g + c * g * g * g));
    r.f = 0.5f * g * (1.0f + t);
    r.d = 0.5f * (1.0f + t) + 0.5f * g * (1.0f - t * t) * k * (1.0f + 3.0f * c * g * g);
  } else {
    r.f = g > 0.0f ? g : (g != g ? g : 0.0f);
    r.d = g > 0.0f ? 1.0f : 0.0f;
  }
  return r;
}

// ---- what the forward keeps ------------------------------------------------

// Planes of [tokens][ldf]: h (16 bit), then the upper 16 and the next 8 bits
// of the two factors. Columns from F to ldf hold zeros, so that a sum over F
// may be taken in whole chunks of eight.
struct Saved {
  short* h;
  uint16_t* p_hi;
  uint16_t* q_hi;
  uint8_t* p_lo;
  uint8_t* q_lo;
  short* h_lo;  // up to kFewTokens: what h lost in rounding, as rows below h's
  int64_t ld;
};

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint8_t  u8x8 __attribute__((ext_vector_type(8)));

// fp32 rounded to its upper 24 bits (nearest; NaN and inf stay what they are).
__device__ inline uint32_t top24(float v) {
  uint32_t b = __builtin_bit_cast(uint32_t, v);
  if ((b & 0x7F800000u) != 0x7F800000u) b += 0x80u;
  else if (b & 0x007FFFFFu) b |= 0x00400000u;  // a NaN whose low bits alone say so
  return b;
}
__device__ inline void put24(uint16_t* hi, uint8_t* lo, int64_t at, const float* v) {
  u16x8 a;
  u8x8 b;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const uint32_t w = top24(v[e]);
    a[e] = (uint16_t)(w >> 16);
    b[e] = (uint8_t)(w >> 8);
  }
  *(u16x8*)(hi + at) = a;
  *(u8x8*)(lo + at) = b;
}
struct Raw24 {
  u16x8 hi;
  u8x8 lo;
};
__device__ inline Raw24 get24(const uint16_t* hi, const uint8_t* lo, int64_t at) {
  return {*(const u16x8*)(hi + at), *(const u8x8*)(lo + at)};
}
__device__ inline float widen24(const Raw24& r, int e) {
  return __builtin_bit_cast(float, ((uint32_t)r.hi[e] << 16) | ((uint32_t)r.lo[e] << 8));
}

// ---- epilogues: eight columns of a row (n is a multiple of 8, below N) ------

// Zeros in the place of columns past the end.
__device__ inline void trim(float* v, int n, int N) {
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = n + e < N ? v[e] : 0.0f;
}

template <class T>
__device__ inline s8v round8(const float* v) {
  s8v w;
#pragma unroll
  for (int e = 0; e < 8; e++) w[e] = T::round(v[e]);
  return w;
}

// What a rounded value lost, in the same type: together they hold 16 (bf16) or
// 22 bits. Nothing beside an infinity or NaN.
template <class T>
__device__ inline short rest(float v) {
  const float w = T::widen(T::round(v));
  return T::round(__builtin_isfinite(w) ? v - w : 0.0f);
}

template <class T>
struct Store {  // C in the inputs' type
  static constexpr bool kPair = false;
  typedef Nothing Raw;
  short* c;
  int64_t ld;
  __device__ inline Raw load(int, int) const { return {}; }
  __device__ inline void one(int m, int n, float v, float) const { c[m * ld + n] = T::round(v); }
  __device__ inline void operator()(int m, int n, int N, const float* v, const float*, const Raw&) const {
    short* o = c + m * ld + n;
    const s8v w = round8<T>(v);
    if (n + 8 <= N)
      *(s8u*)o = w;
    else
      for (int e = 0; e < 8; e++)
        if (n + e < N) o[e] = w[e];
  }
};

template <class T>
struct Up {  // h and the factors from g and u
  static constexpr bool kPair = true;
  typedef Nothing Raw;
  Saved s;
  int act, keep;
  float* h32;  // for `one`: h unrounded, which the few tokens' second product takes
  __device__ inline Raw load(int, int) const { return {}; }
  __device__ inline void one(int m, int n, float g, float u) const {
    const int64_t at = m * s.ld + n;
    const ActValue a = activate(act, g);
    h32[at] = a.f * u;
    if (keep) {
      s.h[at] = T::round(a.f * u);
      s.h_lo[at] = rest<T>(a.f * u);
      const uint32_t p = top24(u * a.d), q = top24(a.f);
      s.p_hi[at] = (uint16_t)(p >> 16);
      s.p_lo[at] = (uint8_t)(p >> 8);
      s.q_hi[at] = (uint16_t)(q >> 16);
      s.q_lo[at] = (uint8_t)(q >> 8);
    }
  }
  __device__ inline void operator()(int m, int n, int N, const float* g, const float* u, const Raw&) const {
    const int64_t at = m * s.ld + n;
    float h[8], p[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const ActValue a = activate(act, g[e]);
      h[e] = a.f * u[e];
      p[e] = u[e] * a.d;
      q[e] = a.f;
    }
    if (n + 8 > N) {
      trim(h, n, N);
      trim(p, n, N);
      trim(q, n, N);
    }
    *(s8v*)(s.h + at) = round8<T>(h);
    if (keep) {
      put24(s.p_hi, s.p_lo, at, p);
      put24(s.q_hi, s.q_lo, at, q);
    }
  }
};

template <class T>
struct Factors {  // dg and du from dh
  static constexpr bool kPair = false;
  struct Raw {
    Raw24 p, q;
  };
  Saved s;
  short* dg;
  short* du;
  short* dg_lo;  // up to kFewTokens (else null): what dg and du lost in rounding
  short* du_lo;
  int rows, cols;
  __device__ inline Raw load(int m, int n) const {
    if (m >= rows || n >= cols) return {};
    const int64_t at = m * s.ld + n;
    return {get24(s.p_hi, s.p_lo, at), get24(s.q_hi, s.q_lo, at)};
  }
  __device__ inline void operator()(int m, int n, int N, const float* v, const float*, const Raw& r) const {
    const int64_t at = m * s.ld + n;
    float p[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      p[e] = widen24(r.p, e) * v[e];
      q[e] = widen24(r.q, e) * v[e];
    }
    if (n + 8 > N) {
      trim(p, n, N);
      trim(q, n, N);
    }
    *(s8v*)(dg + at) = round8<T>(p);
    *(s8v*)(du + at) = round8<T>(q);
    if (dg_lo) {
      s8v a, b;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        a[e] = rest<T>(p[e]);
        b[e] = rest<T>(q[e]);
      }
      *(s8v*)(dg_lo + at) = a;
      *(s8v*)(du_lo + at) = b;
    }
  }
};

// ---- one product: C = sum over segments of A_s B_s^T ------------------------

struct Product {
  Operand a[2], b[2];  // b[1] is the second half tile's operand for a pair, else segment 1's
  int k;               // of each segment
  int segments;
  int m, n;
  int mt, nt;
  int splits, per;     // K tiles per split, over all segments
  float* part;         // fp32 partial sums [split][m][ldp] where splits > 1 (a pair: u at ldp / 2)
  int64_t ldp;
};

__device__ inline Operand at_k(Operand o, bool row, int k) {
  o.p += row ? k : k * o.ld;
  return o;
}

template <class G, bool RA, bool RB, class E>
__global__ DSX_TILE_KERNEL(G) void k_product(Product p, E e) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  constexpr int TN = E::kPair ? G::TN / 2 : G::TN;
  const int tiles = p.mt * p.nt;
  const int bid = xcd_order(blockIdx.x, gridDim.x);
  const int split = bid / tiles;
  int ti, tj;
  band_order(bid - split * tiles, p.mt, p.nt, 8, &ti, &tj);
  G g;
  g.init();
  const int kt = (p.k + kBK - 1) / kBK;
  const int lo = split * p.per, hi = min(lo + p.per, kt * p.segments);
  for (int s = 0; s < p.segments; s++) {
    const int k0 = max(lo - s * kt, 0) * kBK, k1 = min(min(hi - s * kt, kt) * kBK, p.k);
    if (k0 >= k1) continue;
    const Operand a = at_k(p.a[s], RA, k0);
    const Operand b = at_k(E::kPair ? p.b[0] : p.b[s], RB, k0);
    const Operand b1 = E::kPair ? at_k(p.b[1], RB, k0) : b;
    g.run(lds, a, b, b1, ti * G::TM, tj * TN, k1 - k0);
  }
  g.template emit<false>(
      lds, [&](int r, int c) { return p.splits > 1 ? typename E::Raw{} : e.load(ti * G::TM + r, tj * TN + c); },
      [&](int r, int c, float* v, float* w, const typename E::Raw& raw) {
        const int m = ti * G::TM + r, n = tj * TN + c;
        if (m >= p.m || n >= p.n) return;
        if (p.splits > 1) {
          float* o = p.part + ((int64_t)split * p.m + m) * p.ldp + n;
          G::put8(o, v);
          if (E::kPair) G::put8(o + p.ldp / 2, w);
        } else {
          e(m, n, p.n, v, w, raw);
        }
      },
      [](int, int, const float*) {});
}

// Adds the splits' partial sums in order and applies the epilogue: a block
// takes 32 runs of eight columns of a row, eight threads a run, each adding
// every eighth split.
template <class E>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, int m, int n, int64_t ldp, int splits,
                                              E e) {
  __shared__ __attribute__((aligned(16))) float sums[8][32][E::kPair ? 16 : 8];
  const int i = threadIdx.x & 31, q = threadIdx.x >> 5, c = (blockIdx.x * 32 + i) * 8, r = blockIdx.y;
  if (c < n) {
    f4v v[4] = {};
    const float* at = part + ((int64_t)q * m + r) * ldp + c;
#pragma unroll 4
    for (int s = q; s < splits; s += 8, at += 8 * m * ldp) {
      v[0] += *(const f4v*)at;
      v[1] += *(const f4v*)(at + 4);
      if (E::kPair) {
        v[2] += *(const f4v*)(at + ldp / 2);
        v[3] += *(const f4v*)(at + ldp / 2 + 4);
      }
    }
#pragma unroll
    for (int k = 0; k < (E::kPair ? 4 : 2); k++) *(f4v*)&sums[q][i][4 * k] = v[k];
  }
  __syncthreads();
  if (q || c >= n) return;
  float v[8], w[8];
#pragma unroll
  for (int k = 0; k < 8; k++) {
    v[k] = w[k] = 0.0f;
    for (int s = 0; s < 8; s++) {
      v[k] += sums[s][i][k];
      if (E::kPair) w[k] += sums[s][i][8 + (k & 7)];
    }
  }
  e(r, c, n, v, w, e.load(r, c));
}

// ---- up to three tokens ------------------------------------------------------

// With so few tokens the forward is the weights' stream: a wave takes two rows
// of weights (one feature of the gate and the up projection, or two outputs)
// and their products with each token's row, eight elements a lane and load,
// sums in fp32. No shared memory, nothing split, and any alignment; the weights
// are read past the caches, being used once. No matrix instruction asks for 16
// bits here, so the second product takes h in fp32 and y is rounded once; what
// the backward keeps of h is 16 bits as ever. 4096 x 14336, bf16, 1 to 3 tokens:
// 59, 62 and 71 us (5.9 TB/s for one; 64 us through the caches; with h in 16
// bits 59, 62 and 68); as matrix-instruction tiles of 16 rows with split sums
// 68, 68 and 70.
constexpr int kFewTokens = 3;

struct Eight {
  float v[8];
};
template <class T>
__device__ inline Eight eight(const short* p) {
  const s8v w = *(const s8u*)p;
  Eight r;
#pragma unroll
  for (int j = 0; j < 8; j++) r.v[j] = T::widen(w[j]);
  return r;
}
template <class T>
__device__ inline Eight eight(const float* p) {
  const f4v a = *(const f4u*)p, b = *(const f4u*)(p + 4);
  return {{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}
template <class T>
__device__ inline float element(const short* p) {
  return T::widen(*p);
}
template <class T>
__device__ inline float element(const float* p) {
  return *p;
}

template <class T, int M, class X, class E>
__global__ __launch_bounds__(256) void k_few(const short* __restrict__ w0, const short* __restrict__ w1, int64_t ld0,
                                             int64_t ld1, const X* __restrict__ x, int64_t ld_x, int n, int k, E e) {
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);  // the pair of rows
  if (E::kPair ? i >= n : 2 * i >= n) return;
  const bool second = E::kPair || 2 * i + 1 < n;
  const short* p = E::kPair ? w0 + i * ld0 : w0 + 2 * i * ld0;
  const short* q = E::kPair ? w1 + i * ld1 : second ? p + ld0 : p;
  float u[M], v[M];
#pragma unroll
  for (int m = 0; m < M; m++) u[m] = v[m] = 0.0f;
  auto add = [&](const s8v& a, const s8v& b, const Eight* c) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float f = T::widen(a[j]), g = T::widen(b[j]);
#pragma unroll
      for (int m = 0; m < M; m++) {
        const float h = c[m].v[j];
        u[m] = fmaf(f, h, u[m]);
        v[m] = fmaf(g, h, v[m]);
      }
    }
  };
  int c = lane * 8;
#pragma unroll 4
  for (; c + 8 <= k; c += 512) {
    Eight t[M];
    const s8v a = __builtin_nontemporal_load((const s8u*)(p + c)), b = __builtin_nontemporal_load((const s8u*)(q + c));
#pragma unroll
    for (int m = 0; m < M; m++) t[m] = eight<T>(x + m * ld_x + c);
    add(a, b, t);
  }
  if (c < k) {  // the row's last elements
    s8v a = {0, 0, 0, 0, 0, 0, 0, 0}, b = a;
    Eight t[M] = {};
    for (int j = 0; j < 8; j++)
      if (c + j < k) {
        a[j] = p[c + j];
        b[j] = q[c + j];
        for (int m = 0; m < M; m++) t[m].v[j] = element<T>(x + m * ld_x + c + j);
      }
    add(a, b, t);
  }
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      u[m] += __shfl_xor(u[m], d);
      v[m] += __shfl_xor(v[m], d);
    }
  if (lane < M) {
    float f = u[0], g = v[0];
#pragma unroll
    for (int m = 1; m < M; m++) {
      f = lane == m ? u[m] : f;
      g = lane == m ? v[m] : g;
    }
    if (E::kPair) {
      e.one(lane, i, f, g);
    } else {
      e.one(lane, 2 * i, f, 0.0f);
      if (second) e.one(lane, 2 * i + 1, g, 0.0f);
    }
  }
}

// ---- the weight gradients: up to three products over the tokens ------------

// Of many tokens the rounding errors of dg, du and h average out in the sums;
// of up to kFewTokens they would be as large as the gradients' own rounding, so
// what those three lost is as many more rows of theirs, which meet x and dy a
// second time within the one K tile.
struct WeightGrad {
  Operand a, b;
  short* out;
  int m, n, tile0, nt;
};
struct WeightGrads {
  WeightGrad w[3];
  int count, tokens;
};

template <class G, class T>
__global__ DSX_TILE_KERNEL(G) void k_weight_grads(WeightGrads t) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  const int bid = xcd_order(blockIdx.x, gridDim.x);
  int i = 0;
  while (i + 1 < t.count && bid >= t.w[i + 1].tile0) i++;
  const WeightGrad& q = t.w[i];
  int ti, tj;
  band_order(bid - q.tile0, (q.m + G::TM - 1) / G::TM, q.nt, 8, &ti, &tj);
  G g;
  g.init();
  g.run(lds, q.a, q.b, q.b, ti * G::TM, tj * G::TN, t.tokens);
  const Store<T> e{q.out, q.n};
  g.template emit<false>(
      lds, [](int, int) { return Nothing{}; },
      [&](int r, int c, float* v, float* w, const Nothing& none) {
        const int m = ti * G::TM + r, n = tj * G::TN + c;
        if (m < q.m && n < q.n) e(m, n, q.n, v, w, none);
      },
      [](int, int, const float*) {});
}

// ---- operands off the direct loads' alignment --------------------------------

// Rows of any length and stride to rows of whole 16-byte chunks, zeros past the
// end; up to seven matrices in one launch, a chunk a thread and pass.
struct Realign {
  const short* from;
  short* to;
  int64_t ld;
  int rows, cols, block0;
};
struct Realigns {
  Realign r[7];
  int count;
};
constexpr int kRealignChunks = 1024;  // of a block

__global__ __launch_bounds__(256) void k_realign(Realigns t) {
  int i = 0;
  while (i + 1 < t.count && (int)blockIdx.x >= t.r[i + 1].block0) i++;
  const Realign& q = t.r[i];
  const uint32_t per = (uint32_t)(q.cols + 7) / 8, n = per * (uint32_t)q.rows;
  const uint32_t at = (blockIdx.x - q.block0) * kRealignChunks + threadIdx.x;
  s8v v[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t k = at + j * 256;
    v[j] = s8v{0, 0, 0, 0, 0, 0, 0, 0};
    if (k >= n) continue;
    const int r = (int)(k / per), c = (int)(k % per) * 8;
    const short* p = q.from + r * q.ld + c;
    if (c + 8 <= q.cols)
      v[j] = *(const s8u*)p;
    else
      for (int e = 0; e < 8; e++)
        if (c + e < q.cols) v[j][e] = p[e];
  }
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (at + j * 256 < n) *(s8v*)(q.to + (int64_t)(at + j * 256) * 8) = v[j];
}

// ---- host ------------------------------------------------------------------

// Tile rows and splits of a product of m x n over kt K tiles.
struct Shape {
  int tm, tn, splits, per;
};

Shape shape_of(int64_t m, int64_t n, int64_t kt, bool pair, bool direct) {
  Shape s{};
  const int64_t cols = pair ? 2 * n : n;
  const int64_t want = 2 * kCus;  // blocks to fill the chip
  int64_t most = kt / 2;          // splits, of two K tiles each at least
  if (!direct) {
    s.tm = m <= 32 ? 32 : 128;
    s.tn = 128;
  } else if (m <= 64) {
    s.tm = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    // 4096 x 14336, 16 tokens forward: 82 us with 128 columns a tile, 94 with 64;
    // 64 x 2048 x 8192 forward and backward: 104 and 96 (two K tiles in shared memory)
    s.tn = m <= 16 ? 128 : 64;
    // A split writes and reads m n fp32 sums: at most half as many bytes as the
    // weights' own 2 n k. (Without the bound, 64 x 2048 x 8192: 135 us.)
    const int64_t bound = kt * kBK / (8 * m);
    if (bound < most) most = bound;
  } else if (const int64_t n64 = ceil_div(m, 64) * ceil_div(cols, 64);
             n64 <= 4 * kCus && kt <= 96 && n64 * kt <= 128 * kCus) {
    // A product of at most about 128 K tiles of 64 x 64 a CU, four blocks to a
    // CU: larger tiles would have to be split over K and joined, or leave CUs
    // idle. Forward, against 128-tiles: 256 x 1024 x 4096 22 us and 56,
    // 2048 x 512 x 1024 23 and 36, 200 x 2048 x 5632 37 and 58. Beyond the bounds
    // the twice as many loads cost more: forward and backward, with n64 <= 1024
    // alone, 1024 x 2048 x 5632 takes 334 us (308 with 128-tiles) and
    // 256 x 4096 x 14336 takes 561 (480).
    s.tm = s.tn = 64;
  } else {
    s.tm = s.tn = square_tile(ceil_div(m, 256) * ceil_div(cols, 256), ceil_div(m, 128) * ceil_div(cols, 128));
  }
  const int64_t tiles = ceil_div(m, s.tm) * ceil_div(cols, s.tn);
  int64_t splits = tiles >= want / 2 ? 1 : ceil_div(want, tiles);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  s.per = (int)ceil_div(kt, splits);
  s.splits = (int)ceil_div(kt, s.per);
  return s;
}

int64_t ld_inner(int64_t inner) { return round_up(inner, 8); }

int64_t part_bytes(int64_t m, int64_t n, const Shape& s, bool pair) {
  return s.splits > 1 ? s.splits * m * round_up(n, 8) * (pair ? 2 : 1) * 4 : 0;
}

template <class T, bool RA, bool RB, class E>
void launch_product(Product p, const Shape& s, bool direct, float* part, const E& e, hipStream_t st) {
  constexpr bool PAIR = E::kPair;
  const int64_t cols = PAIR ? 2 * (int64_t)p.n : p.n;
  p.mt = (int)ceil_div(p.m, s.tm);
  p.nt = (int)ceil_div(cols, s.tn);
  p.splits = s.splits;
  p.per = s.per;
  p.part = part;
  p.ldp = round_up(p.n, 8) * (PAIR ? 2 : 1);
  const dim3 grid((unsigned)(p.mt * p.nt * p.splits));
  // At most two blocks a CU of the 32- and 64-tiles: four K tiles in shared
  // memory (forward, 64 x 2048 x 8192 33 us, 44 with two, 32 x 2048 x 8192 28 and
  // 40; at three blocks a CU 200 x 2048 x 5632 takes 43, with two 37; the 16-tiles
  // gain nothing: 5 x 4096 x 14336 71.5 and 70.9).
  const bool deep = (int)grid.x <= 2 * kCus;
#define DSX_RUN(TM, TN, WM, WN, DIRECT, STAGES)                      \
  do {                                                               \
    using G = Gemm<T, TM, TN, WM, WN, RA, RB, DIRECT, PAIR, STAGES>; \
    k_product<G, RA, RB, E><<<grid, G::THREADS, 0, st>>>(p, e);      \
  } while (0)
  if (direct) {
    if (s.tm == 16) DSX_RUN(16, 128, 1, 4, true, 2);
    else if (s.tm == 32 && deep) DSX_RUN(32, 64, 2, 2, true, 4);
    else if (s.tm == 32) DSX_RUN(32, 64, 2, 2, true, 2);
    else if (s.tm == 64 && deep) DSX_RUN(64, 64, 2, 2, true, 4);
    else if (s.tm == 64) DSX_RUN(64, 64, 2, 2, true, 2);
    else if (s.tm == 128) DSX_RUN(128, 128, 2, 4, true, 2);
    else DSX_RUN(256, 256, 2, 4, true, 2);
  } else {
    if (s.tm == 32) DSX_RUN(32, 128, 1, 4, false, 2);
    else DSX_RUN(128, 128, 2, 4, false, 2);
  }
#undef DSX_RUN
  if (p.splits > 1)
    k_join<E><<<dim3((unsigned)ceil_div(p.n, 256), (unsigned)p.m), 256, 0, st>>>(part, p.m, p.n, p.ldp, p.splits, e);
}

// The direct loads' demands of one operand (rows or columns of `contiguous`
// elements at a stride of ld).
bool direct_ok(const void* p, int64_t ld, int64_t contiguous) {
  return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && contiguous % 8 == 0 && ld <= (1 << 22);
}

struct Sizes {
  int64_t m, d, f, ldf;
  int kd, kf;  // K tiles over D and over F
};
Sizes sizes_of(const DsxFfn& q) {
  Sizes z{q.tokens, q.width, q.inner, ld_inner(q.inner), 0, 0};
  z.kd = (int)ceil_div(z.d, kBK);
  z.kf = (int)ceil_div(z.f, kBK);
  return z;
}

Saved saved_of(const DsxFfn& q) {
  const int64_t ld = ld_inner(q.inner), n = q.tokens * ld;
  Saved s{};
  char* p = (char*)q.saved;
  s.ld = ld;
  s.h = (short*)p;
  if (q.tokens <= kFewTokens) p += 2 * n;
  s.h_lo = (short*)p;
  s.p_hi = (uint16_t*)(p + 2 * n);
  s.q_hi = (uint16_t*)(p + 4 * n);
  s.p_lo = (uint8_t*)(p + 6 * n);
  s.q_lo = (uint8_t*)(p + 7 * n);
  return s;
}

struct Direct {
  bool up, down, dh, dx, dw;
};
// Elements of each operand's rows that may be read (and, past the row's own,
// are zeros).
struct Lengths {
  int64_t x, gate, up, down, dy;
};
Direct direct_of(const DsxFfn& q, const void* dy, int64_t ld_dy, const Lengths& n) {
  const bool x = direct_ok(q.x, q.ld_x, n.x), wg = direct_ok(q.w_gate, q.ld_gate, n.gate),
             wu = direct_ok(q.w_up, q.ld_up, n.up), wd = direct_ok(q.w_down, q.ld_down, n.down),
             y = dy && direct_ok(dy, ld_dy, n.dy);
  Direct d{};
  d.up = x && wg && wu;
  d.down = wd;
  d.dh = y && wd;
  d.dx = wg && wu;
  d.dw = x && y;
  return d;
}

// Operands whose rows' length or stride rule the direct loads out are first
// copied to rows that do not: always in the backward, which reads each twice or
// more, and in a forward of more than kRealignTokens. Forward and backward in
// us, with the loads through registers and with the copies: 3000 x 2049 x 8001
// 494 / 1734 and 410 / 1299, 200 x 2047 x 5631 78 / 280 and 68 / 181,
// 3000 x 255 x 1023 43 / 444 and 36 / 104; forward only, 128 x 2047 x 5631 65
// and 63, 130 x 1025 x 1025 26 and 31, 16 x 2047 x 5631 36 and 53 (there the
// weights' bytes bound the time, which the copies triple). An operand that is
// off by its address alone is not copied.
constexpr int64_t kRealignTokens = 192;
bool realigns(int64_t tokens, bool backward) { return backward || tokens > kRealignTokens; }

bool realigned(int64_t rows, int64_t ld, int64_t cols) {
  return !direct_ok(nullptr, ld, cols) &&
         rows * ceil_div(cols, 8) < (int64_t)1 << 31;  // the copy's 32-bit chunk numbers
}
int64_t realigned_bytes(int64_t rows, int64_t ld, int64_t cols) {
  return realigned(rows, ld, cols) ? round_up(rows * ld_inner(cols) * 2, 256) : 0;
}

int64_t twice_bytes(int64_t rows, int64_t cols) { return round_up(2 * rows * ld_inner(cols) * 2, 256); }

// Collects the copies and puts the operands in their place.
struct Realigner {
  bool wanted;
  char* at;
  Realigns t;
  int64_t blocks;

  void add(const void** p, int64_t* ld, int64_t rows, int64_t* cols) {
    if (!wanted || !realigned(rows, *ld, *cols)) return;
    t.r[t.count++] = {(const short*)*p, (short*)at, *ld, (int)rows, (int)*cols, (int)blocks};
    blocks += ceil_div(rows * ceil_div(*cols, 8), kRealignChunks);
    *p = at;
    at += realigned_bytes(rows, *ld, *cols);
    *ld = *cols = ld_inner(*cols);
  }
  // Of few rows: two copies, one below the other.
  void twice(const void** p, int64_t* ld, int64_t rows, int64_t* cols) {
    const int64_t to = ld_inner(*cols);
    for (int k = 0; k < 2; k++) {
      t.r[t.count++] = {(const short*)*p, (short*)at + k * rows * to, *ld, (int)rows, (int)*cols, (int)blocks};
      blocks += ceil_div(rows * to / 8, kRealignChunks);
    }
    *p = at;
    at += twice_bytes(rows, *cols);
    *ld = *cols = to;
  }
  void launch(hipStream_t st) {
    if (t.count) k_realign<<<dim3((unsigned)blocks), 256, 0, st>>>(t);
  }
};

// Bytes of the split sums, which follow dg and du in the workspace; the copies
// follow them.
int64_t part_of(const DsxFfn& q, bool backward) {
  const Sizes z = sizes_of(q);
  // both load forms, so that the size does not hang on addresses
  int64_t part = 0;
  for (int direct = 0; direct < 2; direct++) {
    int64_t b[4] = {part_bytes(z.m, z.f, shape_of(z.m, z.f, z.kd, true, direct), true),
                    part_bytes(z.m, z.d, shape_of(z.m, z.d, z.kf, false, direct), false), 0, 0};
    if (backward) {
      b[2] = part_bytes(z.m, z.f, shape_of(z.m, z.f, z.kd, false, direct), false);
      b[3] = part_bytes(z.m, z.d, shape_of(z.m, z.d, 2 * z.kf, false, direct), false);
      b[0] = b[1] = 0;
    }
    for (int64_t v : b)
      if (v > part) part = v;
  }
  return round_up(part, 256);
}

int64_t workspace_of(const DsxFfn& q, bool backward) {
  const Sizes z = sizes_of(q);
  if (!z.m) return 256;
  int64_t bytes = part_of(q, backward) + 256;
  if (z.m <= kFewTokens)  // h in fp32; what dg and du lost, and x and dy twice
    bytes += backward ? 2 * round_up(z.m * z.ldf * 2, 256) + 2 * twice_bytes(z.m, z.d) : z.m * z.ldf * 4;
  if (backward) bytes += 2 * round_up(z.m * z.ldf * 2, 256) + realigned_bytes(z.m, z.d, z.d);
  if (realigns(z.m, backward))
    bytes += realigned_bytes(z.m, q.ld_x, z.d) + realigned_bytes(z.f, q.ld_gate, z.d) +
             realigned_bytes(z.f, q.ld_up, z.d) + realigned_bytes(z.d, q.ld_down, z.f);
  return bytes;
}

template <class T, int M>
void forward_few(const DsxFfn& q, const Saved& s, void* y, int64_t ld_y, hipStream_t st) {
  const int d = (int)q.width, f = (int)q.inner;
  const short *wg = (const short*)q.w_gate, *wu = (const short*)q.w_up, *wd = (const short*)q.w_down;
  float* h = (float*)q.workspace;
  k_few<T, M, short><<<dim3((unsigned)ceil_div(f, 4)), 256, 0, st>>>(
      wg, wu, q.ld_gate, q.ld_up, (const short*)q.x, q.ld_x, f, d, Up<T>{s, q.activation, q.keep, h});
  k_few<T, M, float><<<dim3((unsigned)ceil_div(d, 8)), 256, 0, st>>>(wd, wd, q.ld_down, q.ld_down, h, s.ld, d, f,
                                                                     Store<T>{(short*)y, ld_y});
}

template <class T>
int forward(DsxFfn q, void* y, int64_t ld_y, hipStream_t st) {
  const Sizes z = sizes_of(q);
  const Saved s = saved_of(q);
  if (z.m <= kFewTokens) {
    if (z.m == 1) forward_few<T, 1>(q, s, y, ld_y, st);
    else if (z.m == 2) forward_few<T, 2>(q, s, y, ld_y, st);
    else forward_few<T, 3>(q, s, y, ld_y, st);
    return launch_status("dsx_ffn_forward");
  }
  float* part = (float*)q.workspace;
  Lengths len{z.d, z.d, z.d, z.f, z.d};
  Realigner copies{realigns(z.m, false), (char*)q.workspace + part_of(q, false), {}, 0};
  copies.add(&q.x, &q.ld_x, z.m, &len.x);
  copies.add(&q.w_gate, &q.ld_gate, z.f, &len.gate);
  copies.add(&q.w_up, &q.ld_up, z.f, &len.up);
  copies.add(&q.w_down, &q.ld_down, z.d, &len.down);
  copies.launch(st);
  const Direct dir = direct_of(q, nullptr, 0, len);
  Product p{};
  p.a[0] = {(const short*)q.x, q.ld_x, (int)z.m};
  p.b[0] = {(const short*)q.w_gate, q.ld_gate, (int)z.f};
  p.b[1] = {(const short*)q.w_up, q.ld_up, (int)z.f};
  p.k = (int)z.d;
  p.segments = 1;
  p.m = (int)z.m;
  p.n = (int)z.f;
  launch_product<T, true, true>(p, shape_of(z.m, z.f, z.kd, true, dir.up), dir.up, part,
                                Up<T>{s, q.activation, q.keep, nullptr}, st);
  Product r{};
  r.a[0] = {s.h, s.ld, (int)z.m};
  r.b[0] = {(const short*)q.w_down, q.ld_down, (int)z.d};
  r.k = (int)z.f;
  r.segments = 1;
  r.m = (int)z.m;
  r.n = (int)z.d;
  launch_product<T, true, true>(r, shape_of(z.m, z.d, z.kf, false, dir.down), dir.down, part,
                                Store<T>{(short*)y, ld_y}, st);
  return launch_status("dsx_ffn_forward");
}

template <class T, bool DIRECT>
void launch_weight_grads(WeightGrads& w, hipStream_t st) {
  int64_t big = 0, small = 0;  // square_tile's rule over the three
  for (int i = 0; i < w.count; i++) {
    big += ceil_div(w.w[i].m, 256) * ceil_div(w.w[i].n, 256);
    small += ceil_div(w.w[i].m, 128) * ceil_div(w.w[i].n, 128);
  }
  const int tile = DIRECT ? square_tile(big, small) : 128;
  int64_t n = 0;
  for (int i = 0; i < w.count; i++) {
    w.w[i].tile0 = (int)n;
    w.w[i].nt = (int)ceil_div(w.w[i].n, tile);
    n += ceil_div(w.w[i].m, tile) * w.w[i].nt;
  }
  if (!n) return;
  if constexpr (DIRECT) {
    if (tile == 256) {
      using G = Gemm<T, 256, 256, 2, 4, false, false, true>;
      k_weight_grads<G, T><<<dim3((unsigned)n), G::THREADS, 0, st>>>(w);
      return;
    }
  }
  using G = Gemm<T, 128, 128, 2, 4, false, false, DIRECT>;
  k_weight_grads<G, T><<<dim3((unsigned)n), G::THREADS, 0, st>>>(w);
}

template <class T>
int backward(DsxFfn q, const void* dy, int64_t ld_dy, void* dx, int64_t ld_dx, void* dw_gate, void* dw_up,
             void* dw_down, hipStream_t st) {
  const Sizes z = sizes_of(q);
  const Saved s = saved_of(q);
  const bool few = z.m <= kFewTokens;
  const int64_t plane = round_up(z.m * z.ldf * 2 * (few ? 2 : 1), 256);
  short* dg = (short*)q.workspace;
  short* du = (short*)((char*)q.workspace + plane);
  short* dg_lo = few ? dg + z.m * z.ldf : nullptr;  // rows below
  short* du_lo = few ? du + z.m * z.ldf : nullptr;
  float* part = (float*)((char*)q.workspace + 2 * plane);
  const int m = (int)z.m;
  Lengths len{z.d, z.d, z.d, z.f, z.d};
  Realigner copies{realigns(z.m, true), (char*)part + part_of(q, true), {}, 0};
  if (few) {
    copies.twice(&q.x, &q.ld_x, z.m, &len.x);
    copies.twice(&dy, &ld_dy, z.m, &len.dy);
  } else {
    if (dw_gate || dw_up) copies.add(&q.x, &q.ld_x, z.m, &len.x);
    if (z.d % 8) copies.add(&dy, &ld_dy, z.m, &len.dy);  // the workspace's size knows the width, not this stride
  }
  if (dx) {
    copies.add(&q.w_gate, &q.ld_gate, z.f, &len.gate);
    copies.add(&q.w_up, &q.ld_up, z.f, &len.up);
  }
  if (dx || dw_gate || dw_up) copies.add(&q.w_down, &q.ld_down, z.d, &len.down);
  copies.launch(st);
  const Direct dir = direct_of(q, dy, ld_dy, len);
  if (dx || dw_gate || dw_up) {
    Product p{};
    p.a[0] = {(const short*)dy, ld_dy, m};
    p.b[0] = {(const short*)q.w_down, q.ld_down, (int)z.f};
    p.k = (int)z.d;
    p.segments = 1;
    p.m = m;
    p.n = (int)z.f;
    launch_product<T, true, false>(p, shape_of(z.m, z.f, z.kd, false, dir.dh), dir.dh, part,
                                   Factors<T>{s, dg, du, dg_lo, du_lo, m, (int)z.f}, st);
  }
  if (dx) {
    Product r{};
    r.a[0] = {dg, z.ldf, m};
    r.a[1] = {du, z.ldf, m};
    r.b[0] = {(const short*)q.w_gate, q.ld_gate, (int)z.d};
    r.b[1] = {(const short*)q.w_up, q.ld_up, (int)z.d};
    r.k = (int)z.f;
    r.segments = 2;
    r.m = m;
    r.n = (int)z.d;
    launch_product<T, true, false>(r, shape_of(z.m, z.d, 2 * z.kf, false, dir.dx), dir.dx, part,
                                   Store<T>{(short*)dx, ld_dx}, st);
  }
  WeightGrads w{};
  w.tokens = few ? 2 * m : m;
  const Operand x{(const short*)q.x, q.ld_x, (int)z.d}, oy{(const short*)dy, ld_dy, (int)z.d};
  const Operand og{dg, z.ldf, (int)z.f}, ou{du, z.ldf, (int)z.f}, oh{s.h, s.ld, (int)z.f};
  if (dw_gate) w.w[w.count++] = {og, x, (short*)dw_gate, (int)z.f, (int)z.d, 0, 0};
  if (dw_up) w.w[w.count++] = {ou, x, (short*)dw_up, (int)z.f, (int)z.d, 0, 0};
  if (dw_down) w.w[w.count++] = {oy, oh, (short*)dw_down, (int)z.d, (int)z.f, 0, 0};
  if (dir.dw)
    launch_weight_grads<T, true>(w, st);
  else
    launch_weight_grads<T, false>(w, st);
  return launch_status("dsx_ffn_backward");
}

int check_sizes(const char* what, const DsxFfn* q) {
  if (!q) return fail(DSX_EINVAL, "%s: the block is NULL", what);
  if (q->tokens < 0 || q->tokens > DSX_MATRIX_MAX_DIM || q->width < 1 || q->width > DSX_MATRIX_MAX_DIM ||
      q->inner < 1 || q->inner > DSX_MATRIX_MAX_DIM)
    return fail(DSX_EINVAL, "%s: tokens in [0, %d], width and inner in [1, %d]", what, DSX_MATRIX_MAX_DIM,
                DSX_MATRIX_MAX_DIM);
  if (!dsxi::is16(q->dtype)) return fail(DSX_EINVAL, "%s: dtype must be DSX_F16 or DSX_BF16", what);
  if (q->activation < DSX_ACT_SILU || q->activation > DSX_ACT_RELU)
    return fail(DSX_EINVAL, "%s: bad activation %d", what, q->activation);
  return DSX_OK;
}

int check_block(const char* what, const DsxFfn* q, bool backward) {
  if (int rc = check_sizes(what, q)) return rc;
  if (!q->tokens) return DSX_OK;
  if (!q->x || !q->w_gate || !q->w_up || !q->w_down || !q->saved || !q->workspace)
    return fail(DSX_EINVAL, "%s: NULL pointer", what);
  if ((((uintptr_t)q->x | (uintptr_t)q->w_gate | (uintptr_t)q->w_up | (uintptr_t)q->w_down) & 1) ||
      (((uintptr_t)q->saved | (uintptr_t)q->workspace) & 255))
    return fail(DSX_EINVAL, "%s: misaligned pointer", what);
  if (q->ld_x < q->width || q->ld_gate < q->width || q->ld_up < q->width || q->ld_down < q->inner)
    return fail(DSX_EINVAL, "%s: a row stride is below the row's length", what);
  if (q->workspace_bytes < workspace_of(*q, backward))
    return fail(DSX_EINVAL, "%s: the workspace has %lld bytes, %lld are needed", what, (long long)q->workspace_bytes,
                (long long)workspace_of(*q, backward));
  return DSX_OK;
}

}  // namespace

extern "C" {

int64_t dsx_ffn_saved_bytes(int64_t tokens, int64_t inner, int32_t keep) {
  if (tokens < 0 || inner < 1 || tokens > DSX_MATRIX_MAX_DIM || inner > DSX_MATRIX_MAX_DIM)
    return fail(-1, "dsx_ffn_saved_bytes: sizes out of range");
  return tokens * ld_inner(inner) * (!keep ? 2 : tokens <= kFewTokens ? 10 : 8);
}

int64_t dsx_ffn_workspace_bytes(const DsxFfn* block, int32_t backward) {
  if (check_sizes("dsx_ffn_workspace_bytes", block)) return -1;
  return workspace_of(*block, backward != 0);
}

int dsx_ffn_forward(const DsxFfn* block, void* y, int64_t ld_y, void* stream) {
  const char* what = "dsx_ffn_forward";
  if (int rc = check_block(what, block, false)) return rc;
  if (!block->tokens) return DSX_OK;
  if (!y || ((uintptr_t)y & 1) || ld_y < block->width) return fail(DSX_EINVAL, "%s: bad output", what);
  hipStream_t s = as_stream(stream);
  return block->dtype == DSX_F16 ? forward<F16>(*block, y, ld_y, s) : forward<BF16>(*block, y, ld_y, s);
}

int dsx_ffn_backward(const DsxFfn* block, const void* dy, int64_t ld_dy, void* dx, int64_t ld_dx, void* dw_gate,
                     void* dw_up, void* dw_down, void* stream) {
  const char* what = "dsx_ffn_backward";
  if (int rc = check_block(what, block, true)) return rc;
  if (!block->keep) return fail(DSX_EINVAL, "%s: the forward kept nothing (keep is 0)", what);
  if (!block->tokens) return DSX_OK;
  if (!dy || ((uintptr_t)dy & 1) || ld_dy < block->width) return fail(DSX_EINVAL, "%s: bad output gradient", what);
  if (dx && (((uintptr_t)dx & 1) || ld_dx < block->width)) return fail(DSX_EINVAL, "%s: bad input gradient", what);
  if (((uintptr_t)dw_gate | (uintptr_t)dw_up | (uintptr_t)dw_down) & 1)
    return fail(DSX_EINVAL, "%s: misaligned weight gradient", what);
  hipStream_t s = as_stream(stream);
  return block->dtype == DSX_F16 ? backward<F16>(*block, dy, ld_dy, dx, ld_dx, dw_gate, dw_up, dw_down, s)
                                 : backward<BF16>(*block, dy, ld_dy, dx, ld_dx, dw_gate, dw_up, dw_down, s);
}

}  // extern "C"
