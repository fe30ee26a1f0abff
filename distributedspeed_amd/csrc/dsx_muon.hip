// dsx_muon.hip -- Newton-Schulz orthogonalisation of matrices, and the Muon
// step around it (see include/dsx.h).
//
// For each matrix G (s x l with s <= l; a matrix with more rows than columns is
// transposed on the way in and out, the result being the same):
//   X0 = G / (|G|_F + eps);   for each step with its coefficients (a, b, c):
//   A = X X^T (s x s),  B = b A + c A A,  X <- a X + B X.
// A and B are symmetric: only the tiles on and above the diagonal are
// computed, each written at both places. A step is three launches for a whole
// list of matrices of any shapes; every launch finds its matrix and tile from a
// table in the kernel's arguments.
//
// Numbers. The iterates are fp16 with fp32 sums: entries of X, A and B are
// bounded by their spectral norms (about 1.2, 1.5 and 2.9 with Muon's
// coefficients), so range is no concern and fp16's 11 bits leave 8 times less
// rounding error than bf16 (all of A, B and X rounded, against 64 bits,
// 1024 x 1024: 1.1e-3 and 8.8e-3).
// All three are stored times kScale, which keeps the small entries of large
// matrices (1e-6 for A) in fp16's normal range. X0 is scaled by a power of two
// alone, so a 16-bit input is not rounded at all; the rest of 1 / |G|, the
// factor r in (1/2, 1], is folded into the first step's sums:
//   A = X0~ X0~^T / (kScale r)^2,  X1 = (a X0~ + B X0~) / (r kScale).
// What rounding X adds has full rank, and a X multiplies it by 3.4 in every
// later step, while a direction that holds something stops growing at 1: a
// matrix of low rank would end up 14% off. So the iterates before the last two
// steps keep a second fp16 with what the first lost, which joins in a X (22
// bits); the products take the first alone, as their noise lies in the
// matrix's own row space. Rank one, 64 x 64: 1.4e-1 without, 2.7e-3 with it.
//
// The diagonals of A and B stay in fp32, apart from the matrices: they are the
// large entries, and in a wide or random matrix nearly equal ones, so that
// rounding them moves all of X by the same 2^-12 and more. With them out, A A is
// A' A' + (d_i + d_j) A' + d_i^2 on the diagonal for the rest A', and B X has
// d_i X added where a X is. Against 64 bits, 192 x 4416: 3.3e-4, with rounded
// diagonals 1.2e-3; 512 x 512: 6.9e-4 and 1.3e-3.
// Matrices whose shorter side is at most 64 take another way to the same
// result, in fp32 throughout: every iterate is a polynomial of A0 = X0 X0^T
// times X0, so with P_k = a I + b A_k + c A_k^2 and A_{k+1} = P_k A_k P_k the
// result is (P_K ... P_1) X0. Three launches: A0 in parts along the longer side,
// everything s x s in one block's shared memory, and the product with X0.
// The recurrence is not stable: A0's rounding moves an eigenvalue near zero by
// about 2^-24, each step multiplies that by a^2, and a negative one runs away.
// So a run of steps ends where the product of their a^2 would pass 2^18
// (small_run; five steps of Muon's coefficients just stay below): X is formed
// in fp32 and the next run begins with its Gram matrix. Modelled in fp32
// against 64 bits, 64 x 64, five steps: 3e-4 off for singular values spread over
// 1e4, 1.4e-4 for rank four, 1e-5 for a random matrix; eight steps 4e-4, 7e-4
// and 2e-5 (in one run 1.1e-1, 9e-3 and 8e-5; twelve in one run: NaN for rank
// four). Where every X is formed, 5e-5, 7e-4 and 2e-6: the rest is the matrix's
// own condition.
// The squares of an fp32 or bf16 matrix may leave fp32's range at either end: a
// part of A0 whose diagonal comes out near one is summed again with its values
// times a power of two, such that none is above 1, and the parts are brought to
// one scale where they are added. (No bit of the result depends on it. Finding
// each tile's largest value before its products instead took a third more time:
// 64 x 14336, 37 us against 25.)

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <new>
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

constexpr float kScale = 4096.0f;
constexpr int kMats = 19;        // matrices of one launch (the table is a kernel argument)
constexpr int kMaxParts = 2048;  // norm partials per matrix
constexpr int kNormTile = 64;    // the norm and cast kernels' square tile
// Scratch of a run of matrices, where it has more than one: a list's scratch does
// not grow with its length, and what fills the card is faster alone (four of
// 14336 x 4096: 15.5 ms one at a time, 16.0 together with 2.1 GiB; 19 of
// 2048 x 2048, 0.9 GiB: 3.9 ms in one run, 4.0, 4.3 and 5.1 in runs of 512, 256
// and 128 MiB; eight of 4096 x 4096: 10.6 with this bound, 10.9 without).
constexpr int64_t kRunBytes = (int64_t)1 << 30;

struct Mat {
  const void* in;
  void*  out;
  float* momentum;
  float* master;
  int64_t ld_in, ld_out;
  int64_t x[2], lo[2], a, b;  // offsets in the workspace, in 16-bit elements
  int32_t rows, cols;   // of the caller's matrix
  int32_t s, l;         // of X: its sides rounded up to multiples of 8, s <= l
  int32_t tall;         // X is the matrix transposed
  int32_t splits;       // of the Gram matrix's sums along l, into ws + part (fp32, a 64-tile after another)
  int64_t part;
  int64_t diag;         // the diagonals of A and of B, s fp32 each (a short side: exponents)
  int32_t part0, parts;
  float   lr;           // Muon: the step size of this matrix
};
struct Table {
  int32_t tile0[kMats];  // first tile of each matrix in the launch at hand
  int32_t n, reserved;
  Mat m[kMats];
};
static_assert(sizeof(Table) <= 3072, "the table travels in the kernel arguments, at most 4 KB with the others");

struct Info {
  float p;      // X0~ = G p, a power of two
  float inv_r;  // 1 / r
  int32_t bad;  // the norm is not finite
  int32_t reserved;
};

struct MuonArgs {
  const float* grad_scale;  // grads are divided by this (NULL: 1)
  int32_t* skip;            // any matrix's norm not finite
  float momentum, decay;
  int32_t nesterov;
};

// The matrix that a block's tile belongs to: all first tiles are read at once.
__device__ inline int find(const Table& t, int tile) {
  const int i = threadIdx.x & 63;
  const bool begun = i < t.n && tile >= t.tile0[i < kMats ? i : 0];
  return __popcll(__ballot(begun)) - 1;
}

// Four values of a row at any element's address (zeros past its end).
typedef s4v s4u __attribute__((aligned(2)));
template <int DT>
__device__ inline void load4(const void* p, int64_t at, int left, float* v) {
  if (DT == DSX_F32) {
    const float* q = (const float*)p + at;
    if (left >= 4) {
      const f4v w = *(const f4u*)q;
      for (int e = 0; e < 4; e++) v[e] = w[e];
    } else {
      for (int e = 0; e < 4; e++) v[e] = e < left ? q[e] : 0.0f;
    }
  } else {
    using T = typename std::conditional<DT == DSX_F16, F16, BF16>::type;
    const short* q = (const short*)p + at;
    if (left >= 4) {
      const s4v w = *(const s4u*)q;
      for (int e = 0; e < 4; e++) v[e] = T::widen(w[e]);
    } else {
      for (int e = 0; e < 4; e++) v[e] = e < left ? T::widen(q[e]) : 0.0f;
    }
  }
}

__device__ inline void store4(float* p, int left, const float* v) {
  if (left >= 4)
    *(f4u*)p = f4v{v[0], v[1], v[2], v[3]};
  else
    for (int e = 0; e < left; e++) p[e] = v[e];
}

// The matrix that is orthogonalised, four values of a row: the input itself,
// or Muon's update (buf = mu buf + (1 - mu) g; u = mu buf + (1 - mu) g with
// Nesterov's correction, else buf).
template <int DT, bool MUON>
__device__ inline void update4(const Mat& m, const MuonArgs& ma, float inv, int r, int c, float* u,
                               float* buf) {
  const int left = m.cols - c;
  load4<DT>(m.in, r * m.ld_in + c, left, u);
  if (MUON) {
    load4<DSX_F32>(m.momentum, (int64_t)r * m.cols + c, left, buf);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float g = u[e] * inv;
      buf[e] = fmaf(ma.momentum, buf[e], (1.0f - ma.momentum) * g);
      u[e] = ma.nesterov ? fmaf(ma.momentum, buf[e], (1.0f - ma.momentum) * g) : buf[e];
    }
  }
}

__device__ inline float inverse_scale(const MuonArgs& ma) { return ma.grad_scale ? 1.0f / *ma.grad_scale : 1.0f; }

// Sums of squares: `parts` blocks per matrix, each over every parts-th tile;
// squares and sums in fp64 (an fp32 input's squares may leave fp32's range). A
// tile a block up to kMaxParts: four a block, the loads waiting for each other's
// sums, took 10.6 us for twelve of 768 x 768 in bf16, one takes 6.4.
template <int DT, bool MUON>
__global__ __launch_bounds__(256) void k_sumsq(Table t, double* __restrict__ partials, MuonArgs ma) {
  const int i = find(t, blockIdx.x);
  const Mat& m = t.m[i];
  const int part = blockIdx.x - t.tile0[i], tid = threadIdx.x;
  const int tc = (m.cols + kNormTile - 1) / kNormTile, tiles = tc * ((m.rows + kNormTile - 1) / kNormTile);
  const float inv = MUON ? inverse_scale(ma) : 1.0f;
  double sum = 0;
  for (int tile = part; tile < tiles; tile += m.parts) {
    const int r0 = tile / tc * kNormTile + (tid >> 4), c = tile % tc * kNormTile + (tid & 15) * 4;
    if (c >= m.cols) continue;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = r0 + 16 * k;
      if (r >= m.rows) break;
      float u[4], buf[4];
      update4<DT, MUON>(m, ma, inv, r, c, u, buf);
#pragma unroll
      for (int e = 0; e < 4; e++) sum += (double)u[e] * u[e];
    }
  }
  __shared__ double part_sum[4];
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((tid & 63) == 0) part_sum[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) partials[m.part0 + part] = part_sum[0] + part_sum[1] + part_sum[2] + part_sum[3];
}

// From the sum of squares: the power of two and the rest of 1 / norm.
__device__ inline Info info_of(double sum, double eps) {
  Info f = {0.0f, 1.0f, 0, 0};
  if (isfinite(sum)) {
    const double inv = (double)kScale / (sqrt(sum) + eps);
    int e;
    frexp(inv, &e);  // inv in [2^(e-1), 2^e)
    f.p = (float)ldexp(1.0, e - 1);
    f.inv_r = (float)(inv / ldexp(1.0, e - 1));
  } else {
    f.bad = 1;
  }
  return f;
}

// A matrix's Info by a block: its partials' sum, in an order set by their
// count, shared by its waves (each wave for itself: 14336 x 4096, whose 2048
// partials every block reads, 85 us for k_cast, 59 so).
__device__ inline Info info_by_block(const double* __restrict__ p, int parts, double eps) {
  __shared__ double of_wave[4];
  __shared__ Info info;
  double sum = 0;
#pragma unroll 4
  for (int k = threadIdx.x; k < parts; k += 256) sum += p[k];
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) info = info_of(of_wave[0] + of_wave[1] + of_wave[2] + of_wave[3], eps);
  __syncthreads();
  return info;
}

// Muon: whether any matrix's norm is not finite, before anything is written.
__global__ __launch_bounds__(256) void k_norms(Table t, const double* __restrict__ partials, double eps,
                                              int32_t* skip) {
  const Mat& m = t.m[blockIdx.x];
  const Info f = info_by_block(partials + m.part0, m.parts, eps);
  if (threadIdx.x == 0 && f.bad) atomicOr(skip, 1);
}

// X0~ = fp16(G p), zero beyond the matrix; all NaN where the norm is not finite
// (every entry of the exact result is). Muon: the momentum buffer is written
// here, once the step is known not to be skipped.
template <int DT, bool MUON>
__global__ __launch_bounds__(256) void k_cast(Table t, short* __restrict__ ws, const double* __restrict__ partials,
                                              Info* __restrict__ info, double eps, MuonArgs ma) {
  constexpr bool LO = MUON || DT == DSX_F32;  // a 16-bit input loses nothing
  __shared__ short turn[LO ? 2 : 1][kNormTile][kNormTile + 4];
  if (MUON && *ma.skip) return;
  const int i = find(t, blockIdx.x);
  const Mat& m = t.m[i];
  const int tile = blockIdx.x - t.tile0[i], tid = threadIdx.x;
  const int tc = (m.l + kNormTile - 1) / kNormTile;  // X's tile, and where it lies in the matrix
  const int xr = tile / tc * kNormTile, xc = tile % tc * kNormTile;
  const int r0 = (m.tall ? xc : xr) + (tid >> 4), c = (m.tall ? xr : xc) + (tid & 15) * 4;
  const float inv = MUON ? inverse_scale(ma) : 1.0f;
  float u[4][4] = {}, buf[4][4];
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (r0 + 16 * k < m.rows && c < m.cols) update4<DT, MUON>(m, ma, inv, r0 + 16 * k, c, u[k], buf[k]);
  const Info f = info_by_block(partials + m.part0, m.parts, eps);  // while the tile is on its way
  if (tile == 0 && tid == 0) info[i] = f;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int r = r0 + 16 * k;
    if (r < m.rows && c < m.cols) {
      if (MUON) store4(m.momentum + (int64_t)r * m.cols + c, m.cols - c, buf[k]);
      for (int e = 0; e < 4; e++) u[k][e] = f.bad ? __builtin_nanf("") : c + e < m.cols ? u[k][e] * f.p : 0.0f;
    }
    s4v o, lo;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      o[e] = F16::round(u[k][e]);
      lo[e] = F16::round(u[k][e] - F16::widen(o[e]));
    }
    if (!m.tall) {
      if (r < m.s && c < m.l) {
        *(s4v*)(ws + m.x[0] + (int64_t)r * m.l + c) = o;
        if (LO) *(s4v*)(ws + m.lo[0] + (int64_t)r * m.l + c) = lo;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        turn[0][(tid & 15) * 4 + e][(tid >> 4) + 16 * k] = o[e];
        if (LO) turn[LO ? 1 : 0][(tid & 15) * 4 + e][(tid >> 4) + 16 * k] = lo[e];
      }
    }
  }
  if (!m.tall) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int r = (tid >> 4) + 16 * k, q = (tid & 15) * 4;
    if (xr + r >= m.s || xc + q >= m.l) continue;
    const int64_t at = (int64_t)(xr + r) * m.l + xc + q;
    *(s4v*)(ws + m.x[0] + at) = *(const s4v*)&turn[0][r][q];
    if (LO) *(s4v*)(ws + m.lo[0] + at) = *(const s4v*)&turn[LO ? 1 : 0][r][q];
  }
}

__device__ inline void triangle(int t, int* i, int* j) {
  int q = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
  while (q * (q + 1) / 2 > t) q--;
  while ((q + 1) * (q + 2) / 2 <= t) q++;
  *j = q;
  *i = t - q * (q + 1) / 2;
}

// A symmetric product's tile, written at (m, n) and, off the diagonal, at (n, m).
// GRAM: A = X X^T of the current X; else B = b A + c A A.
template <class G, bool GRAM, bool SPLIT>
__global__ DSX_TILE_KERNEL(G) void k_symmetric(Table t, short* __restrict__ ws, const Info* __restrict__ info, int cur,
                                               int first, float b, float c, const int32_t* skip) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  if (skip && *skip) return;
  const int bid = xcd_order(blockIdx.x, gridDim.x);
  const int i = find(t, bid);
  const Mat& m = t.m[i];
  const int s = m.s;
  int ti, tj;
  const int side = (s + G::TM - 1) / G::TM, tiles = side * (side + 1) / 2;
  const bool split = SPLIT && m.splits > 1;
  const int at = bid - t.tile0[i], run = split ? at / tiles : 0, tile = at - run * tiles;
  triangle(tile, &ti, &tj);
  G g;
  g.init();
  const float inv_r = first ? info[i].inv_r : 1.0f;
  const short* src = ws + (GRAM ? m.x[cur] : m.a);
  Operand o{src, GRAM ? m.l : s, s};
  int k_all = GRAM ? m.l : s;
  if (split) {  // K tiles [lo, hi) of l
    const int kt = (m.l + kBK - 1) / kBK, lo = (int)((int64_t)kt * run / m.splits),
              hi = (int)((int64_t)kt * (run + 1) / m.splits);
    o.p += lo * kBK;
    k_all = min(hi * kBK, m.l) - lo * kBK;
  }
  const int r0 = ti * G::TM, c0 = tj * G::TN;
  g.run(lds, o, o, o, r0, c0, k_all);
  if (split) {
    float* out = (float*)(ws + m.part) + ((int64_t)run * tiles + tile) * G::TM * G::TN;
    g.template emit<false>(
        lds, [](int, int) { return Nothing{}; },
        [&](int r, int q, float* v, float*, const Nothing&) { G::put8(out + r * G::TN + q, v); },
        [](int, int, const float*) {});
    return;
  }
  const float k = inv_r * inv_r * (1.0f / kScale);
  short* dst = ws + (GRAM ? m.a : m.b);
  float* da = (float*)(ws + m.diag);
  float* db = da + s;
  struct Raw {
    s8v a;
    float row;
    f4v lo, hi;  // the diagonal of A at the row and at the eight columns
  };
  auto pre = [&](int r, int q) {  // s is a multiple of 8: eight values are inside or outside together
    r += r0;
    q += c0;
    Raw raw{};
    if (!GRAM && r < s && q < s)
      raw = {*(const s8v*)(src + (int64_t)r * s + q), da[r], *(const f4v*)(da + q), *(const f4v*)(da + q + 4)};
    return raw;
  };
  auto put = [&](int r, int q, float* v, float*, const Raw& raw) {
    r += r0;
    q += c0;
    s8v w;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const bool on = r == q + e;
      if (GRAM) {
        v[e] *= k;
        if (on && r < s) da[r] = v[e] * (1.0f / kScale);
      } else {
        const float a = F16::widen(raw.a[e]), d = raw.row + (e < 4 ? raw.lo[e & 3] : raw.hi[e & 3]);
        if (on && r < s)
          db[r] = fmaf(c, fmaf(v[e], 1.0f / (kScale * kScale), raw.row * raw.row), b * raw.row);
        v[e] = fmaf(c, fmaf(d, a, v[e] * (1.0f / kScale)), b * a);
      }
      if (on) v[e] = 0.0f;
      w[e] = F16::round(v[e]);
    }
    if (r < s && q < s) *(s8v*)(dst + (int64_t)r * s + q) = w;
  };
  auto mirror = [&](int q, int r, const float* v) {
    r += r0;
    q += c0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s8v w;
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = F16::round(v[8 * h + e]);
      if (q < s && r + 8 * h < s) *(s8v*)(dst + (int64_t)q * s + r + 8 * h) = w;
    }
  };
  if (ti == tj)
    g.template emit<false>(lds, pre, put, mirror);
  else
    g.template emit<true>(lds, pre, put, mirror);
}

// A from the partial sums of a split Gram matrix's 64-tiles, added in order.
__global__ __launch_bounds__(256) void k_gram_join(Table t, short* __restrict__ ws, const Info* __restrict__ info,
                                                   int first, const int32_t* skip) {
  __shared__ float x[64][68];
  if (skip && *skip) return;
  const int i = find(t, blockIdx.x);
  const Mat& m = t.m[i];
  const int tile = blockIdx.x - t.tile0[i], s = m.s, side = (s + 63) / 64, tiles = side * (side + 1) / 2;
  if (m.splits <= 1) return;
  int ti, tj;
  triangle(tile, &ti, &tj);
  const float inv_r = first ? info[i].inv_r : 1.0f, k = inv_r * inv_r * (1.0f / kScale);
  const float* p = (const float*)(ws + m.part) + (int64_t)tile * 4096;
  short* dst = ws + m.a;
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
  f4v v[4] = {};
#pragma unroll 4
  for (int n = 0; n < m.splits; n++, p += (int64_t)tiles * 4096)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += *(const f4v*)(p + r * 64 + c + 4 * e);
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const bool on = ti == tj && r == c + e;
    x[r][c + e] = on ? 0.0f : k * v[e >> 2][e & 3];
    if (on && ti * 64 + r < s) ((float*)(ws + m.diag))[ti * 64 + r] = k * v[e >> 2][e & 3] * (1.0f / kScale);
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 16; h += 8) {
    s8v w, z;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      w[e] = F16::round(x[r][c + h + e]);
      z[e] = F16::round(x[c + h + e][r]);
    }
    const int a = ti * 64, b = tj * 64;
    if (a + r < s && b + c + h < s) *(s8v*)(dst + (int64_t)(a + r) * s + b + c + h) = w;
    if (ti != tj && b + r < s && a + c + h < s) *(s8v*)(dst + (int64_t)(b + r) * s + a + c + h) = z;
  }
}

// Muon's update of N parameters of a row: w = w decay - lr O (v holds kScale O).
template <int N>
__device__ inline void step_params(const Mat& m, const MuonArgs& ma, int out_dt, int64_t r, int c, const float* v) {
  float* w = m.master + r * m.cols + c;
  short* o = (short*)m.out + r * m.ld_out + c;
#pragma unroll
  for (int h = 0; h < N; h += 8) {
    const int left = m.cols - c - h;
    if (left <= 0) continue;
    float p[8];
    s8v q;
    if (left >= 8) {
      const f4v lo = *(const f4u*)(w + h), hi = *(const f4u*)(w + h + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        p[e] = lo[e];
        p[e + 4] = hi[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] = e < left ? w[h + e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      p[e] = fmaf(-m.lr * (1.0f / kScale), v[h + e], p[e] * ma.decay);
      asm("" : "+v"(p[e]));  // the cast is of the rounded master, not of the exact sum (a fused add and cast)
      q[e] = out_dt == DSX_F16 ? F16::round(p[e]) : BF16::round(p[e]);
    }
    if (left >= 8) {
      *(f4u*)(w + h) = f4v{p[0], p[1], p[2], p[3]};
      *(f4u*)(w + h + 4) = f4v{p[4], p[5], p[6], p[7]};
      if (m.out) *(s8u*)(o + h) = q;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < left) {
          w[h + e] = p[e];
          if (m.out) o[h + e] = q[e];
        }
    }
  }
}
// N values of a row of the result in bf16 (v holds kScale O).
template <int N>
__device__ inline void store_row(const Mat& m, int64_t r, int c, const float* v) {
  short* o = (short*)m.out + r * m.ld_out + c;
#pragma unroll
  for (int h = 0; h < N; h += 8) {
    s8v w;
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = BF16::round(v[h + e] * (1.0f / kScale));
    if (c + h + 8 <= m.cols)
      *(s8u*)(o + h) = w;
    else
      for (int e = 0; e < 8; e++)
        if (c + h + e < m.cols) o[h + e] = w[e];
  }
}

// X <- (a X + B X) / r. LAST: the result itself, transposed back where the
// matrix was, to the output in bf16 or as Muon's parameter update (fp32 master
// and, where there is one, its 16-bit copy of out_dt). take_lo, give_lo: whether
// the iterate read and the one written have their second fp16.
struct XRaw {
  s8v hi, lo;
  float d;  // B's diagonal at the row
};
template <class G, bool LAST, bool MUON>
__global__ DSX_TILE_KERNEL(G) void k_apply(Table t, short* __restrict__ ws, const Info* __restrict__ info, int cur,
                                           int first, float a, int take_lo, int give_lo, MuonArgs ma, int out_dt) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  if (MUON && *ma.skip) return;
  const int bid = xcd_order(blockIdx.x, gridDim.x);
  const int i = find(t, bid);
  const Mat& m = t.m[i];
  const int s = m.s, l = m.l;
  int ti, tj;
  band_order(bid - t.tile0[i], (s + G::TM - 1) / G::TM, (l + G::TN - 1) / G::TN, 8, &ti, &tj);
  const float inv_r = first ? info[i].inv_r : 1.0f;
  const short* x = ws + m.x[cur];
  const short* x_lo = ws + m.lo[cur];
  const float* db = (const float*)(ws + m.diag) + s;
  short* y = ws + m.x[cur ^ 1];
  short* y_lo = ws + m.lo[cur ^ 1];
  const Operand ob{ws + m.b, s, s}, ox{x, l, l};
  const int r0 = ti * G::TM, c0 = tj * G::TN;
  G g;
  g.init();
  g.run(lds, ob, ox, ox, r0, c0, s);
  auto pre = [&](int r, int c) {
    r += r0;
    c += c0;
    XRaw raw{};
    if (r < s && c < l) {
      const int64_t at = (int64_t)r * l + c;
      raw.hi = *(const s8v*)(x + at);
      raw.d = db[r];
      if (take_lo) raw.lo = *(const s8v*)(x_lo + at);
    }
    return raw;
  };
  auto value = [&](float* v, const XRaw& old) {
#pragma unroll
    for (int e = 0; e < 8; e++)
      v[e] = fmaf(a + old.d, F16::widen(old.hi[e]) + F16::widen(old.lo[e]), v[e] * (1.0f / kScale)) * inv_r;
  };
  auto none = [](int, int, const float*) {};
  if (!LAST) {
    g.template emit<false>(
        lds, pre,
        [&](int r, int c, float* v, float*, const XRaw& old) {
          value(v, old);
          s8v w, lo;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            w[e] = F16::round(v[e]);
            lo[e] = F16::round(v[e] - F16::widen(w[e]));
          }
          r += r0;
          c += c0;
          if (r >= s || c >= l) return;
          const int64_t at = (int64_t)r * l + c;
          *(s8v*)(y + at) = w;
          if (give_lo) *(s8v*)(y_lo + at) = lo;
        },
        none);
  } else if (!m.tall) {
    g.template emit<false>(
        lds, pre,
        [&](int r, int c, float* v, float*, const XRaw& old) {
          value(v, old);
          r += r0;
          c += c0;
          if (r >= m.rows || c >= m.cols) return;
          if (MUON) step_params<8>(m, ma, out_dt, r, c, v);
          else store_row<8>(m, r, c, v);
        },
        none);
  } else {
    g.template emit<true>(
        lds, pre, [&](int, int, float* v, float*, const XRaw& old) { value(v, old); },
        [&](int r, int c, const float* v) {  // a column of X is a row of the matrix
          r += c0;
          c += r0;
          if (r >= m.rows || c >= m.cols) return;
          if (MUON) step_params<16>(m, ma, out_dt, r, c, v);
          else store_row<16>(m, r, c, v);
        });
  }
}

// ---- a shorter side of at most 64 --------------------------------------------

constexpr int kSmall = 64;       // X's rows, padded
constexpr int kLdS = kSmall + 4;  // floats: a fragment's 16 rows and 4 columns fall on 64 banks
constexpr int kLdX = 80;          // the same for 4 rows and 16 columns
constexpr int kSmallParts = 32;
constexpr int kNoExponent = -200;  // of zeros: below every fp32's
// A part's sums of squares as they come: room for the parts' sum above, and below
// for products 2^-66 of the largest.
constexpr float kLargest = 0x1p120f, kLeast = 0x1p-60f;

// 64 columns of X from `x0` on, as fp32: four values along the matrix's row in
// each of four rows a thread, and their places in the tile. KEPT: of the X that
// an earlier run of steps left in the workspace, s x l and never transposed.
template <int DT, bool MUON, bool KEPT>
struct SmallTile {
  float u[4][4], buf[4][4];
  static __device__ inline void place(const Mat& m, int x0, int k, int* r, int* c) {
    const bool tall = !KEPT && m.tall;
    *r = (tall ? x0 : 0) + (threadIdx.x >> 4) + 16 * k;
    *c = (tall ? 0 : x0) + (threadIdx.x & 15) * 4;
  }
  __device__ inline void load_kept(const Mat& m, const float* ws, int x0) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      int r, c;
      place(m, x0, k, &r, &c);
      const f4v v = r < m.s && c < m.l ? *(const f4v*)(ws + m.x[0] + (int64_t)r * m.l + c) : f4v{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; e++) u[k][e] = v[e];
    }
  }
  __device__ inline void load(const Mat& m, const MuonArgs& ma, float inv, int x0) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      int r, c;
      place(m, x0, k, &r, &c);
#pragma unroll
      for (int e = 0; e < 4; e++) u[k][e] = 0.0f;
      if (r < m.rows && c < m.cols) update4<DT, MUON>(m, ma, inv, r, c, u[k], buf[k]);
    }
  }
  // The largest magnitude (a NaN aside, which stays one at any scale).
  __device__ inline float most() const {
    float v = 0;
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) v = fmaxf(v, fabsf(u[k][e]));
    return v;
  }
  // Into x [row of X][column], rows LD apart; SCALED: times 2^-scale.
  template <int LD, bool SCALED>
  __device__ inline void store(const Mat& m, int x0, float* x, int scale) const {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      int r, c;
      place(m, x0, k, &r, &c);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float v = KEPT || c + e < m.cols ? u[k][e] : 0.0f;
        if (SCALED) v = ldexpf(v, -scale);
        if (!KEPT && m.tall) x[(c + e) * LD + r - x0] = v;
        else x[r * LD + c - x0 + e] = v;
      }
    }
  }
};

typedef float f4acc __attribute__((ext_vector_type(4)));

// The largest of a block's values, in every thread.
__device__ inline float block_max(float v, float* of_wave) {
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
}

// The partial sums of X X^T over a run of X's columns: parts[part][64][64], and
// the exponent of two that a part's values were divided by.
template <int DT, bool MUON, bool KEPT>
__global__ __launch_bounds__(256) void k_small_gram(Table t, float* __restrict__ ws, MuonArgs ma) {
  __shared__ float x[kSmall * kLdS], of_wave[4];
  const int i = find(t, blockIdx.x);
  const Mat& m = t.m[i];
  const int part = blockIdx.x - t.tile0[i], tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float inv = MUON ? inverse_scale(ma) : 1.0f;
  const int tiles = (m.l + 63) / 64, lo = (int)((int64_t)tiles * part / m.parts),
            hi = (int)((int64_t)tiles * (part + 1) / m.parts), nb = (m.s + 15) / 16;
  f4acc acc[4] = {};
  SmallTile<DT, MUON, KEPT> next;
  auto load = [&](int tile) {
    if (KEPT) next.load_kept(m, ws, tile * 64);
    else next.load(m, ma, inv, tile * 64);
  };
  auto sum = [&](auto scaled, int scale) {
    load(lo);
#pragma unroll
    for (int j = 0; j < 4; j++) acc[j] = f4acc{0, 0, 0, 0};
    for (int tile = lo; tile < hi; tile++) {
      __syncthreads();
      next.template store<kLdS, decltype(scaled)::value>(m, tile * 64, x, scale);
      if (tile + 1 < hi) load(tile + 1);
      __syncthreads();
      if (w < nb)
#pragma unroll 4
        for (int k = 0; k < 64; k += 4) {
          const float a = x[(w * 16 + (lane & 15)) * kLdS + k + (lane >> 4)];
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (j < nb)
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, x[(j * 16 + (lane & 15)) * kLdS + k + (lane >> 4)],
                                                            acc[j], 0, 0, 0);
        }
    }
  };
  int scale = 0;
  sum(std::false_type{}, 0);
  if (!KEPT) {
    float most = 0;  // of the diagonal; a lane's column of the wave's own tile meets it in one of its four rows
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (j == w && (lane >> 4) * 4 + e == (lane & 15)) most = acc[j][e] < kLargest ? acc[j][e] : kLargest;
    most = block_max(most, of_wave);
    if (!(most >= kLeast && most < kLargest)) {
      most = 0;
      for (int tile = lo; tile < hi; tile++) {
        load(tile);
        most = fmaxf(most, next.most());
      }
      most = block_max(most, of_wave);
      scale = kNoExponent;
      if (most > 0.0f) frexpf(most, &scale);
      sum(std::true_type{}, scale);
    }
  }
  if (!KEPT && tid == 0) ((int*)(ws + m.diag))[part] = scale;
  float* out = ws + m.a + (int64_t)part * kSmall * kSmall;
  if (w < nb)
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < nb)
#pragma unroll
        for (int e = 0; e < 4; e++) out[(w * 16 + (lane >> 4) * 4 + e) * kSmall + j * 16 + (lane & 15)] = acc[j][e];
}

// Ten waves, one for each 16 x 16 tile on or above the diagonal of a product of
// two symmetric matrices that commute (polynomials of the same A0), so that the
// product is symmetric too and rows serve as columns.
template <int NB>
struct SmallProduct {
  int ti, tj, lane;
  bool on;
  __device__ inline f4acc operator()(const float* a, const float* b) const {
    f4acc acc = {0, 0, 0, 0};
    if (on)
#pragma unroll
      for (int k = 0; k < 4 * NB; k++)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[(ti * 16 + (lane & 15)) * kLdS + 4 * k + (lane >> 4)],
                                                   b[(tj * 16 + (lane & 15)) * kLdS + 4 * k + (lane >> 4)], acc, 0, 0,
                                                   0);
    return acc;
  }
  __device__ inline void put(float* c, const f4acc& v) const {
    if (!on) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int r = ti * 16 + (lane >> 4) * 4 + e, q = tj * 16 + (lane & 15);
      if (r > q) continue;  // of a tile on the diagonal: its other half is written from above
      c[r * kLdS + q] = v[e];
      c[q * kLdS + r] = v[e];
    }
  }
};

struct SmallCoef {
  float c[3 * 64];
};

// A run of steps (from step k0 on) on its Gram matrix in shared memory;
// P_K ... P_1, over |G| (at the input's scale) in the first run, to ws + m.b. NB:
// 16-tiles a side.
template <int NB>
__device__ inline void small_steps(const Mat& m, float* __restrict__ ws, const SmallCoef& coef, int k0, int steps,
                                   double eps, int32_t* skip, float* A, float* P, float* T, float* Q, double& norm2) {
  const int tid = threadIdx.x, lane = tid & 63;
  constexpr int n = NB * 16;
  SmallProduct<NB> mul;
  triangle(__builtin_amdgcn_readfirstlane(tid >> 6), &mul.ti, &mul.tj);
  mul.lane = lane;
  mul.on = mul.tj < NB;
  const float* in = ws + m.a;
  int* exps = (int*)(ws + m.diag);
  int scale = 0, shift = 0;  // the matrix's exponent; twice a part's below it, in lane `part`
  if (!k0) {
    const int e = exps[lane < m.parts ? lane : 0];
    scale = e;
    for (int d = 32; d; d >>= 1) scale = max(scale, __shfl_xor(scale, d));
    shift = 2 * (e - scale);
    if (tid == 0) exps[kSmallParts] = scale;
  }
  const bool mixed = __any(shift != 0);
  for (int e = tid; e < n * n; e += 640) {
    const int r = e / n, c = e - r * n;
    float sum = 0;
    if (!mixed) {
#pragma unroll 8
      for (int p = 0; p < m.parts; p++) sum += in[(int64_t)p * kSmall * kSmall + r * kSmall + c];
    } else {
      for (int p = 0; p < m.parts; p++)
        sum += ldexpf(in[(int64_t)p * kSmall * kSmall + r * kSmall + c], __builtin_amdgcn_readlane(shift, p));
    }
    A[r * kLdS + c] = sum;
  }
  __syncthreads();
  if (tid < 64) {
    double d = tid < n ? (double)A[tid * kLdS + tid] : 0.0;
    for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
    if (tid == 0) norm2 = d;
  }
  __syncthreads();
  const bool bad = !isfinite(norm2);
  if (bad && skip && tid == 0) atomicOr(skip, 1);
  const double inv = bad ? __builtin_nan("") : k0 ? 1.0 : 1.0 / (sqrt(norm2) + ldexp(eps, -scale));  // 2^scale / (|G| + eps)
  for (int e = tid; e < n * n; e += 640) {
    const int r = e / n, c = e - r * n;
    A[r * kLdS + c] = (float)(A[r * kLdS + c] * inv * inv);
  }
  __syncthreads();
  for (int k = 0; k < steps; k++) {
    const float a = coef.c[3 * (k0 + k)], b = coef.c[3 * (k0 + k) + 1], c = coef.c[3 * (k0 + k) + 2];
    f4acc p = mul(A, A);
    if (mul.on)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = mul.ti * 16 + (lane >> 4) * 4 + e, q = mul.tj * 16 + (lane & 15);
        p[e] = fmaf(c, p[e], b * A[r * kLdS + q]) + (r == q ? a : 0.0f);
      }
    mul.put(P, p);
    if (k == 0) mul.put(Q, p);
    __syncthreads();
    const bool more = k + 1 < steps;
    f4acc s = {0, 0, 0, 0}, q = s;
    if (more) s = mul(P, A);
    if (k) q = mul(P, Q);
    __syncthreads();
    if (more) mul.put(T, s);
    if (k) mul.put(Q, q);
    __syncthreads();
    if (more) {
      s = mul(P, T);
      __syncthreads();
      mul.put(A, s);
      __syncthreads();
    }
  }
  float* out = ws + m.b;
  for (int e = tid; e < n * n; e += 640) {
    const int r = e / n, c = e - r * n;
    out[r * kSmall + c] = (float)(Q[r * kLdS + c] * inv);
  }
}

__global__ __launch_bounds__(640) void k_small_steps(Table t, float* __restrict__ ws, SmallCoef coef, int k0,
                                                     int steps, double eps, int32_t* skip) {
  __shared__ float A[kSmall * kLdS], P[kSmall * kLdS], T[kSmall * kLdS], Q[kSmall * kLdS];
  __shared__ double norm2;
  const Mat& m = t.m[blockIdx.x];
  if (m.s <= 16) small_steps<1>(m, ws, coef, k0, steps, eps, skip, A, P, T, Q, norm2);
  else if (m.s <= 32) small_steps<2>(m, ws, coef, k0, steps, eps, skip, A, P, T, Q, norm2);
  else if (m.s <= 48) small_steps<3>(m, ws, coef, k0, steps, eps, skip, A, P, T, Q, norm2);
  else small_steps<4>(m, ws, coef, k0, steps, eps, skip, A, P, T, Q, norm2);
}

// 64 columns of the product of a run's P_K ... P_1 and X: the result, to the
// output or the parameters, after the LAST run, else the next run's X (a block
// reads and writes its own columns alone).
template <int DT, bool MUON, bool KEPT, bool LAST>
__global__ __launch_bounds__(256) void k_small_apply(Table t, float* __restrict__ ws, MuonArgs ma, int out_dt) {
  __shared__ __attribute__((aligned(16))) float q[kSmall * kLdS], x[kSmall * kLdX];
  if (MUON && *ma.skip) return;
  const int i = find(t, blockIdx.x);
  const Mat& m = t.m[i];
  const int x0 = (blockIdx.x - t.tile0[i]) * 64, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int nb = (m.s + 15) / 16, n = nb * 16;
  const float inv = MUON ? inverse_scale(ma) : 1.0f;
  for (int e = tid; e < n * n; e += 256) {
    const int r = e / n, c = e - r * n;
    q[r * kLdS + c] = ws[m.b + r * kSmall + c];
  }
  SmallTile<DT, MUON, KEPT> tile;
  if (KEPT) tile.load_kept(m, ws, x0);
  else tile.load(m, ma, inv, x0);
  tile.template store<kLdX, !KEPT>(m, x0, x, KEPT ? 0 : ((const int*)(ws + m.diag))[kSmallParts]);
  if (MUON && !KEPT)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      int r, c;
      tile.place(m, x0, k, &r, &c);
      if (r < m.rows) store4(m.momentum + (int64_t)r * m.cols + c, m.cols - c, tile.buf[k]);
    }
  __syncthreads();
  f4acc acc[4] = {};  // the wave's 16 columns
#pragma unroll 4
  for (int k = 0; k < n; k += 4) {
    const float b = x[(k + (lane >> 4)) * kLdX + w * 16 + (lane & 15)];
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < nb)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[(j * 16 + (lane & 15)) * kLdS + k + (lane >> 4)], b, acc[j], 0,
                                                      0, 0);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int e = 0; e < 4; e++)
      x[(j * 16 + (lane >> 4) * 4 + e) * kLdX + w * 16 + (lane & 15)] = acc[j][e] * (LAST ? kScale : 1.0f);
  __syncthreads();
  if (!LAST) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = (tid >> 4) + 16 * k, c = (tid & 15) * 4;
      if (r < m.s && x0 + c < m.l)
        *(f4v*)(ws + m.x[0] + (int64_t)r * m.l + x0 + c) = *(const f4v*)&x[r * kLdX + c];
    }
    return;
  }
  // eight values of a row of the matrix a thread
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int r = (tid >> 3) + 32 * k, c = (tid & 7) * 8;
    const int row = m.tall ? x0 + r : r, col = m.tall ? c : x0 + c;
    if (row < m.rows && col < m.cols) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = m.tall ? x[(c + e) * kLdX + r] : x[r * kLdX + c + e];
      if (MUON) step_params<8>(m, ma, out_dt, row, col, v);
      else store_row<8>(m, row, col, v);
    }
  }
}

__global__ void k_clear(int32_t* p) { *p = 0; }

// ---- host ------------------------------------------------------------------

template <bool RB>
using Big = Gemm<F16, 256, 256, 2, 4, true, RB, true>;
template <bool RB>
using Mid = Gemm<F16, 192, 192, 2, 4, true, RB, true>;
template <bool RB>
using Small = Gemm<F16, 128, 128, 2, 4, true, RB, true>;
template <bool RB>
using Tiny = Gemm<F16, 64, 64, 2, 2, true, RB, true>;

struct Source {  // one matrix of the caller's list
  const void* in;
  void* out;
  float* momentum;
  float* master;
  int64_t ld_in, ld_out;
  int32_t rows, cols;
  float lr;
};

int32_t parts_of(int32_t rows, int32_t cols) {
  const int64_t p = ceil_div(rows, kNormTile) * ceil_div(cols, kNormTile);
  return (int32_t)(p < 1 ? 1 : p > kMaxParts ? kMaxParts : p);
}

struct Plan {
  int64_t info_bytes = 0, partial_bytes = 0, run_bytes = 0;
};

bool is_small(const Source& q) { return (q.rows < q.cols ? q.rows : q.cols) <= kSmall; }

// The list in runs of at most kMats matrices and kRunBytes, the ones with a side of at most
// 64 apart: f(table, index of the first, small). The workspace: skip flag, norm
// records, partials, then what the largest run needs (a small matrix's offsets
// count floats from there, another's 16-bit elements).
template <class F>
Plan each_run(const Source* src, int32_t count, F&& f) {
  Plan plan;
  int64_t part0 = 0;
  int32_t index = 0;
  for (int small = 0; small < 2; small++) {
    Table t{};
    int64_t at = 0;
    auto flush = [&]() {
      if (t.n && !small) {
        // A Gram matrix of few 64-tiles leaves CUs idle while each walks all of
        // l: its sums are split so that there are up to two blocks a CU, eight
        // K tiles each at least, and only below 160 tiles. Calls without the
        // split and with it: 65 x 8192 241 and 135 us, 200 x 3000 163 and 136,
        // 700 x 4000 (66 tiles) 210 and 193, 1024 x 4096 (136) 245 and 237,
        // 512 x 512 112 and 112; 1100 x 2731 (171) 252 and 265, 1200 x 3000 (190)
        // 270 and 290. Below the bound it loses where l is short: 768 x 1024
        // (78) 144 and 160, 1024 x 1024 (136) 156 and 178, 1001 x 2731 226 and 233.
        int64_t n = 0;
        auto tiles = [](const Mat& m) { return ceil_div(m.s, 64) * (ceil_div(m.s, 64) + 1) / 2; };
        for (int i = 0; i < t.n; i++) n += tiles(t.m[i]);
        for (int i = 0; i < t.n; i++) {
          Mat& m = t.m[i];
          int64_t splits = n >= 160 ? 1 : 512 / n;
          if (splits > m.l / (8 * kBK)) splits = m.l / (8 * kBK);
          m.splits = (int32_t)(splits < 1 ? 1 : splits);
          m.part = at;
          if (m.splits > 1) at += m.splits * tiles(m) * 64 * 64 * 2;
        }
      }
      if (t.n) f(t, index - t.n, small != 0);
      const int64_t bytes = at * (small ? 4 : 2);
      if (bytes > plan.run_bytes) plan.run_bytes = bytes;
      t.n = 0;
      at = 0;
    };
    for (int32_t k = 0; k < count; k++) {
      const Source& q = src[k];
      if (q.rows <= 0 || q.cols <= 0 || is_small(q) != (small != 0)) continue;
      Mat m{};
      m.in = q.in;
      m.out = q.out;
      m.momentum = q.momentum;
      m.master = q.master;
      m.ld_in = q.ld_in;
      m.ld_out = q.ld_out;
      m.rows = q.rows;
      m.cols = q.cols;
      m.tall = q.rows > q.cols;
      m.s = (int32_t)round_up(m.tall ? q.cols : q.rows, 8);
      m.l = (int32_t)round_up(m.tall ? q.rows : q.cols, 8);
      m.lr = q.lr;
      m.parts = small ? (int32_t)(ceil_div(m.l, 128) > kSmallParts ? kSmallParts : ceil_div(m.l, 128))
                      : parts_of(q.rows, q.cols);
      const int64_t x = round_up((int64_t)m.s * m.l, 128), sq = round_up((int64_t)m.s * m.s, 128);
      const int64_t need = small ? (int64_t)(m.parts + 1) * kSmall * kSmall + 64 + x
                                 : 4 * x + 2 * sq + round_up(4 * (int64_t)m.s, 128);
      if (t.n && (at + need) * (small ? 4 : 2) > kRunBytes) flush();
      if (small) {
        m.a = at;
        m.b = at + (int64_t)m.parts * kSmall * kSmall;
        m.diag = m.b + kSmall * kSmall;  // the parts' exponents and the matrix's
        m.x[0] = m.diag + 64;
      } else {
        m.x[0] = at;
        m.x[1] = at + x;
        m.lo[0] = at + 2 * x;
        m.lo[1] = at + 3 * x;
        m.a = at + 4 * x;
        m.b = m.a + sq;
        m.diag = m.b + sq;
        m.part0 = (int32_t)part0;
        part0 += m.parts;
        index++;
      }
      at += need;
      t.m[t.n++] = m;
      if (t.n == kMats) flush();
    }
    flush();
  }
  plan.info_bytes = 256 + round_up((int64_t)index * (int64_t)sizeof(Info), 256);
  plan.partial_bytes = round_up(part0 * 8, 256);
  return plan;
}

// Sets the launch's first tile of each matrix; returns the tile count.
template <class F>
int64_t tiles_of(Table& t, F&& per) {
  int64_t n = 0;
  for (int i = 0; i < t.n; i++) {
    t.tile0[i] = (int32_t)n;
    n += per(t.m[i]);
  }
  return n;
}

// The 64-tiles of a launch of at most two blocks a CU keep four K tiles (Gemm).
template <class G>
using Deep = typename G::template Staged<G::TM == 64 ? 4 : 2>;
template <class G>
bool is_deep(int64_t blocks) {
  return G::TM == 64 && blocks <= 512;
}

template <class G, bool GRAM>
void launch_symmetric(Table& t, short* ws, const Info* info, int cur, int first, float b, float c, const int32_t* skip,
                      hipStream_t s) {
  constexpr bool SPLIT = GRAM && G::TM == 64;
  auto tiles = [](const Mat& m) {
    const int64_t k = ceil_div(m.s, G::TM);
    return k * (k + 1) / 2;
  };
  bool any = false;
  const int64_t n = tiles_of(t, [&](const Mat& m) {
    any = any || (SPLIT && m.splits > 1);
    return tiles(m) * (SPLIT ? m.splits : 1);
  });
  auto go = [&](auto tile) {
    using H = decltype(tile);
    k_symmetric<H, GRAM, SPLIT><<<dim3((unsigned)n), H::THREADS, 0, s>>>(t, ws, info, cur, first, b, c, skip);
  };
  if (is_deep<G>(n)) go(Deep<G>{});
  else go(G{});
  if (any) k_gram_join<<<dim3((unsigned)tiles_of(t, tiles)), 256, 0, s>>>(t, ws, info, first, skip);
}

template <class G, bool MUON>
void launch_apply(Table& t, short* ws, const Info* info, int cur, int first, bool last, float a, int take_lo,
                  int give_lo, const MuonArgs& ma, int out_dt, hipStream_t s) {
  const int64_t n = tiles_of(t, [](const Mat& m) { return ceil_div(m.s, G::TM) * ceil_div(m.l, G::TN); });
  auto go = [&](auto tile) {
    using H = decltype(tile);
    const dim3 grid((unsigned)n);
    if (last)
      k_apply<H, true, MUON><<<grid, H::THREADS, 0, s>>>(t, ws, info, cur, first, a, take_lo, give_lo, ma, out_dt);
    else
      k_apply<H, false, false><<<grid, H::THREADS, 0, s>>>(t, ws, info, cur, first, a, take_lo, give_lo, ma, out_dt);
  };
  if (is_deep<G>(n)) go(Deep<G>{});
  else go(G{});
}

// The square tile of a launch. Few tiles are bound by the latency of a K tile,
// not by products: 64-tiles while three a CU cover the launch (one 1001 x 2731:
// 233 us with 64-tiles, 382 with 128; one 1024^2: 176 and 250; beyond it, as
// for twelve 768^2, 297 and 279). Else a CU runs one block of 256 or 192 at a
// time or two of 128, whose products take 1.2 times as long for the same area
// (a lone block of 128 on a CU: 1.4 times), and the rounds over the CUs decide.
// (The Gram matrix of 4096 x 14336: 136, 253 and 528 tiles, of which only the
// 192s fill the chip once and no more: 370, 247 and 520 us.)
int tile_of(const Table& t, bool triangle) {
  const int64_t cus = 256, size[4] = {256, 192, 128, 64};
  int64_t n[4] = {0, 0, 0, 0};
  for (int k = 0; k < 4; k++)
    for (int i = 0; i < t.n; i++) {
      const int64_t a = ceil_div(t.m[i].s, size[k]), b = ceil_div(t.m[i].l, size[k]);
      n[k] += triangle ? a * (a + 1) / 2 : a * b;
    }
  if (n[3] <= 3 * cus) return 64;
  const int64_t rest = n[2] % (2 * cus);
  const int64_t cost[3] = {ceil_div(n[0], cus) * 256 * 256 * 10, ceil_div(n[1], cus) * 192 * 192 * 12,
                           (n[2] / (2 * cus) * 24 + (rest > cus ? 24 : rest ? 14 : 0)) * 128 * 128};
  const int k = cost[0] <= cost[1] ? (cost[0] <= cost[2] ? 0 : 2) : (cost[1] <= cost[2] ? 1 : 2);
  return (int)size[k];
}

template <bool MUON>
void iterate(Table& t, short* ws, const Info* info, int steps, const double* coef, bool input_lo, const MuonArgs& ma,
             int out_dt, hipStream_t s) {
  const int sym = tile_of(t, true), app = tile_of(t, false);
  const int32_t* skip = MUON ? ma.skip : nullptr;
  for (int k = 0; k < steps; k++) {
    const float a = (float)coef[3 * k], b = (float)coef[3 * k + 1], c = (float)coef[3 * k + 2];
    const int cur = k & 1, first = k == 0, last = k == steps - 1;
    auto lo = [&](int i) { return i < steps - 2 && (i || input_lo); };
#define DSX_BY_TILE(TILE, F, RB, ...)             \
  do {                                            \
    if (TILE == 256) F<Big<RB>, __VA_ARGS__;      \
    else if (TILE == 192) F<Mid<RB>, __VA_ARGS__; \
    else if (TILE == 128) F<Small<RB>, __VA_ARGS__; \
    else F<Tiny<RB>, __VA_ARGS__;                 \
  } while (0)
    DSX_BY_TILE(sym, launch_symmetric, true, true>(t, ws, info, cur, first, b, c, skip, s));
    DSX_BY_TILE(sym, launch_symmetric, true, false>(t, ws, info, cur, first, b, c, skip, s));
    DSX_BY_TILE(app, launch_apply, false, MUON>(t, ws, info, cur, first, last, a, lo(k), lo(k + 1), ma, out_dt, s));
#undef DSX_BY_TILE
  }
}

// Steps from k0 on that one Gram matrix carries: see the top of this file.
int small_run(const double* coef, int k0, int steps) {
  double growth = 1.0;
  int n = 0;
  for (; k0 + n < steps; n++) {
    const double a = coef[3 * (k0 + n)];
    if (a * a > 1.0) growth *= a * a;
    if (n && growth > 262144.0) break;
  }
  return n;
}

template <int DT, bool MUON>
int drive(const Source* src, int32_t count, int steps, const double* coef, double eps, MuonArgs ma, int out_dt,
          char* base, int64_t bytes, const char* what, hipStream_t s) {
  const Plan plan = each_run(src, count, [](Table&, int, bool) {});
  const int64_t need = plan.info_bytes + plan.partial_bytes + plan.run_bytes;
  if (bytes < need)
    return fail(DSX_EINVAL, "%s: the workspace has %lld bytes, %lld are needed", what, (long long)bytes,
                (long long)need);
  int32_t* skip = (int32_t*)base;
  Info* info = (Info*)(base + 256);
  double* partials = (double*)(base + plan.info_bytes);
  char* run = base + plan.info_bytes + plan.partial_bytes;
  ma.skip = MUON ? skip : nullptr;
  SmallCoef sc{};
  for (int k = 0; k < 3 * steps; k++) sc.c[k] = (float)coef[k];
  // The run of steps from k0 on, without its product; the flag is the input's alone.
  auto small_steps = [&](Table& t, int k0) {
    const dim3 grid((unsigned)tiles_of(t, [](const Mat& m) { return (int64_t)m.parts; }));
    const int n = small_run(coef, k0, steps);
    if (k0) k_small_gram<DSX_F32, false, true><<<grid, 256, 0, s>>>(t, (float*)run, ma);
    else k_small_gram<DT, MUON, false><<<grid, 256, 0, s>>>(t, (float*)run, ma);
    k_small_steps<<<t.n, 640, 0, s>>>(t, (float*)run, sc, k0, n, eps, k0 ? nullptr : ma.skip);
    return k0 + n;
  };
  auto small_apply = [&](Table& t, int k0, bool last) {
    const dim3 grid((unsigned)tiles_of(t, [](const Mat& m) { return ceil_div(m.l, 64); }));
    float* ws = (float*)run;
    if (k0 && last) k_small_apply<DSX_F32, MUON, true, true><<<grid, 256, 0, s>>>(t, ws, ma, out_dt);
    else if (k0) k_small_apply<DSX_F32, MUON, true, false><<<grid, 256, 0, s>>>(t, ws, ma, out_dt);
    else if (last) k_small_apply<DT, MUON, false, true><<<grid, 256, 0, s>>>(t, ws, ma, out_dt);
    else k_small_apply<DT, MUON, false, false><<<grid, 256, 0, s>>>(t, ws, ma, out_dt);
  };
  auto sums = [&](Table& t) {
    const int64_t n = tiles_of(t, [](const Mat& m) { return (int64_t)m.parts; });
    k_sumsq<DT, MUON><<<dim3((unsigned)n), 256, 0, s>>>(t, partials, ma);
  };
  auto rest = [&](Table& t, int at) {
    const int64_t n =
        tiles_of(t, [](const Mat& m) { return ceil_div(m.s, kNormTile) * ceil_div(m.l, kNormTile); });
    k_cast<DT, MUON><<<dim3((unsigned)n), 256, 0, s>>>(t, (short*)run, partials, info + at, eps, ma);
    iterate<MUON>(t, (short*)run, info + at, steps, coef, MUON || DT == DSX_F32, ma, out_dt, s);
  };
  if (MUON) {
    // Every norm is known before anything is written: a small matrix's is the
    // trace of A0, so its steps run (and are run again below, as the runs share
    // their place) before the first cast.
    k_clear<<<1, 1, 0, s>>>(skip);
    each_run(src, count, [&](Table& t, int, bool small) {
      if (small) {
        small_steps(t, 0);
      } else {
        sums(t);
        k_norms<<<t.n, 256, 0, s>>>(t, partials, eps, skip);
      }
    });
  } else {
    each_run(src, count, [&](Table& t, int, bool small) {
      if (!small) sums(t);
    });
  }
  each_run(src, count, [&](Table& t, int at, bool small) {
    if (small) {
      for (int k = 0; k < steps;) {
        const int next = small_steps(t, k);
        small_apply(t, k, next == steps);
        k = next;
      }
    } else {
      rest(t, at);
    }
  });
  return launch_status(what);
}

int check_common(const char* what, int32_t count, int steps, const double* coef, double eps, const void* ws) {
  if (count < 0) return fail(DSX_EINVAL, "%s: count must be >= 0", what);
  if (steps < 1 || steps > 64) return fail(DSX_EINVAL, "%s: steps must be in [1, 64]", what);
  if (!coef) return fail(DSX_EINVAL, "%s: coefficients is NULL", what);
  for (int k = 0; k < 3 * steps; k++)
    if (!isfinite(coef[k])) return fail(DSX_EINVAL, "%s: coefficients must be finite", what);
  if (!(eps >= 1e-20 && eps <= 1.0)) return fail(DSX_EINVAL, "%s: eps must be in [1e-20, 1]", what);
  if (!ws || ((uintptr_t)ws & 255)) return fail(DSX_EINVAL, "%s: the workspace must be 256-byte aligned", what);
  return DSX_OK;
}

int check_shape(const char* what, int32_t k, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows > DSX_MATRIX_MAX_DIM || cols > DSX_MATRIX_MAX_DIM)
    return fail(DSX_EINVAL, "%s: matrix %d is %lld x %lld: dimensions must be in [0, %d]", what, (int)k,
                (long long)rows, (long long)cols, DSX_MATRIX_MAX_DIM);
  return DSX_OK;
}

constexpr int32_t kMaxList = 4096;

}  // namespace

extern "C" {

int64_t dsx_orthogonalize_workspace(const DsxMatrix* mats, int32_t count) {
  if (count < 0 || count > kMaxList || (count && !mats))
    return fail(-1, "dsx_orthogonalize_workspace: bad list");
  Source* src = new (std::nothrow) Source[count ? count : 1];
  if (!src) return fail(-1, "dsx_orthogonalize_workspace: out of memory");
  for (int32_t k = 0; k < count; k++) {
    if (check_shape("dsx_orthogonalize_workspace", k, mats[k].rows, mats[k].cols)) {
      delete[] src;
      return -1;
    }
    src[k] = Source{};
    src[k].rows = (int32_t)mats[k].rows;
    src[k].cols = (int32_t)mats[k].cols;
  }
  const Plan plan = each_run(src, count, [](Table&, int, bool) {});
  delete[] src;
  return plan.info_bytes + plan.partial_bytes + plan.run_bytes;
}

int dsx_orthogonalize(const DsxMatrix* mats, int32_t count, int dtype, int32_t steps, const double* coefficients,
                      double eps, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "dsx_orthogonalize";
  if (count > kMaxList) return fail(DSX_EINVAL, "%s: at most %d matrices", what, kMaxList);
  if (int rc = check_common(what, count, steps, coefficients, eps, workspace)) return rc;
  if (count && !mats) return fail(DSX_EINVAL, "%s: mats is NULL", what);
  if (dtype != DSX_F32 && !dsxi::is16(dtype)) return fail(DSX_EINVAL, "%s: bad dtype %d", what, dtype);
  Source* src = new (std::nothrow) Source[count ? count : 1];
  if (!src) return fail(DSX_EINVAL, "%s: out of memory", what);
  int rc = DSX_OK;
  const uintptr_t unit = dtype == DSX_F32 ? 3 : 1;
  for (int32_t k = 0; k < count && !rc; k++) {
    const DsxMatrix& q = mats[k];
    rc = check_shape(what, k, q.rows, q.cols);
    if (rc || !q.rows || !q.cols) {
      src[k] = Source{};
      continue;
    }
    if (!q.in || !q.out || ((uintptr_t)q.in & unit) || ((uintptr_t)q.out & 1))
      rc = fail(DSX_EINVAL, "%s: matrix %d has a NULL or misaligned pointer", what, (int)k);
    else if (q.ld_in < q.cols || q.ld_out < q.cols)
      rc = fail(DSX_EINVAL, "%s: matrix %d has a row stride below its columns", what, (int)k);
    src[k] = Source{q.in, q.out, nullptr, nullptr, q.ld_in, q.ld_out, (int32_t)q.rows, (int32_t)q.cols, 0.0f};
  }
  if (!rc) {
    const MuonArgs ma{};
    char* base = (char*)workspace;
    hipStream_t s = as_stream(stream);
    if (dtype == DSX_F32)
      rc = drive<DSX_F32, false>(src, count, steps, coefficients, eps, ma, DSX_BF16, base, workspace_bytes, what, s);
    else if (dtype == DSX_F16)
      rc = drive<DSX_F16, false>(src, count, steps, coefficients, eps, ma, DSX_BF16, base, workspace_bytes, what, s);
    else
      rc = drive<DSX_BF16, false>(src, count, steps, coefficients, eps, ma, DSX_BF16, base, workspace_bytes, what, s);
  }
  delete[] src;
  return rc;
}


int64_t dsx_muon_workspace(const DsxMuonParam* params, int32_t count) {
  if (count < 0 || count > kMaxList || (count && !params)) return fail(-1, "dsx_muon_workspace: bad list");
  Source* src = new (std::nothrow) Source[count ? count : 1];
  if (!src) return fail(-1, "dsx_muon_workspace: out of memory");
  for (int32_t k = 0; k < count; k++) {
    if (check_shape("dsx_muon_workspace", k, params[k].rows, params[k].cols)) {
      delete[] src;
      return -1;
    }
    src[k] = Source{};
    src[k].rows = (int32_t)params[k].rows;
    src[k].cols = (int32_t)params[k].cols;
  }
  const Plan plan = each_run(src, count, [](Table&, int, bool) {});
  delete[] src;
  return plan.info_bytes + plan.partial_bytes + plan.run_bytes;
}

int dsx_muon_step(const DsxMuonParam* params, int32_t count, int grad_dtype, int param_dtype, DsxMuonHyper hyper,
                  const float* grad_scale, const double* coefficients, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  const char* what = "dsx_muon_step";
  if (count > kMaxList) return fail(DSX_EINVAL, "%s: at most %d matrices", what, kMaxList);
  if (int rc = check_common(what, count, hyper.steps, coefficients, hyper.eps, workspace)) return rc;
  if (count && !params) return fail(DSX_EINVAL, "%s: params is NULL", what);
  if (grad_dtype != DSX_F32 && !dsxi::is16(grad_dtype)) return fail(DSX_EINVAL, "%s: bad grad dtype", what);
  if (!dsxi::is16(param_dtype)) return fail(DSX_EINVAL, "%s: bad param dtype", what);
  if (!(hyper.momentum >= 0.0 && hyper.momentum < 1.0)) return fail(DSX_EINVAL, "%s: momentum in [0, 1)", what);
  if (!(hyper.decay >= 0.0 && hyper.decay <= 1.0)) return fail(DSX_EINVAL, "%s: decay in [0, 1]", what);
  if ((uintptr_t)grad_scale & 3) return fail(DSX_EINVAL, "%s: misaligned grad_scale", what);
  Source* src = new (std::nothrow) Source[count ? count : 1];
  if (!src) return fail(DSX_EINVAL, "%s: out of memory", what);
  int rc = DSX_OK;
  const uintptr_t unit = grad_dtype == DSX_F32 ? 3 : 1;
  for (int32_t k = 0; k < count && !rc; k++) {
    const DsxMuonParam& q = params[k];
    src[k] = Source{};
    rc = check_shape(what, k, q.rows, q.cols);
    if (rc || !q.rows || !q.cols) continue;
    if (!q.grad || !q.momentum || !q.master || ((uintptr_t)q.grad & unit) || ((uintptr_t)q.momentum & 15) ||
        ((uintptr_t)q.master & 15) || ((uintptr_t)q.param16 & 1))
      rc = fail(DSX_EINVAL, "%s: matrix %d has a NULL or misaligned pointer", what, (int)k);
    else if (q.ld_grad < q.cols)
      rc = fail(DSX_EINVAL, "%s: matrix %d has a row stride below its columns", what, (int)k);
    else if (!isfinite(q.lr))
      rc = fail(DSX_EINVAL, "%s: matrix %d has a step size that is not finite", what, (int)k);
    src[k] = Source{q.grad, q.param16, q.momentum, q.master, q.ld_grad, q.cols, (int32_t)q.rows, (int32_t)q.cols,
                    q.lr};
  }
  if (!rc) {
    MuonArgs ma{};
    ma.grad_scale = grad_scale;
    ma.momentum = (float)hyper.momentum;
    ma.decay = (float)hyper.decay;
    ma.nesterov = hyper.nesterov;
    char* base = (char*)workspace;
    hipStream_t s = as_stream(stream);
    if (grad_dtype == DSX_F32)
      rc = drive<DSX_F32, true>(src, count, hyper.steps, coefficients, hyper.eps, ma, param_dtype, base,
                                workspace_bytes, what, s);
    else if (grad_dtype == DSX_F16)
      rc = drive<DSX_F16, true>(src, count, hyper.steps, coefficients, hyper.eps, ma, param_dtype, base,
                                workspace_bytes, what, s);
    else
      rc = drive<DSX_BF16, true>(src, count, hyper.steps, coefficients, hyper.eps, ma, param_dtype, base,
                                 workspace_bytes, what, s);
  }
  delete[] src;
  return rc;
}

}  // extern "C"
