// dsx_loss.hip -- the cross entropy of a linear layer's logits, and its
// gradients (see include/dsx.h).
//
//   z = x W^T,  loss_t = log sum_v exp z_tv - z_t,target
//   dz_tv = w_t (exp(z_tv - lse_t) - [v = target_t]),  dx = dz W,  dW = dz^T x
//
// The logits are never stored. Forward: a product tile (dsx_gemm.h) reduces its
// columns to a maximum and a sum of exponentials a row in its epilogue, and a
// second launch joins the tiles of a row in order. Backward: for a piece of the
// vocabulary at a time the logits are computed again, the epilogue turns them
// into dz, rounded to the inputs' type for the two products that read it; dW's
// rows of the piece are then complete, and dx's sums stay in fp32 from piece to
// piece.
//
// Rows that do not count take no part in any product: the others are copied
// side by side first (their number is known to the device alone, so grids are
// of the largest size and blocks without rows end at once). The copy also
// gives the product's direct loads the aligned rows that they need.
//
// Bound by the matrix instructions, and where the products are large by the power
// that they take: 8192 rows, 15% of them ignored, of 4096 against 128256, bf16, 25.4
// ms; k_logits 1.14 PFLOP/s, k_dlogits 1.05, dx 1.17, dW 1.28, where one product of
// 8192^3 reaches 1.42 in the library. A fourth of the backward's products computes
// the logits again: kept, they would take 2.1 GB in bf16, and their gradients would
// begin from rounded values. With 768 features (4096 rows against 50257, 1.41 ms) a
// tile's sum is of 12 steps, whose start and epilogue show: k_logits 0.99 PFLOP/s,
// k_dlogits, which writes 412 MB, 0.72, dx and dW 0.95.
//
// In fp16, dz is held times a power of two that takes the largest factor to
// about 2^14, so that probabilities down to 2^-28 keep their digits. (Where the rows'
// factors differ, those of a row 2^r below the largest: down to 2^(r-28). The results'
// own least step is met before that, unless the largest factor is above 2^11.)

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

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

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// What the forward keeps, for the rows that count: row i of them is the
// caller's row index[i].
struct Saved {
  int* count;     // of them
  int* index;     // [tokens]
  int* target;    // [tokens], -1: outside the vocabulary
  int* place;     // [tokens]: the caller's row among those that count, -1: it does not
  float2* stat;   // [tokens]: the largest logit and log2 of the sum of exp2((z - it) log2 e)
  short* x;       // [tokens][ld]
  int64_t ld;
};

// ---- the rows that count ------------------------------------------------------

// Row `from` to rows of whole 16-byte chunks, zeros past the end: chunk c.
__device__ inline s8v chunk_of(const short* from, int c, int cols) {
  if (c * 8 + 8 <= cols) return *(const s8u*)(from + c * 8);
  s8v v = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int e = 0; e < 8; e++)
    if (c * 8 + e < cols) v[e] = from[c * 8 + e];
  return v;
}

// One block: runs of 4096 targets, four a thread, numbered by a scan. `each`
// (may be NULL) gets the loss of the rows that do not count. Where x is given,
// the block then copies the rows that count as well: kCopyHere bytes at most,
// which take it less time than k_copy_rows takes to launch.
constexpr int64_t kCopyHere = 32 << 10;
template <class I>
__global__ __launch_bounds__(1024) void k_select(const I* __restrict__ targets, int tokens, int64_t ignore, int vocab,
                                                 Saved s, float* __restrict__ each, const short* __restrict__ x,
                                                 int64_t ld, int cols) {
  __shared__ int sums[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int base = 0;
  for (int t0 = 0; t0 < tokens; t0 += 4096) {
    const int at = t0 + threadIdx.x * 4;
    int64_t v[4];
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[e] = at + e < tokens ? (int64_t)targets[at + e] : ignore;
      n += v[e] != ignore;
    }
    int before = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(before, d);
      before += lane >= d ? o : 0;
    }
    if (lane == 63) sums[w] = before;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      before += i < w ? sums[i] : 0;
      all += sums[i];
    }
    int to = base + before - n;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (v[e] != ignore) {
        s.place[at + e] = to;
        s.index[to] = at + e;
        s.target[to] = v[e] >= 0 && v[e] < vocab ? (int)v[e] : -1;
        to++;
      } else if (at + e < tokens) {
        s.place[at + e] = -1;
        if (each) each[at + e] = 0.0f;
      }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *s.count = base;
  if (!x) return;
  const int per = (int)(s.ld / 8);  // (the block's own writes to index are visible behind the last barrier)
  for (int i = threadIdx.x; i < base * per; i += 1024) {
    const int r = i / per, c = i - r * per;
    *(s8v*)(s.x + r * s.ld + c * 8) = chunk_of(x + s.index[r] * ld, c, cols);
  }
}

// Rows of any stride and alignment to rows of whole 16-byte chunks, zeros past
// the end: those that count (`index`), or all.
__global__ __launch_bounds__(256) void k_copy_rows(const short* __restrict__ from, int64_t ld, int cols,
                                                   const int* __restrict__ index, const int* __restrict__ count,
                                                   int rows, short* __restrict__ to, int64_t ld_to) {
  const int n = count ? *count : rows;
  const int per = (int)(ld_to / 8);
  for (int r = blockIdx.y * blockDim.y + threadIdx.y; r < n; r += gridDim.y * blockDim.y) {
    const short* p = from + (index ? index[r] : r) * ld;
    for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < per; c += gridDim.x * blockDim.x)
      *(s8v*)(to + r * ld_to + c * 8) = chunk_of(p, c, cols);
  }
}

// ---- the products ---------------------------------------------------------------

struct Logits {
  Operand x, w;      // rows that count (at most), rows of the vocabulary from the piece's first
  int k, m, n;       // width; rows (at most), vocabulary rows of the piece
  int v0;            // the piece's first
  int mt, nt;
  const int* count;
  const int* target;
};

// A block's tile; false: no row of it counts.
template <class G>
__device__ inline bool tile_of(const Logits& p, int* ti, int* tj, int* rows) {
  band_order(xcd_order(blockIdx.x, gridDim.x), p.mt, p.nt, 8, ti, tj);
  *rows = min(*p.count, p.m);
  return *ti * G::TM < *rows;
}

// The largest logit and the sum of exponentials of each row of the tile, and
// the target's logit where it is among its columns.
template <class G>
__global__ DSX_TILE_KERNEL(G) void k_logits(Logits p, float2* __restrict__ part, float* __restrict__ hit) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  int ti, tj, rows;
  if (!tile_of<G>(p, &ti, &tj, &rows)) return;
  const int m0 = ti * G::TM, n0 = tj * G::TN;
  G g;
  g.init();
  Operand x = p.x;
  x.rows = rows;
  g.run(lds, x, p.w, p.w, m0, n0, p.k);
  constexpr int WN = G::TN / G::WTN;
  float2* strip = (float2*)lds;  // [WN][TM]
  const int col0 = n0 + g.wn * G::WTN + (g.lane >> 4) * 4;  // of j = 0, e = 0
#pragma unroll
  for (int i = 0; i < G::MF; i++) {
    const int r = g.wm * G::WTM + i * 16 + (g.lane & 15);
    if (n0 + G::TN > p.n) {
#pragma unroll
      for (int j = 0; j < G::NF; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) g.acc[i][j][e] = col0 + j * 16 + e < p.n ? g.acc[i][j][e] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < G::NF; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) top = fmaxf(top, g.acc[i][j][e]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float base = top == -INFINITY ? 0.0f : top;  // columns past the end alone
    float sum = 0;
#pragma unroll
    for (int j = 0; j < G::NF; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) sum += __builtin_amdgcn_exp2f((g.acc[i][j][e] - base) * kLog2e);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (g.lane < 16) strip[g.wn * G::TM + r] = {top, sum};
    const int at = m0 + r < rows ? p.target[m0 + r] - col0 : -1;
    if (at >= 0 && at < G::WTN && (at & 15) < 4) {
      float z = 0;
#pragma unroll
      for (int j = 0; j < G::NF; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) z = at == j * 16 + e ? g.acc[i][j][e] : z;
      hit[m0 + r] = z;
    }
  }
  __syncthreads();
  for (int r = threadIdx.x; r < G::TM; r += G::THREADS) {
    if (m0 + r >= rows) continue;
    float2 s = strip[r];
#pragma unroll
    for (int i = 1; i < WN; i++) {
      const float2 o = strip[i * G::TM + r];
      const float top = fmaxf(s.x, o.x), base = top == -INFINITY ? 0.0f : top;
      s.y = s.y * exp2f((s.x - base) * kLog2e) + o.y * exp2f((o.x - base) * kLog2e);
      s.x = top;
    }
    part[(int64_t)tj * p.m + m0 + r] = s;
  }
}

// Joins a row's tiles: 32 rows a block, 32 runs of tiles each. `total` (where
// one block has all rows; or NULL): their sum, with `mean` divided by their number.
__global__ __launch_bounds__(1024) void k_rows(const float2* __restrict__ part, const float* __restrict__ hit, int m,
                                               int nt, Saved s, float* __restrict__ loss, float* __restrict__ total,
                                               int mean) {
  __shared__ float2 runs[32][33];
  const int rows = min(*s.count, m), i = threadIdx.x & 31, q = threadIdx.x >> 5, r = blockIdx.x * 32 + i;
  if (blockIdx.x * 32 >= rows && !total) return;
  float top = -INFINITY, sum = 0;
  auto join = [&](const float2& o) {
    const float next = fmaxf(top, o.x), base = next == -INFINITY ? 0.0f : next;
    sum = sum * exp2f((top - base) * kLog2e) + o.y * exp2f((o.x - base) * kLog2e);
    top = next;
  };
  if (r < rows) {
    const int hi = (int)((int64_t)nt * (q + 1) / 32);
#pragma unroll 8
    for (int t = (int)((int64_t)nt * q / 32); t < hi; t++) join(part[(int64_t)t * m + r]);
  }
  runs[q][i] = {top, sum};
  __syncthreads();
  if (q) return;
  float own = 0;
  if (r < rows) {
    for (int k = 1; k < 32; k++) join(runs[k][i]);
    const float log = log2f(sum);
    s.stat[r] = {top, log};
    own = s.target[r] < 0 ? NAN : fmaf(log, kLn2, top - hit[r]);
    loss[s.index[r]] = own;
  }
  if (!total) return;
  double v = own;
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor(v, d);
  if (i == 0) *total = mean ? (float)(v / rows) : (float)v;
}

// The rows' sum, in an order of its own whatever the tokens; with `mean`
// divided by their number.
__global__ __launch_bounds__(1024) void k_total(const float* __restrict__ each, Saved s, int mean,
                                                float* __restrict__ out) {
  __shared__ double sums[16];
  const int rows = *s.count;
  double v = 0;
  for (int r = threadIdx.x; r < rows; r += 1024) v += each[s.index[r]];
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; i++) v += sums[i];
  *out = mean ? (float)(v / rows) : (float)v;
}

// ---- backward -----------------------------------------------------------------

// The factor of a row in dz, and what takes the products with dz to the
// gradients. Where all rows weigh alike, as in a mean, that weight stays out of
// dz: near a target dz is then close to -1, which 16 bits hold, where w times it
// would be off by the same 2^-9 of bf16 in every row. fp16's power of two goes by
// the largest factor.
struct Weights {
  const float* d_loss;
  const float* power;  // the power of two in device memory, or NULL: `one`
  float one;
  int reduction;
  __device__ inline float times() const { return power ? *power : one; }
  __device__ inline float of_row(const int* index, int r, int target) const {
    return target < 0 ? NAN : reduction == DSX_REDUCE_NONE ? d_loss[index[r]] * times() : times();
  }
  // (The mean of no row is NaN, but there is nothing it could reach.)
  __device__ inline float of_products(int rows) const {
    const float w = reduction == DSX_REDUCE_NONE ? 1.0f : reduction == DSX_REDUCE_MEAN ? *d_loss / (float)rows : *d_loss;
    return rows ? w / times() : 0.0f;
  }
};

// Takes the largest finite of the rows' factors to [2^14, 2^15).
__global__ __launch_bounds__(1024) void k_power(const float* __restrict__ d_loss, Saved s, float* __restrict__ power) {
  __shared__ float tops[16];
  const int rows = *s.count;
  float top = 0;
  for (int r = threadIdx.x; r < rows; r += 1024) {
    const float v = fabsf(d_loss[s.index[r]]);
    top = fmaxf(top, v < INFINITY ? v : 0.0f);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; i++) top = fmaxf(top, tops[i]);
  int e = 15;
  if (top > 0.0f) frexpf(top, &e);  // top < 2^e
  *power = ldexpf(1.0f, max(-100, min(100, 15 - e)));
}

// dz of a piece, [rows][ld] with zeros from the piece's end to ld.
template <class G, class T>
__global__ DSX_TILE_KERNEL(G) void k_dlogits(Logits p, const float2* __restrict__ stat,
                                             Weights weights, const int* __restrict__ index,
                                             short* __restrict__ dz, int64_t ld) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  int ti, tj, rows;
  if (!tile_of<G>(p, &ti, &tj, &rows)) return;
  const int m0 = ti * G::TM, n0 = tj * G::TN;
  G g;
  g.init();
  Operand x = p.x;
  x.rows = rows;
  g.run(lds, x, p.w, p.w, m0, n0, p.k);
  struct Row {
    float top, log, w;
    int target;
  };
  g.template emit<false>(
      lds,
      [&](int r, int) {
        if (m0 + r >= rows) return Row{};
        const float2 s = stat[m0 + r];
        const int target = p.target[m0 + r];
        return Row{s.x, s.y, weights.of_row(index, m0 + r, target), target - p.v0};
      },
      [&](int r, int c, float* v, float*, const Row& q) {
        const int n = n0 + c;
        if (m0 + r >= rows || n >= ld) return;
        s8v o;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float y = __builtin_amdgcn_exp2f(fmaf(v[e] - q.top, kLog2e, -q.log));
          o[e] = n + e < p.n ? T::round(q.w * (n + e == q.target ? y - 1.0f : y)) : (short)0;
        }
        *(s8v*)(dz + (m0 + r) * ld + n) = o;
      },
      [](int, int, const float*) {});
}

// dx's sums of a piece: split s of the blocks adds its part of the piece to
// plane s.
struct InputGrad {
  Operand dz, w;
  int k, m, n;      // vocabulary rows of the piece, rows (at most), width
  int mt, nt, splits, per;
  const int* count;
  float* planes;    // [splits][m][ld]
  int64_t ld;
  int first;        // the planes hold nothing yet
};
template <class G>
__global__ DSX_TILE_KERNEL(G) void k_input_grad(InputGrad p) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  const int tiles = p.mt * p.nt, bid = xcd_order(blockIdx.x, gridDim.x), split = bid / tiles;
  int ti, tj;
  band_order(bid - split * tiles, p.mt, p.nt, 8, &ti, &tj);
  const int rows = min(*p.count, p.m);
  if (ti * G::TM >= rows) return;
  G g;
  g.init();
  const int k0 = split * p.per * kBK, k1 = min(k0 + p.per * kBK, p.k);
  Operand a = p.dz, b = p.w;
  a.rows = rows;
  a.p += k0;
  b.p += k0 * b.ld;
  g.run(lds, a, b, b, ti * G::TM, tj * G::TN, k1 - k0);
  float* plane = p.planes + (int64_t)split * p.m * p.ld;
  struct Raw {
    f4v a, b;
  };
  g.template emit<false>(
      lds,
      [&](int r, int c) {
        const int m = ti * G::TM + r, n = tj * G::TN + c;
        if (p.first || m >= rows || n >= p.n) return Raw{};
        const float* q = plane + m * p.ld + n;
        return Raw{*(const f4v*)q, *(const f4v*)(q + 4)};
      },
      [&](int r, int c, float* v, float*, const Raw& raw) {
        const int m = ti * G::TM + r, n = tj * G::TN + c;
        if (m >= rows || n >= p.n) return;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[e] += raw.a[e];
          v[e + 4] += raw.b[e];
        }
        G::put8(plane + m * p.ld + n, v);
      },
      [](int, int, const float*) {});
}

// The planes added in order and rounded; zeros in rows that do not count.
template <class T>
__global__ __launch_bounds__(256) void k_input_join(const float* __restrict__ planes, int splits, int m, int64_t ld,
                                                    int n, Saved s, Weights weights,
                                                    short* __restrict__ dx) {
  const float f = weights.of_products(*s.count);
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= n) return;
  for (int t = blockIdx.y; t < m; t += gridDim.y) {
    const int r = s.place[t];
    f4v a = {}, b = {};
#pragma unroll 8
    for (int k = 0; k < (r < 0 ? 0 : splits); k++) {
      const float* q = planes + ((int64_t)k * m + r) * ld + c;
      a += *(const f4v*)q;
      b += *(const f4v*)(q + 4);
    }
    s8v o;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      o[e] = r < 0 ? (short)0 : T::round(a[e] * f);
      o[e + 4] = r < 0 ? (short)0 : T::round(b[e] * f);
    }
    short* to = dx + (int64_t)t * n + c;
    if (c + 8 <= n)
      *(s8u*)to = o;
    else
      for (int e = 0; e < 8; e++)
        if (c + e < n) to[e] = o[e];
  }
}

struct WeightGrad {
  Operand dz, x;
  int m, n, mt, nt;  // vocabulary rows of the piece, width
  const int* count;
  Weights weights;
  short* out;        // the piece's rows, contiguous
};
template <class G, class T>
__global__ DSX_TILE_KERNEL(G) void k_weight_grad(WeightGrad p) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  int ti, tj;
  band_order(xcd_order(blockIdx.x, gridDim.x), p.mt, p.nt, 8, &ti, &tj);
  G g;
  g.init();
  g.run(lds, p.dz, p.x, p.x, ti * G::TM, tj * G::TN, *p.count);
  const float f = p.weights.of_products(*p.count);
  g.template emit<false>(
      lds, [](int, int) { return Nothing{}; },
      [&](int r, int c, float* v, float*, const Nothing&) {
        const int m = ti * G::TM + r, n = tj * G::TN + c;
        if (m >= p.m || n >= p.n) return;
        s8v o;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = T::round(v[e] * f);
        short* to = p.out + (int64_t)m * p.n + n;
        if (n + 8 <= p.n)
          *(s8u*)to = o;
        else
          for (int e = 0; e < 8; e++)
            if (n + e < p.n) to[e] = o[e];
      },
      [](int, int, const float*) {});
}

// ---- host ------------------------------------------------------------------

bool aligned(const void* p, int64_t ld, int64_t cols) {
  return !((uintptr_t)p & 15) && ld % 8 == 0 && cols % 8 == 0 && ld <= (1 << 22);
}

// The tile of a product of m x n: as few rows as a few tokens need, else
// square ones, 64 wide where there are few.
int tile_of(int64_t m, int64_t n) {
  if (m <= 16) return 16;
  if (m <= 32) return 32;
  if (m <= 64 || ceil_div(m, 64) * ceil_div(n, 64) <= 2 * kCus) return 64;
  return square_tile(ceil_div(m, 256) * ceil_div(n, 256), ceil_div(m, 128) * ceil_div(n, 128));
}
int rows_of_tile(int tile) { return tile; }
int cols_of_tile(int tile) { return tile == 16 ? 128 : tile == 32 ? 64 : tile; }

struct Sizes {
  int64_t t, d, v, ld;      // ld: the width in whole chunks
  bool copied;              // the weight is
  int tile;                 // of the logits
  int64_t nt;               // its columns' tiles, of the whole vocabulary
  int64_t piece, ld_piece;  // vocabulary rows of a piece of the backward, and dz's row stride
  int dx_tile, splits;
};

// dz of a piece: at most this many bytes. (8192 x 4096 against 128256 rows, bf16,
// dz and both products: 19.0 ms with 128 MiB, 18.8 with 256, 19.4 with 512, 19.3
// with 1 GiB; 4096 x 768 against 50257: 1.17 ms with 256, 1.06 in one piece. One size
// for all widths, 3% from the best for the wide one.)
constexpr int64_t kPieceBytes = (int64_t)512 << 20;

// Tile and splits of dx's sum over k vocabulary rows, which is long where its
// tiles are few. In us: a K tile of 64 takes a block of 256 1.6 us and two of 128
// on a CU 1.2 times as long for the same area (square_tile); a round of small
// tiles that fills half the CUs' places takes 0.58 of one; a split's sums are
// written and read at 4 TB/s.
void share_out(int64_t m, int64_t n, int64_t k, int* tile, int* splits) {
  const int64_t kt = ceil_div(k, kBK);
  *tile = tile_of(m, n);
  *splits = 1;
  double least = INFINITY;
  for (int t = *tile < 128 ? *tile : 128; t <= (*tile < 128 ? *tile : 256); t *= 2) {
    const int64_t tiles = ceil_div(m, rows_of_tile(t)) * ceil_div(n, cols_of_tile(t));
    for (int64_t s = 1; s <= 64 && (s == 1 || kt / s >= 4); s++) {
      const int64_t blocks = tiles * s, slots = t == 256 ? kCus : t == 128 ? 2 * kCus : 4 * kCus;
      const int64_t rest = blocks % slots;
      double rounds = (double)(blocks / slots) + (rest == 0 ? 0.0 : t == 256 || rest > slots / 2 ? 1.0 : 0.58);
      const double area = (double)rows_of_tile(t) * cols_of_tile(t) * (double)(slots / kCus) / 65536.0;
      const double us = rounds * (double)ceil_div(kt, s) * 1.6 * (t == 256 ? 1.0 : area < 0.3 ? 0.36 : 1.2 * area) +
                        (double)s * (double)(m * n) * 8.0 / 4e6;
      if (us < least) {
        least = us;
        *tile = t;
        *splits = (int)s;
      }
    }
  }
}

Sizes sizes_of(const DsxLoss& q) {
  Sizes z{};
  z.t = q.tokens;
  z.d = q.width;
  z.v = q.vocab;
  z.ld = round_up(q.width, 8);
  z.copied = !aligned(q.weight, q.ld_weight, q.width);
  z.tile = tile_of(z.t, z.v);
  z.nt = ceil_div(z.v, cols_of_tile(z.tile));
  const int64_t fit = kPieceBytes / 2 / (z.t > 0 ? z.t : 1) / 256 * 256, least = 1024;
  const int64_t most = fit > least ? fit : least;
  const int64_t pieces = ceil_div(z.v, most);
  z.piece = pieces > 1 ? round_up(ceil_div(z.v, pieces), 256) : z.v;
  z.ld_piece = round_up(z.piece, 8);
  share_out(z.t, z.d, z.piece, &z.dx_tile, &z.splits);
  return z;
}

Saved saved_of(const DsxLoss& q, int64_t* bytes) {
  Saved s{};
  const uintptr_t p = (uintptr_t)q.saved;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    char* r = (char*)(p + at);
    at += round_up(n, 256);
    return r;
  };
  s.ld = round_up(q.width, 8);
  s.count = (int*)take(4);
  s.index = (int*)take(q.tokens * 4);
  s.target = (int*)take(q.tokens * 4);
  s.place = (int*)take(q.tokens * 4);
  s.stat = (float2*)take(q.tokens * 8);
  s.x = (short*)take(q.tokens * s.ld * 2);
  if (bytes) *bytes = at;
  return s;
}

struct Work {
  short* weight;          // aligned copy
  float2* part;           // forward: [nt][tokens]
  float* hit;
  float* each;
  float* power;           // backward
  short* dz;
  float* planes;
  int64_t total;
};
Work work_of(const DsxLoss& q, const Sizes& z, bool backward) {
  Work w{};
  const uintptr_t p = (uintptr_t)q.workspace;  // sizes are asked for with none
  int64_t at = 0;
  auto take = [&](int64_t n) {
    char* r = (char*)(p + at);
    at += round_up(n, 256);
    return r;
  };
  if (z.copied) w.weight = (short*)take(z.v * z.ld * 2);
  if (!backward) {
    w.part = (float2*)take(z.nt * z.t * 8);
    w.hit = (float*)take(z.t * 4);
    w.each = (float*)take(z.t * 4);
  } else {
    w.power = (float*)take(4);
    w.dz = (short*)take(z.t * z.ld_piece * 2);
    w.planes = (float*)take(z.splits * z.t * z.ld * 4);
  }
  w.total = at + 256;
  return w;
}

// As many threads for a row as it has chunks, rows for the others of a block of 256.
void copy_rows(const short* from, int64_t ld, int64_t cols, const int* index, const int* count, int64_t rows, short* to,
               int64_t ld_to, hipStream_t s) {
  unsigned x = 1;
  while (x < 256 && x < ld_to / 8) x *= 2;
  const int64_t blocks = ceil_div(rows, 256 / x);
  k_copy_rows<<<dim3((unsigned)ceil_div(ld_to / 8, x), (unsigned)(blocks < 65535 ? blocks : 65535)), dim3(x, 256 / x), 0,
                s>>>(from, ld, (int)cols, index, count, (int)rows, to, ld_to);
}

void copy_weight(const DsxLoss& q, const Sizes& z, const Work& w, hipStream_t s) {
  if (!z.copied) return;
  copy_rows((const short*)q.weight, q.ld_weight, z.d, nullptr, nullptr, z.v, w.weight, z.ld, s);
}

Logits logits_of(const DsxLoss& q, const Sizes& z, const Saved& s, const Work& w, int64_t v0, int64_t n, int tile) {
  Logits p{};
  const int64_t ld = z.copied ? z.ld : q.ld_weight;
  p.x = {s.x, s.ld, (int)z.t};
  p.w = {(z.copied ? w.weight : (const short*)q.weight) + v0 * ld, ld, (int)n};
  p.k = (int)z.ld;
  p.m = (int)z.t;
  p.n = (int)n;
  p.v0 = (int)v0;
  p.mt = (int)ceil_div(z.t, rows_of_tile(tile));
  p.nt = (int)ceil_div(n, cols_of_tile(tile));
  p.count = s.count;
  p.target = s.target;
  return p;
}

// RUN(TM, TN, WM, WN, STAGES) for the tile of a launch of `blocks`.
#define DSX_BY_TILE(TILE, BLOCKS, RUN)                                   \
  do {                                                                   \
    const bool deep_ = (BLOCKS) <= 2 * kCus;                             \
    if ((TILE) == 16) RUN(16, 128, 1, 4, 2);                             \
    else if ((TILE) == 32 && deep_) RUN(32, 64, 2, 2, 4);                \
    else if ((TILE) == 32) RUN(32, 64, 2, 2, 2);                         \
    else if ((TILE) == 64 && deep_) RUN(64, 64, 2, 2, 4);                \
    else if ((TILE) == 64) RUN(64, 64, 2, 2, 2);                         \
    else if ((TILE) == 128) RUN(128, 128, 2, 4, 2);                      \
    else RUN(256, 256, 2, 4, 2);                                         \
  } while (0)

template <class T>
int forward(const DsxLoss& q, float* loss, hipStream_t st) {
  const Sizes z = sizes_of(q);
  const Saved s = saved_of(q, nullptr);
  const Work w = work_of(q, z, false);
  const bool none = q.reduction == DSX_REDUCE_NONE;
  float* each = none ? loss : w.each;
  const bool here = z.t * z.ld * 2 <= kCopyHere;
  const short* x = here ? (const short*)q.x : nullptr;
  if (q.target_bytes == 8)
    k_select<<<1, 1024, 0, st>>>((const int64_t*)q.targets, (int)z.t, q.ignore_index, (int)z.v, s, none ? loss : nullptr, x,
                                 q.ld_x, (int)z.d);
  else
    k_select<<<1, 1024, 0, st>>>((const int32_t*)q.targets, (int)z.t, q.ignore_index, (int)z.v, s, none ? loss : nullptr, x,
                                 q.ld_x, (int)z.d);
  if (!z.t) {
    if (!none) k_total<<<1, 1024, 0, st>>>(nullptr, s, q.reduction == DSX_REDUCE_MEAN, loss);
    return launch_status("dsx_loss_forward");
  }
  if (!here) copy_rows((const short*)q.x, q.ld_x, z.d, s.index, s.count, z.t, s.x, s.ld, st);
  copy_weight(q, z, w, st);
  const Logits p = logits_of(q, z, s, w, 0, z.v, z.tile);
  const dim3 grid((unsigned)(p.mt * p.nt));
#define RUN(TM, TN, WM, WN, STAGES)                                             \
  do {                                                                          \
    using G = Gemm<T, TM, TN, WM, WN, true, true, true, false, STAGES>;         \
    k_logits<G><<<grid, G::THREADS, 0, st>>>(p, w.part, w.hit);                 \
  } while (0)
  DSX_BY_TILE(z.tile, (int64_t)p.mt * p.nt, RUN);
#undef RUN
  const bool one = !none && z.t <= 32, mean = q.reduction == DSX_REDUCE_MEAN;
  k_rows<<<dim3((unsigned)ceil_div(z.t, 32)), 1024, 0, st>>>(w.part, w.hit, (int)z.t, (int)z.nt, s, each,
                                                             one ? loss : nullptr, mean);
  if (!none && !one) k_total<<<1, 1024, 0, st>>>(each, s, mean, loss);
  return launch_status("dsx_loss_forward");
}

template <class T>
int backward(const DsxLoss& q, const float* d_loss, short* dx, short* dw, hipStream_t st) {
  const Sizes z = sizes_of(q);
  const Saved s = saved_of(q, nullptr);
  const Work w = work_of(q, z, true);
  const bool half = q.dtype == DSX_F16, none = q.reduction == DSX_REDUCE_NONE;
  const Weights weights{d_loss, half && none ? w.power : nullptr, half ? 0x1p14f : 1.0f, q.reduction};
  if (weights.power) k_power<<<1, 1024, 0, st>>>(d_loss, s, w.power);
  copy_weight(q, z, w, st);
  for (int64_t v0 = 0; v0 < z.v; v0 += z.piece) {
    const int64_t n = z.v - v0 < z.piece ? z.v - v0 : z.piece, ld = round_up(n, 8);
    // Up to 512 features the epilogue, dz's way to memory, takes as long as the sum:
    // beside a second block's products it costs less. With gradients, 4096 rows
    // against 50257, bf16, 256- and 128-tiles: 128 features 650 and 605 us, 384 1169
    // and 1112, 512 1343 and 1327; 8192 rows of 768, 2932 and 2963.
    const int whole = tile_of(z.t, n), tile = whole == 256 && z.d <= 512 ? 128 : whole;
    const Logits p = logits_of(q, z, s, w, v0, n, tile);
    const dim3 grid((unsigned)(p.mt * p.nt));
#define RUN(TM, TN, WM, WN, STAGES)                                                              \
  do {                                                                                           \
    using G = Gemm<T, TM, TN, WM, WN, true, true, true, false, STAGES>;                          \
    k_dlogits<G, T><<<grid, G::THREADS, 0, st>>>(p, s.stat, weights, s.index, w.dz, ld);         \
  } while (0)
    if (z.t) DSX_BY_TILE(tile, (int64_t)p.mt * p.nt, RUN);
#undef RUN
    if (dx && z.t) {
      InputGrad g{};
      g.dz = {w.dz, ld, (int)z.t};
      g.w = p.w;
      g.w.rows = (int)z.ld;
      g.k = (int)n;
      g.m = (int)z.t;
      g.n = (int)z.d;
      g.mt = (int)ceil_div(z.t, rows_of_tile(z.dx_tile));
      g.nt = (int)ceil_div(z.d, cols_of_tile(z.dx_tile));
      g.splits = z.splits;
      g.per = (int)ceil_div(ceil_div(n, kBK), z.splits);
      g.count = s.count;
      g.planes = w.planes;
      g.ld = z.ld;
      g.first = v0 == 0;
      const dim3 dgrid((unsigned)(g.mt * g.nt * g.splits));
#define RUN(TM, TN, WM, WN, STAGES)                                              \
  do {                                                                           \
    using G = Gemm<T, TM, TN, WM, WN, true, false, true, false, STAGES>;         \
    k_input_grad<G><<<dgrid, G::THREADS, 0, st>>>(g);                            \
  } while (0)
      DSX_BY_TILE(z.dx_tile, (int64_t)g.mt * g.nt * g.splits, RUN);
#undef RUN
    }
    if (dw) {
      WeightGrad g{};
      g.dz = {w.dz, ld, (int)ld};
      g.x = {s.x, s.ld, (int)z.ld};
      g.m = (int)n;
      g.n = (int)z.d;
      g.count = s.count;
      g.weights = weights;
      g.out = dw + v0 * z.d;
      const int tile = square_tile(ceil_div(n, 256) * ceil_div(z.d, 256), ceil_div(n, 128) * ceil_div(z.d, 128));
      g.mt = (int)ceil_div(n, tile);
      g.nt = (int)ceil_div(z.d, tile);
      const dim3 wgrid((unsigned)(g.mt * g.nt));
      if (tile == 256) {
        using G = Gemm<T, 256, 256, 2, 4, false, false, true>;
        k_weight_grad<G, T><<<wgrid, G::THREADS, 0, st>>>(g);
      } else {
        using G = Gemm<T, 128, 128, 2, 4, false, false, true>;
        k_weight_grad<G, T><<<wgrid, G::THREADS, 0, st>>>(g);
      }
    }
  }
  if (dx && z.t)
    k_input_join<T><<<dim3((unsigned)ceil_div(z.d, 2048), (unsigned)(z.t < 65535 ? z.t : 65535)), 256, 0, st>>>(
        w.planes, z.splits, (int)z.t, z.ld, (int)z.d, s, weights, dx);
  return launch_status("dsx_loss_backward");
}

int check(const char* what, const DsxLoss* q) {
  if (!q) return fail(DSX_EINVAL, "%s: the argument block is NULL", what);
  if (!dsxi::is16(q->dtype)) return fail(DSX_EINVAL, "%s: dtype must be DSX_F16 or DSX_BF16", what);
  if (q->tokens < 0 || q->tokens > DSX_MATRIX_MAX_DIM || q->width < 1 || q->width > DSX_MATRIX_MAX_DIM ||
      q->vocab < 1 || q->vocab > DSX_MATRIX_MAX_DIM)
    return fail(DSX_EINVAL, "%s: tokens in [0, %d], width and vocab in [1, %d]", what, DSX_MATRIX_MAX_DIM,
                DSX_MATRIX_MAX_DIM);
  if (q->target_bytes != 4 && q->target_bytes != 8) return fail(DSX_EINVAL, "%s: targets are of 4 or 8 bytes", what);
  if (q->reduction < DSX_REDUCE_NONE || q->reduction > DSX_REDUCE_SUM)
    return fail(DSX_EINVAL, "%s: bad reduction %d", what, q->reduction);
  if (q->ld_weight < q->width) return fail(DSX_EINVAL, "%s: a row stride is below the row's length", what);
  return DSX_OK;
}

int check_device(const char* what, const DsxLoss* q, bool backward) {
  if (!q->weight || ((uintptr_t)q->weight & 1)) return fail(DSX_EINVAL, "%s: weight is NULL or misaligned", what);
  if (!q->saved || ((uintptr_t)q->saved & 255)) return fail(DSX_EINVAL, "%s: saved is NULL or misaligned", what);
  const int64_t need = work_of(*q, sizes_of(*q), backward).total;
  if (!q->workspace || ((uintptr_t)q->workspace & 255) || q->workspace_bytes < need)
    return fail(DSX_EINVAL, "%s: the workspace must be 256-byte aligned and of %lld bytes", what, (long long)need);
  return DSX_OK;
}

}  // namespace

extern "C" {

int64_t dsx_loss_saved_bytes(const DsxLoss* args) {
  if (check("dsx_loss_saved_bytes", args)) return -1;
  int64_t bytes;
  saved_of(*args, &bytes);
  return bytes;
}

int64_t dsx_loss_workspace_bytes(const DsxLoss* args, int32_t backward) {
  if (check("dsx_loss_workspace_bytes", args)) return -1;
  return work_of(*args, sizes_of(*args), backward != 0).total;
}

int dsx_loss_forward(const DsxLoss* args, float* loss, void* stream) {
  const char* what = "dsx_loss_forward";
  if (int rc = check(what, args)) return rc;
  if (int rc = check_device(what, args, false)) return rc;
  if (!loss || ((uintptr_t)loss & 3)) return fail(DSX_EINVAL, "%s: loss is NULL or misaligned", what);
  if (args->tokens * args->vocab > (int64_t)1 << 38)  // a launch's threads are counted in 32 bits
    return fail(DSX_EINVAL, "%s: tokens times vocab must be at most 2^38", what);
  if (args->tokens && (!args->x || ((uintptr_t)args->x & 1) || args->ld_x < args->width))
    return fail(DSX_EINVAL, "%s: x is NULL or misaligned, or its row stride below the row's length", what);
  if (args->tokens && (!args->targets || ((uintptr_t)args->targets & (args->target_bytes - 1))))
    return fail(DSX_EINVAL, "%s: targets is NULL or misaligned", what);
  hipStream_t s = as_stream(stream);
  return args->dtype == DSX_F16 ? forward<F16>(*args, loss, s) : forward<BF16>(*args, loss, s);
}

int dsx_loss_backward(const DsxLoss* args, const float* d_loss, void* dx, void* dweight, void* stream) {
  const char* what = "dsx_loss_backward";
  if (int rc = check(what, args)) return rc;
  if (int rc = check_device(what, args, true)) return rc;
  if ((!d_loss && (args->tokens || args->reduction)) || ((uintptr_t)d_loss & 3))
    return fail(DSX_EINVAL, "%s: d_loss is NULL or misaligned", what);
  if (((uintptr_t)dx | (uintptr_t)dweight) & 1) return fail(DSX_EINVAL, "%s: misaligned gradient", what);
  hipStream_t s = as_stream(stream);
  return args->dtype == DSX_F16 ? backward<F16>(*args, d_loss, (short*)dx, (short*)dweight, s)
                                : backward<BF16>(*args, d_loss, (short*)dx, (short*)dweight, s);
}

}  // extern "C"
