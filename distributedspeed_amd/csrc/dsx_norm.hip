// dsx_norm.hip -- the RMS norms before and after a block, fused with the
// block's gate and its residual (see include/dsx.h).
//
//   z = rms(y) w1 (or y);  h = beta r + alpha gate z;  n = rms(h) w2 (or none)
//   rms(v) = v rstd, rstd = 1 / sqrt(mean(v^2) + eps)
//
// and, with t = w2 dn, the gradients
//   dH = dh + rstd2 (t - hhat mean(t hhat)),   dr = beta dH,
//   dgate = sum alpha z dH,   dz = alpha gate dH,   dw2 = sum dn hhat,
//   dy = rstd1 (w1 dz - yhat mean(w1 dz yhat)),     dw1 = sum dz yhat.
//
// Both directions are one pass over the rows. A row belongs to one block, eight
// elements a thread, and stays in registers between the sums over it. The
// backward's second mean depends on dH and so on the first, but expands to sums
// that do not:  with q = alpha gate w1 y,
//   sum(w1 dz y) = sum q (dh + rstd2 t) - rstd2^2 mean(t hhat) sum q h,
// so that all three sums are taken at once, with one exchange between waves.
// h is computed again from r and y in fp32 rather than read back rounded. The
// column sums stay in registers over all the rows of a block, which writes one
// row of partial sums; a second launch adds those in order (no atomics: the
// result does not depend on timing).
//
// Rows wider than 8192 take the same formulas in column-strided loops that
// read the inputs again (k_wide_*).

#include <hip/hip_runtime.h>
#include <math.h>
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

constexpr int kWidest = 8192;  // of a row kept in registers: 512 threads of two chunks of eight elements

struct Args {
  const void* r;
  const void* y;     // NULL: no branch
  const void* w1;    // NULL: no norm after the block
  const void* gate;  // NULL: none
  const void* w2;    // NULL: no norm before the next block
  int64_t ld_r, ld_y;
  int rows, width;
  int per_sample;    // rows that share a row of the gate
  float alpha, beta, eps;
  float* rstd;       // [2][rows], or NULL
};

template <int DT>
struct Elem {
  using T = typename std::conditional<DT == DSX_F16, F16, BF16>::type;
  typedef s8v Raw;
  static __device__ inline Raw load(const void* p, int64_t at, int left) {
    const short* q = (const short*)p + at;
    if (left >= 8) return *(const s8u*)q;
    Raw v = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int e = 0; e < 8; e++)
      if (e < left) v[e] = q[e];
    return v;
  }
  static __device__ inline float at(const Raw& v, int e) { return T::widen(v[e]); }
  static __device__ inline void store(void* p, int64_t at, int left, const float* v) {
    short* q = (short*)p + at;
    s8v w;
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = T::round(v[e]);
    if (left >= 8)
      *(s8u*)q = w;
    else
      for (int e = 0; e < 8; e++)
        if (e < left) q[e] = w[e];
  }
  static __device__ inline void put(void* p, int64_t at, float v) { ((short*)p)[at] = T::round(v); }
  static __device__ inline float get(const void* p, int64_t at) { return T::widen(((const short*)p)[at]); }
};
template <>
struct Elem<DSX_F32> {
  struct Raw {
    f4v a, b;
  };
  static __device__ inline Raw load(const void* p, int64_t at, int left) {
    const float* q = (const float*)p + at;
    Raw v;
    if (left >= 8) {
      v.a = *(const f4u*)q;
      v.b = *(const f4u*)(q + 4);
    } else {
      v.a = v.b = f4v{0, 0, 0, 0};
      for (int e = 0; e < 4; e++) {
        if (e < left) v.a[e] = q[e];
        if (e + 4 < left) v.b[e] = q[e + 4];
      }
    }
    return v;
  }
  static __device__ inline float at(const Raw& v, int e) { return e < 4 ? v.a[e] : v.b[e & 3]; }
  static __device__ inline void store(void* p, int64_t at, int left, const float* v) {
    float* q = (float*)p + at;
    if (left >= 8) {
      *(f4u*)q = f4v{v[0], v[1], v[2], v[3]};
      *(f4u*)(q + 4) = f4v{v[4], v[5], v[6], v[7]};
    } else {
      for (int e = 0; e < 8; e++)
        if (e < left) q[e] = v[e];
    }
  }
  static __device__ inline void put(void* p, int64_t at, float v) { ((float*)p)[at] = v; }
  static __device__ inline float get(const void* p, int64_t at) { return ((const float*)p)[at]; }
};

// Sums of N values over a block of W threads, the same in every thread. The
// buffer is used in turn (`turn` counts the calls), so one barrier a call is
// enough.
template <int W, int N>
__device__ inline void block_sum(float* v, float (*buf)[16][N], int turn) {
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int d = 32; d; d >>= 1) v[k] += __shfl_xor(v[k], d);
  if (W == 64) return;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < N; k++) buf[turn & 1][w][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++) {
    float s = 0;
#pragma unroll
    for (int i = 0; i < W / 64; i++) s += buf[turn & 1][i][k];
    v[k] = s;
  }
}

template <int DT>
__device__ inline void widen8(const typename Elem<DT>::Raw& v, float* f) {
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = Elem<DT>::at(v, e);
}

// Eight elements a thread and chunk; chunk v of a row begins at column
// (v W + thread) 8.
template <int DT, int W, int NV>
__global__ __launch_bounds__(W) void k_forward(Args a, void* __restrict__ hidden, void* __restrict__ normed) {
  using E = Elem<DT>;
  __shared__ float buf[2][16][1];
  int c[NV], left[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) {
    c[v] = (v * W + threadIdx.x) * 8;
    left[v] = a.width - c[v];
  }
  const float inv_width = 1.0f / a.width;
  float w1[NV][8], w2[NV][8], gate[NV][8];
  auto vector = [&](const void* p, int64_t at, float (*f)[8]) {
#pragma unroll
    for (int v = 0; v < NV; v++) widen8<DT>(left[v] > 0 ? E::load(p, at + c[v], left[v]) : typename E::Raw{}, f[v]);
  };
  if (a.w1) vector(a.w1, 0, w1);
  if (a.w2) vector(a.w2, 0, w2);
  int sample = -1, turn = 0;
  int row = blockIdx.x;
  typename E::Raw nr[NV] = {}, ny[NV] = {};
  auto fetch = [&](int k) {
    if (k >= a.rows) return;
#pragma unroll
    for (int v = 0; v < NV; v++) {
      if (left[v] <= 0) continue;
      nr[v] = E::load(a.r, k * a.ld_r + c[v], left[v]);
      if (a.y) ny[v] = E::load(a.y, k * a.ld_y + c[v], left[v]);
    }
  };
  fetch(row);
  for (; row < a.rows; row += gridDim.x) {
    float r[NV][8], y[NV][8], h[NV][8];
#pragma unroll
    for (int v = 0; v < NV; v++) {
      widen8<DT>(nr[v], r[v]);
      widen8<DT>(ny[v], y[v]);
    }
    fetch(row + gridDim.x);
    if (a.gate && row / a.per_sample != sample) {
      sample = row / a.per_sample;
      vector(a.gate, (int64_t)sample * a.width, gate);
    }
    float rstd1 = 1.0f;
    if (a.w1) {
      float s = 0;
#pragma unroll
      for (int v = 0; v < NV; v++)
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf(y[v][e], y[v][e], s);
      block_sum<W, 1>(&s, buf, turn++);
      rstd1 = 1.0f / sqrtf(s * inv_width + a.eps);
    }
    float s = 0;
#pragma unroll
    for (int v = 0; v < NV; v++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float z = y[v][e];
        if (a.w1) z = z * rstd1 * w1[v][e];
        if (a.gate) z *= gate[v][e];
        h[v][e] = fmaf(a.beta, r[v][e], a.alpha * z);
        s = fmaf(h[v][e], h[v][e], s);
      }
      if (left[v] > 0) E::store(hidden, (int64_t)row * a.width + c[v], left[v], h[v]);
    }
    float rstd2 = 1.0f;
    if (a.w2) {
      block_sum<W, 1>(&s, buf, turn++);
      rstd2 = 1.0f / sqrtf(s * inv_width + a.eps);
#pragma unroll
      for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int e = 0; e < 8; e++) h[v][e] *= rstd2 * w2[v][e];
        if (left[v] > 0) E::store(normed, (int64_t)row * a.width + c[v], left[v], h[v]);
      }
    }
    if (a.rstd && threadIdx.x == 0) {
      a.rstd[row] = rstd1;
      a.rstd[a.rows + row] = rstd2;
    }
  }
}

struct Grads {
  const void* dh;  // NULL: zero
  const void* dn;  // NULL: zero
  int64_t ld_dh, ld_dn;
  void* dr;        // each may be NULL
  void* dy;
  void* dw1;
  void* dgate;
  void* dw2;
  float* part;     // [3][units][width]: of w1, gate, w2
  int units;       // runs of rows, `slices` for each sample of the gate
  int slices;
};

// The rows of a unit, all of one sample.
__device__ inline void unit_rows(const Args& a, const Grads& g, int u, int* lo, int* hi) {
  const int sample = u / g.slices, slice = u - sample * g.slices;
  const int first = sample * a.per_sample;
  *lo = first + (int)((int64_t)a.per_sample * slice / g.slices);
  *hi = first + (int)((int64_t)a.per_sample * (slice + 1) / g.slices);
}

template <int DT, int W, int NV>
__global__ __launch_bounds__(W) void k_backward(Args a, Grads g) {
  using E = Elem<DT>;
  __shared__ float buf[2][16][3];
  int c[NV], left[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) {
    c[v] = (v * W + threadIdx.x) * 8;
    left[v] = a.width - c[v];
  }
  const float inv_width = 1.0f / a.width;
  float w1[NV][8], w2[NV][8], gate[NV][8];
  auto vector = [&](const void* p, int64_t at, float (*f)[8]) {
#pragma unroll
    for (int v = 0; v < NV; v++) {
      if (p) {
        widen8<DT>(left[v] > 0 ? E::load(p, at + c[v], left[v]) : typename E::Raw{}, f[v]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f[v][e] = 1.0f;
      }
    }
  };
  vector(a.w1, 0, w1);
  vector(a.w2, 0, w2);
  vector(a.gate, (int64_t)(blockIdx.x / g.slices) * a.width, gate);
  int row, end, turn = 0;
  unit_rows(a, g, blockIdx.x, &row, &end);
  float s1[NV][8] = {}, sg[NV][8] = {}, s2[NV][8] = {};
  typename E::Raw nr[NV] = {}, ny[NV] = {}, nh[NV] = {}, nn[NV] = {};
  auto fetch = [&](int k) {
    if (k >= end) return;
#pragma unroll
    for (int v = 0; v < NV; v++) {
      if (left[v] <= 0) continue;
      nr[v] = E::load(a.r, k * a.ld_r + c[v], left[v]);
      if (a.y) ny[v] = E::load(a.y, k * a.ld_y + c[v], left[v]);
      if (g.dh) nh[v] = E::load(g.dh, k * g.ld_dh + c[v], left[v]);
      if (g.dn) nn[v] = E::load(g.dn, k * g.ld_dn + c[v], left[v]);
    }
  };
  fetch(row);
  for (; row < end; row++) {
    float y[NV][8], dh[NV][8], dn[NV][8], h[NV][8];
#pragma unroll
    for (int v = 0; v < NV; v++) {
      widen8<DT>(nr[v], h[v]);
      widen8<DT>(ny[v], y[v]);
      widen8<DT>(nh[v], dh[v]);
      widen8<DT>(nn[v], dn[v]);
    }
    fetch(row + 1);
    const float rstd1 = a.rstd[row], rstd2 = a.rstd[a.rows + row];
    float sum[3] = {0, 0, 0};  // of t h, q (dh + rstd2 t), q h
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float q = a.alpha * gate[v][e] * w1[v][e] * y[v][e];
        h[v][e] = fmaf(a.beta, h[v][e], q * rstd1);
        const float t = w2[v][e] * dn[v][e];
        sum[0] = fmaf(t, h[v][e], sum[0]);
        sum[1] = fmaf(q, fmaf(rstd2, t, dh[v][e]), sum[1]);
        sum[2] = fmaf(q, h[v][e], sum[2]);
      }
    block_sum<W, 3>(sum, buf, turn++);
    const float mean2 = a.w2 ? sum[0] * rstd2 * inv_width : 0.0f;  // mean(t hhat)
    const float k2 = rstd2 * rstd2 * mean2;
    const float mean1 = (sum[1] - k2 * sum[2]) * rstd1 * inv_width;  // mean(w1 dz yhat)
#pragma unroll
    for (int v = 0; v < NV; v++) {
      float dr[8], dy[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float d = dh[v][e];
        if (a.w2) {
          d = fmaf(rstd2, w2[v][e] * dn[v][e], d) - k2 * h[v][e];
          s2[v][e] = fmaf(dn[v][e], h[v][e] * rstd2, s2[v][e]);
        }
        dr[e] = a.beta * d;
        const float yhat = y[v][e] * rstd1;
        sg[v][e] = fmaf(a.alpha * (yhat * w1[v][e]), d, sg[v][e]);
        const float dz = a.alpha * gate[v][e] * d;
        s1[v][e] = fmaf(dz, yhat, s1[v][e]);
        dy[e] = a.w1 ? rstd1 * (w1[v][e] * dz - yhat * mean1) : dz;
      }
      if (left[v] > 0) {
        const int64_t at = (int64_t)row * a.width + c[v];
        if (g.dr) E::store(g.dr, at, left[v], dr);
        if (g.dy) E::store(g.dy, at, left[v], dy);
      }
    }
  }
  const int64_t plane = (int64_t)g.units * a.width;
#pragma unroll
  for (int v = 0; v < NV; v++) {
    if (left[v] <= 0) continue;
    const int64_t at = (int64_t)blockIdx.x * a.width + c[v];
    if (g.dw1) Elem<DSX_F32>::store(g.part, at, left[v], s1[v]);
    if (g.dgate) {
      if (g.slices == 1)
        E::store(g.dgate, at, left[v], sg[v]);  // a unit is a whole sample
      else
        Elem<DSX_F32>::store(g.part, plane + at, left[v], sg[v]);
    }
    if (g.dw2) Elem<DSX_F32>::store(g.part, 2 * plane + at, left[v], s2[v]);
  }
}

// The partial rows of up to three vectors, added in order: for each, out[sample]
// [col] = the sum over that sample's rows. A block takes 32 columns; its eight
// runs of rows are added one after another.
struct Columns {
  const float* part[3];
  void* out[3];
  int count[3];    // partial rows per sample
  int samples[3];
  int n;
};
template <int DT>
__global__ __launch_bounds__(256) void k_columns(Columns t, int width) {
  __shared__ float run[8][32];
  int sample = blockIdx.y, v = 0;
  while (v + 1 < t.n && sample >= t.samples[v]) sample -= t.samples[v++];
  const int count = t.count[v], i = threadIdx.x & 31, q = threadIdx.x >> 5, c = blockIdx.x * 32 + i;
  const float* p = t.part[v] + (int64_t)sample * count * width + c;
  float s = 0;
  if (c < width) {
    const int hi = (int)((int64_t)count * (q + 1) / 8);
#pragma unroll 8
    for (int k = (int)((int64_t)count * q / 8); k < hi; k++) s += p[(int64_t)k * width];
  }
  run[q][i] = s;
  __syncthreads();
  if (q || c >= width) return;
  s = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) s += run[k][i];
  Elem<DT>::put(t.out[v], (int64_t)sample * width + c, s);
}

// ---- rows wider than 8192 ---------------------------------------------------

// h of one element, given rstd1.
template <int DT>
__device__ inline float hidden_at(const Args& a, int row, int c, float rstd1, float* q) {
  float z = a.y ? Elem<DT>::get(a.y, row * a.ld_y + c) : 0.0f;
  if (a.w1) z *= Elem<DT>::get(a.w1, c);
  if (a.gate) z *= Elem<DT>::get(a.gate, (int64_t)(row / a.per_sample) * a.width + c);
  z *= a.alpha;
  *q = z;
  return fmaf(a.beta, Elem<DT>::get(a.r, row * a.ld_r + c), z * rstd1);
}

template <int DT>
__global__ __launch_bounds__(1024) void k_wide_forward(Args a, void* __restrict__ hidden, void* __restrict__ normed) {
  __shared__ float buf[2][16][1];
  const int row = blockIdx.x;
  const float inv_width = 1.0f / a.width;
  float rstd1 = 1.0f, rstd2 = 1.0f, s = 0, q;
  if (a.w1) {
    for (int c = threadIdx.x; c < a.width; c += 1024) {
      const float y = Elem<DT>::get(a.y, row * a.ld_y + c);
      s = fmaf(y, y, s);
    }
    block_sum<1024, 1>(&s, buf, 0);
    rstd1 = 1.0f / sqrtf(s * inv_width + a.eps);
  }
  s = 0;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float h = hidden_at<DT>(a, row, c, rstd1, &q);
    s = fmaf(h, h, s);
    Elem<DT>::put(hidden, (int64_t)row * a.width + c, h);
  }
  if (a.w2) {
    block_sum<1024, 1>(&s, buf, 1);
    rstd2 = 1.0f / sqrtf(s * inv_width + a.eps);
    for (int c = threadIdx.x; c < a.width; c += 1024)
      Elem<DT>::put(normed, (int64_t)row * a.width + c,
                    hidden_at<DT>(a, row, c, rstd1, &q) * rstd2 * Elem<DT>::get(a.w2, c));
  }
  if (a.rstd && threadIdx.x == 0) {
    a.rstd[row] = rstd1;
    a.rstd[a.rows + row] = rstd2;
  }
}

// The two means of a row (of t hhat and of w1 dz yhat) into means[2][rows].
template <int DT>
__global__ __launch_bounds__(1024) void k_wide_means(Args a, Grads g, float* __restrict__ means) {
  __shared__ float buf[2][16][3];
  const int row = blockIdx.x;
  const float inv_width = 1.0f / a.width, rstd1 = a.rstd[row], rstd2 = a.rstd[a.rows + row];
  float sum[3] = {0, 0, 0};
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    float q;
    const float h = hidden_at<DT>(a, row, c, rstd1, &q);
    const float t = g.dn ? Elem<DT>::get(a.w2, c) * Elem<DT>::get(g.dn, row * g.ld_dn + c) : 0.0f;
    const float dh = g.dh ? Elem<DT>::get(g.dh, row * g.ld_dh + c) : 0.0f;
    sum[0] = fmaf(t, h, sum[0]);
    sum[1] = fmaf(q, fmaf(rstd2, t, dh), sum[1]);
    sum[2] = fmaf(q, h, sum[2]);
  }
  block_sum<1024, 3>(sum, buf, 0);
  if (threadIdx.x == 0) {
    const float mean2 = a.w2 ? sum[0] * rstd2 * inv_width : 0.0f;
    means[row] = mean2;
    means[a.rows + row] = (sum[1] - rstd2 * rstd2 * mean2 * sum[2]) * rstd1 * inv_width;
  }
}

// The gradients of 256 columns over a unit's rows.
template <int DT>
__global__ __launch_bounds__(256) void k_wide_backward(Args a, Grads g, const float* __restrict__ means) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  int row, end;
  unit_rows(a, g, blockIdx.y, &row, &end);
  const float w1 = a.w1 ? Elem<DT>::get(a.w1, c) : 1.0f, w2 = a.w2 ? Elem<DT>::get(a.w2, c) : 1.0f;
  const float gate = a.gate ? Elem<DT>::get(a.gate, (int64_t)(blockIdx.y / g.slices) * a.width + c) : 1.0f;
  float s1 = 0, sg = 0, s2 = 0;
  for (; row < end; row++) {
    const float rstd1 = a.rstd[row], rstd2 = a.rstd[a.rows + row];
    float q;
    const float h = hidden_at<DT>(a, row, c, rstd1, &q);
    const float yhat = (a.y ? Elem<DT>::get(a.y, row * a.ld_y + c) : 0.0f) * rstd1;
    const float dn = g.dn ? Elem<DT>::get(g.dn, row * g.ld_dn + c) : 0.0f;
    float d = g.dh ? Elem<DT>::get(g.dh, row * g.ld_dh + c) : 0.0f;
    if (a.w2) {
      d = fmaf(rstd2, w2 * dn, d) - rstd2 * rstd2 * means[row] * h;
      s2 = fmaf(dn, h * rstd2, s2);
    }
    sg = fmaf(a.alpha * (yhat * w1), d, sg);
    const float dz = a.alpha * gate * d;
    s1 = fmaf(dz, yhat, s1);
    const int64_t at = (int64_t)row * a.width + c;
    if (g.dr) Elem<DT>::put(g.dr, at, a.beta * d);
    if (g.dy) Elem<DT>::put(g.dy, at, a.w1 ? rstd1 * (w1 * dz - yhat * means[a.rows + row]) : dz);
  }
  const int64_t plane = (int64_t)g.units * a.width, at = (int64_t)blockIdx.y * a.width + c;
  if (g.dw1) g.part[at] = s1;
  if (g.dgate) {
    if (g.slices == 1)
      Elem<DT>::put(g.dgate, at, sg);
    else
      g.part[plane + at] = sg;
  }
  if (g.dw2) g.part[2 * plane + at] = s2;
}

// ---- host ------------------------------------------------------------------

int block_of(int64_t width) {
  int w = 64;
  while (w < 512 && w * 8 < width) w *= 2;
  return w;
}

// Runs of rows for the backward: enough blocks for eight waves a CU, but four
// rows a run at least, since every run costs a row of partial sums for each of
// up to three vectors. (8192 rows of 4096, bf16, forward and backward: 152 us;
// with two, four and eight times as many blocks 157, 170 and 198.)
int slices_of(int64_t rows, int64_t samples, int64_t width) {
  const int64_t per = rows / samples, target = 256 * 512 / block_of(width);
  int64_t s = ceil_div(target, samples);
  if (s > per / 4) s = per / 4;
  return (int)(s < 1 ? 1 : s);
}

int64_t samples_of(const DsxNorm& q) { return q.gate && q.gate_rows > 1 ? q.gate_rows : 1; }

int64_t workspace_of(const DsxNorm& q) {
  if (!q.rows) return 256;
  const int64_t samples = samples_of(q);
  const int64_t units = samples * slices_of(q.rows, samples, q.width);
  return round_up(3 * units * q.width * 4, 256) + round_up(2 * q.rows * 4, 256);
}

Args args_of(const DsxNorm& q) {
  Args a{};
  a.r = q.residual;
  a.y = q.branch;
  a.w1 = q.post_weight;
  a.gate = q.gate;
  a.w2 = q.next_weight;
  a.ld_r = q.ld_residual;
  a.ld_y = q.ld_branch;
  a.rows = (int)q.rows;
  a.width = (int)q.width;
  a.per_sample = (int)(q.rows / samples_of(q));
  a.alpha = q.branch_scale;
  a.beta = q.residual_scale;
  a.eps = q.eps;
  a.rstd = q.rstd;
  return a;
}

template <int DT>
void forward(const Args& a, void* hidden, void* normed, hipStream_t s) {
  if (a.width > kWidest) {
    k_wide_forward<DT><<<a.rows, 1024, 0, s>>>(a, hidden, normed);
    return;
  }
  const int w = block_of(a.width);
  // enough blocks for every wave slot; each walks every grid-th row
  const int64_t most = (int64_t)256 * (2048 / w);
  const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
  switch (w) {
    case 64: k_forward<DT, 64, 1><<<grid, 64, 0, s>>>(a, hidden, normed); break;
    case 128: k_forward<DT, 128, 1><<<grid, 128, 0, s>>>(a, hidden, normed); break;
    case 256: k_forward<DT, 256, 1><<<grid, 256, 0, s>>>(a, hidden, normed); break;
    default:
      if (a.width <= 4096) k_forward<DT, 512, 1><<<grid, 512, 0, s>>>(a, hidden, normed);
      else k_forward<DT, 512, 2><<<grid, 512, 0, s>>>(a, hidden, normed);
  }
}

template <int DT>
void backward(const Args& a, Grads g, float* means, int samples, hipStream_t s) {
  if (a.width > kWidest) {
    k_wide_means<DT><<<a.rows, 1024, 0, s>>>(a, g, means);
    k_wide_backward<DT><<<dim3((unsigned)ceil_div(a.width, 256), (unsigned)g.units), 256, 0, s>>>(a, g, means);
  } else {
    const unsigned grid = (unsigned)g.units;
    switch (block_of(a.width)) {
      case 64: k_backward<DT, 64, 1><<<grid, 64, 0, s>>>(a, g); break;
      case 128: k_backward<DT, 128, 1><<<grid, 128, 0, s>>>(a, g); break;
      case 256: k_backward<DT, 256, 1><<<grid, 256, 0, s>>>(a, g); break;
      default:
        if (a.width <= 4096) k_backward<DT, 512, 1><<<grid, 512, 0, s>>>(a, g);
        else k_backward<DT, 512, 2><<<grid, 512, 0, s>>>(a, g);
    }
  }
  const int64_t plane = (int64_t)g.units * a.width;
  Columns t{};
  int total = 0;
  auto add = [&](void* out, int which, int count, int n) {
    t.part[t.n] = g.part + which * plane;
    t.out[t.n] = out;
    t.count[t.n] = count;
    t.samples[t.n++] = n;
    total += n;
  };
  if (g.dw1) add(g.dw1, 0, g.units, 1);
  if (g.dw2) add(g.dw2, 2, g.units, 1);
  if (g.dgate && g.slices > 1) add(g.dgate, 1, g.slices, samples);
  if (t.n) k_columns<DT><<<dim3((unsigned)ceil_div(a.width, 32), (unsigned)total), 256, 0, s>>>(t, a.width);
}

bool off(const void* p, int dtype) { return p && ((uintptr_t)p & (dtype == DSX_F32 ? 3 : 1)); }

int check(const char* what, const DsxNorm* q) {
  if (!q) return fail(DSX_EINVAL, "%s: the argument block is NULL", what);
  if (q->dtype != DSX_F32 && !dsxi::is16(q->dtype)) return fail(DSX_EINVAL, "%s: bad dtype %d", what, q->dtype);
  if (q->rows < 0 || q->rows > DSX_NORM_MAX_ROWS || q->width < 1 || q->width > DSX_MATRIX_MAX_DIM)
    return fail(DSX_EINVAL, "%s: rows in [0, %d], width in [1, %d]", what, DSX_NORM_MAX_ROWS, DSX_MATRIX_MAX_DIM);
  if (q->rows && !q->branch && (q->post_weight || q->gate))
    return fail(DSX_EINVAL, "%s: a weight or gate of a branch that is NULL", what);
  if (q->gate && (q->gate_rows < 1 || q->gate_rows > 65533 || (q->rows && q->rows % q->gate_rows)))
    return fail(DSX_EINVAL, "%s: gate_rows must divide rows and lie in [1, 65533]", what);
  if (!(q->eps >= 0.0f)) return fail(DSX_EINVAL, "%s: eps must be >= 0", what);
  return DSX_OK;
}

int check_device(const char* what, const DsxNorm* q) {
  if (!q->residual) return fail(DSX_EINVAL, "%s: residual is NULL", what);
  if (off(q->residual, q->dtype) || off(q->branch, q->dtype) || off(q->post_weight, q->dtype) ||
      off(q->gate, q->dtype) || off(q->next_weight, q->dtype) || off(q->rstd, DSX_F32))
    return fail(DSX_EINVAL, "%s: misaligned pointer", what);
  if (q->ld_residual < q->width || (q->branch && q->ld_branch < q->width))
    return fail(DSX_EINVAL, "%s: a row stride is below the row's length", what);
  return DSX_OK;
}

}  // namespace

extern "C" {

int64_t dsx_norm_workspace_bytes(const DsxNorm* args) {
  if (check("dsx_norm_workspace_bytes", args)) return -1;
  return workspace_of(*args);
}

int dsx_norm_forward(const DsxNorm* args, void* hidden, void* normed, void* stream) {
  const char* what = "dsx_norm_forward";
  if (int rc = check(what, args)) return rc;
  if (!args->rows) return DSX_OK;
  if (int rc = check_device(what, args)) return rc;
  if (!hidden || off(hidden, args->dtype) || (args->next_weight && !normed) || off(normed, args->dtype))
    return fail(DSX_EINVAL, "%s: NULL or misaligned output", what);
  const Args a = args_of(*args);
  hipStream_t s = as_stream(stream);
  if (args->dtype == DSX_F32) forward<DSX_F32>(a, hidden, normed, s);
  else if (args->dtype == DSX_F16) forward<DSX_F16>(a, hidden, normed, s);
  else forward<DSX_BF16>(a, hidden, normed, s);
  return launch_status(what);
}

int dsx_norm_backward(const DsxNorm* args, const void* d_hidden, int64_t ld_dh, const void* d_normed, int64_t ld_dn,
                      void* d_residual, void* d_branch, void* d_post_weight, void* d_gate, void* d_next_weight,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "dsx_norm_backward";
  if (int rc = check(what, args)) return rc;
  if (!args->rows) return DSX_OK;
  if (int rc = check_device(what, args)) return rc;
  const int dt = args->dtype;
  if (!args->rstd) return fail(DSX_EINVAL, "%s: rstd is NULL", what);
  if ((d_branch && !args->branch) || (d_post_weight && !args->post_weight) || (d_gate && !args->gate) ||
      (d_next_weight && !args->next_weight) || (d_normed && !args->next_weight))
    return fail(DSX_EINVAL, "%s: a gradient of an input that is NULL", what);
  if (off(d_hidden, dt) || off(d_normed, dt) || off(d_residual, dt) || off(d_branch, dt) || off(d_post_weight, dt) ||
      off(d_gate, dt) || off(d_next_weight, dt))
    return fail(DSX_EINVAL, "%s: misaligned gradient", what);
  if ((d_hidden && ld_dh < args->width) || (d_normed && ld_dn < args->width))
    return fail(DSX_EINVAL, "%s: a row stride is below the row's length", what);
  if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < workspace_of(*args))
    return fail(DSX_EINVAL, "%s: the workspace must be 256-byte aligned and of %lld bytes", what,
                (long long)workspace_of(*args));
  const Args a = args_of(*args);
  const int samples = (int)samples_of(*args);
  Grads g{};
  g.dh = d_hidden;
  g.dn = d_normed;
  g.ld_dh = ld_dh;
  g.ld_dn = ld_dn;
  g.dr = d_residual;
  g.dy = d_branch;
  g.dw1 = d_post_weight;
  g.dgate = d_gate;
  g.dw2 = d_next_weight;
  g.slices = slices_of(args->rows, samples, args->width);
  g.units = samples * g.slices;
  g.part = (float*)workspace;
  float* means = (float*)((char*)workspace + round_up((int64_t)3 * g.units * a.width * 4, 256));
  hipStream_t s = as_stream(stream);
  if (dt == DSX_F32) backward<DSX_F32>(a, g, means, samples, s);
  else if (dt == DSX_F16) backward<DSX_F16>(a, g, means, samples, s);
  else backward<DSX_BF16>(a, g, means, samples, s);
  return launch_status(what);
}

}  // extern "C"
