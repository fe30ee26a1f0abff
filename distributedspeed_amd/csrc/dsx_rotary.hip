// dsx_rotary.hip -- the rotation of query and key heads by their positions
// (see include/dsx.h).
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position base^(-2 i / dims)
//
// for pair i of a head; the gradient is the rotation by -t. Every byte is read
// and written once. The angles of a row are the same for all its heads: a
// block computes those of a few rows, keeps them in shared memory and turns all
// heads of these rows. An angle is formed in fp64, as a part of a turn, and
// only what is left of whole turns goes to fp32: at position 131071 fp32 would
// be off by 0.004 of a radian before the rotation begins.
//
// Bound by memory: 8192 rows of 32 and 8 heads of 128, bf16, on their own 36 us,
// 4.6 TB/s, where a copy of 2 GiB runs at 4.86; 29 us where the 84 MB are still in
// the last cache.

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

struct Part {  // [tokens][heads][d], d contiguous
  const void* from;
  void* to;
  int64_t ld, head;
  int heads;
};
struct Args {
  Part part[2];
  const void* positions;
  int tokens, d, half, wide;  // wide: positions in 64 bits
  int per;                    // rows of a block
  double step;                // log2 of the ratio of neighbouring frequencies
  float sign;
};

template <int DT>
struct Elem {
  using T = typename std::conditional<DT == DSX_F16, F16, BF16>::type;
  typedef short Stored;
  static __device__ inline void load(const Stored* p, int n, float* v) {
    if (n >= 8) {
      const s8v w = *(const s8u*)p;
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = T::widen(w[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = e < n ? T::widen(p[e]) : 0.0f;
    }
  }
  static __device__ inline void store(Stored* p, int n, const float* v) {
    s8v w;
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = T::round(v[e]);
    if (n >= 8) {
      *(s8u*)p = w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < n) p[e] = w[e];
    }
  }
};
template <>
struct Elem<DSX_F32> {
  typedef float Stored;
  static __device__ inline void load(const float* p, int n, float* v) {
    if (n >= 8) {
      const f4v a = *(const f4u*)p, b = *(const f4u*)(p + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[e] = a[e];
        v[e + 4] = b[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = e < n ? p[e] : 0.0f;
    }
  }
  static __device__ inline void store(float* p, int n, const float* v) {
    if (n >= 8) {
      *(f4u*)p = f4v{v[0], v[1], v[2], v[3]};
      *(f4u*)(p + 4) = f4v{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < n) p[e] = v[e];
    }
  }
};

constexpr int kThreads = 256;
constexpr int kPairs = 512;  // of a block's rows
constexpr int64_t kMostBlocks = 1 << 22;  // a launch's threads are counted in 32 bits

// A thread takes eight pairs, or eight of the features that are not turned.
template <int DT, bool SIDE>
__global__ __launch_bounds__(kThreads) void k_rotary(Args a) {
  using E = Elem<DT>;
  using S = typename E::Stored;
  __shared__ float2 turn[kPairs];
  for (int64_t first = (int64_t)blockIdx.x * a.per; first < a.tokens; first += (int64_t)gridDim.x * a.per) {
    const int t0 = (int)first, rows = min(a.per, a.tokens - t0);
    for (int i = threadIdx.x; i < rows * a.half; i += kThreads) {
      const int r = i / a.half, p = i - r * a.half;
      const double at = a.wide ? (double)((const int64_t*)a.positions)[t0 + r] : (double)((const int32_t*)a.positions)[t0 + r];
      double x = at * (exp2(p * a.step) * 0.15915494309189533577);  // turns
      x -= rint(x);
      float s, c;
      sincospif(2.0f * (float)x, &s, &c);
      turn[i] = {c, s * a.sign};
    }
    __syncthreads();
    const int pairs = (a.half + 7) / 8, rest = a.d - 2 * a.half, per_head = pairs + (rest + 7) / 8;
    const int heads = a.part[0].heads + a.part[1].heads;
    const int n = rows * heads * per_head;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int row = i / per_head, c = i - row * per_head;
      const int r = row / heads;
      int h = row - r * heads;
      const bool second = h >= a.part[0].heads;
      const Part& q = a.part[second];
      h -= second ? a.part[0].heads : 0;
      const S* from = (const S*)q.from + (t0 + r) * q.ld + h * q.head;
      S* to = (S*)q.to + ((int64_t)(t0 + r) * q.heads + h) * a.d;
      float x[8], y[8];
      if (c >= pairs) {
        const int f = 2 * a.half + (c - pairs) * 8;
        E::load(from + f, a.d - f, x);
        E::store(to + f, a.d - f, x);
        continue;
      }
      const int p = c * 8, left = a.half - p;
      float v[16];
      if (SIDE) {
        E::load(from + 2 * p, 2 * left, v);
        E::load(from + 2 * p + 8, 2 * left - 8, v + 8);
  #pragma unroll
        for (int e = 0; e < 8; e++) {
          x[e] = v[2 * e];
          y[e] = v[2 * e + 1];
        }
      } else {
        E::load(from + p, left, x);
        E::load(from + a.half + p, left, y);
      }
  #pragma unroll
      for (int e = 0; e < 8; e++) {
        const float2 w = e < left ? turn[r * a.half + p + e] : float2{1, 0};
        const float s = x[e];
        x[e] = fmaf(s, w.x, -y[e] * w.y);
        y[e] = fmaf(y[e], w.x, s * w.y);
      }
      if (SIDE) {
  #pragma unroll
        for (int e = 0; e < 8; e++) {
          v[2 * e] = x[e];
          v[2 * e + 1] = y[e];
        }
        E::store(to + 2 * p, 2 * left, v);
        E::store(to + 2 * p + 8, 2 * left - 8, v + 8);
      } else {
        E::store(to + p, left, x);
        E::store(to + a.half + p, left, y);
      }
    }
    __syncthreads();
  }
}

template <int DT>
void launch(const Args& a, bool side, hipStream_t s) {
  const int64_t blocks = ceil_div(a.tokens, a.per);
  const dim3 grid((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks));
  if (side) k_rotary<DT, true><<<grid, kThreads, 0, s>>>(a);
  else k_rotary<DT, false><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

extern "C" int dsx_rotary(const DsxRotary* q, void* q_out, void* k_out, int32_t inverse, void* stream) {
  const char* what = "dsx_rotary";
  if (!q) return fail(DSX_EINVAL, "%s: the argument block is NULL", what);
  if (q->dtype != DSX_F32 && !dsxi::is16(q->dtype)) return fail(DSX_EINVAL, "%s: bad dtype %d", what, q->dtype);
  if (q->tokens < 0 || q->tokens > DSX_ATTENTION_MAX_TOKENS)
    return fail(DSX_EINVAL, "%s: tokens in [0, %d]", what, DSX_ATTENTION_MAX_TOKENS);
  if (q->heads < 1 || q->heads > DSX_ATTENTION_MAX_HEADS || q->kv_heads < 0 || q->kv_heads > DSX_ATTENTION_MAX_HEADS)
    return fail(DSX_EINVAL, "%s: heads in [1, %d], kv_heads in [0, %d]", what, DSX_ATTENTION_MAX_HEADS,
                DSX_ATTENTION_MAX_HEADS);
  if (q->head_dim < 1 || q->head_dim > 2 * kPairs || q->dims < 0 || q->dims > q->head_dim || q->dims % 2)
    return fail(DSX_EINVAL, "%s: head_dim in [1, %d], dims even and at most head_dim", what, 2 * kPairs);
  if (!(q->base > 0.0) || !(q->base < INFINITY)) return fail(DSX_EINVAL, "%s: base must be positive and finite", what);
  if (q->position_bytes != 4 && q->position_bytes != 8)
    return fail(DSX_EINVAL, "%s: positions are of 4 or 8 bytes", what);
  if (!q->tokens) return DSX_OK;
  const uintptr_t mask = q->dtype == DSX_F32 ? 3 : 1;
  const bool two = q->kv_heads > 0;
  if (!q->q || !q_out || (two && (!q->k || !k_out)) || !q->positions)
    return fail(DSX_EINVAL, "%s: NULL pointer", what);
  if ((((uintptr_t)q->q | (uintptr_t)q_out | (two ? (uintptr_t)q->k | (uintptr_t)k_out : 0)) & mask) ||
      ((uintptr_t)q->positions & (q->position_bytes - 1)))
    return fail(DSX_EINVAL, "%s: misaligned pointer", what);
  Args a{};
  a.part[0] = {q->q, q_out, q->ld_q, q->head_q, q->heads};
  a.part[1] = {q->k, k_out, q->ld_k, q->head_k, q->kv_heads};
  a.positions = q->positions;
  a.wide = q->position_bytes == 8;
  a.tokens = (int)q->tokens;
  a.d = q->head_dim;
  a.half = q->dims / 2;
  a.step = q->dims ? -2.0 * log2(q->base) / q->dims : 0.0;
  a.sign = inverse ? -1.0f : 1.0f;
  // Rows of a block: an angle a thread. (8192 rows, bf16: 32 and 8 heads of 128, four
  // rows, 29.0 us, with one 30.2, with eight 29.4; 12 and 12 of 64, eight, 11.9, with
  // one 18.0, with two 13.9.)
  a.per = a.half ? kThreads / a.half : 8;
  a.per = a.per < 1 ? 1 : a.per > 8 ? 8 : a.per;
  hipStream_t s = as_stream(stream);
  const bool side = q->interleaved != 0;
  if (q->dtype == DSX_F32) launch<DSX_F32>(a, side, s);
  else if (q->dtype == DSX_F16) launch<DSX_F16>(a, side, s);
  else launch<DSX_BF16>(a, side, s);
  return launch_status(what);
}
