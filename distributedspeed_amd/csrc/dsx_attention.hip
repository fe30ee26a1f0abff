// dsx_attention.hip -- attention over packed sequences and its gradients (see
// include/dsx.h).
//
//   s_ij = q_i k_j,  P_ij = exp(scale s_ij - lse_i),  o_i = sum_j P_ij v_j
//   dP_ij = do_i v_j,  dS_ij = P_ij (dP_ij - delta_i),  delta_i = do_i o_i
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij do_i
//
// over the pairs (i, j) of one sequence (causal: j <= i); heads of a group
// share k and v, whose gradients are summed over them.
//
// All three kernels are one pass: a wave keeps 32 rows of its own (queries in
// k_attend and k_query_grads, keys in k_key_grads) and the other side comes by
// in tiles of 64 rows through shared memory, two of them there at a time. The
// products run on the 32x32x16 matrix instruction with the wave's own rows as
// its columns: a lane then holds one row's values of 16 rows of the other
// side, so that a row's maximum and sum are one exchange between two lanes,
// and the registers of P and dS, rounded, are the second operand of the next
// product as they lie: its sum runs over the rows in the order in which the
// first one left them, and the transposing LDS read brings the first operand
// in the same order.
//
// The gradients come from two kernels that compute P twice rather than from
// one that adds up dq across blocks: nothing is added by atomics, so that
// results do not depend on timing.
//
// What bounds them: a matrix instruction of 32x32x16 takes 32 clocks of a SIMD's
// unit and wants a fragment of 1 KB, eight clocks of the LDS that four SIMDs share:
// both are busy alike, so that what the vector unit and the loads take beside them
// shows in part. k_attend, 4096 causal rows, 32 heads (8 of keys) of 128, bf16: 152
// us, 0.91 PFLOP/s of the visible pairs' products (a large product reaches 1.42);
// without the softmax's arithmetic 139, without the loads 151, without both 126.
// With 64 features there is twice the softmax for a product: 16384 rows, 16 heads
// (2), k_attend 0.60 to 0.64 ms, 0.89 PFLOP/s; k_query_grads 0.90 to 0.95 ms, 0.92
// (pack_rest's products not counted); k_key_grads 1.05 to 1.11 ms, 1.02. Waves of 64
// rows would halve the LDS reads: with 128 features their registers leave one wave a
// SIMD, which was slower; with 64 they would leave two, which has not been tried.
// Computing the next tile's scores beside a tile's softmax was slower.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <new>

#include "dsx.h"
#include "dsx_gemm.h"
#include "dsx_internal.h"

namespace {

using dsxg::b8v;
using dsxg::h8v;
using dsxg::kCus;
using dsxg::LdsBlock;
using dsxg::read_transposed;
using dsxg::s4v;
using dsxg::s8v;
using dsxi::as_stream;
using dsxi::ceil_div;
using dsxi::fail;
using dsxi::launch_status;
using dsxi::round_up;

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s2v __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));

// kBias: P is held as exp2(s - m + kBias). fp16's 2^-14 would lose the small
// values of long rows; with the running maximum up to kLazy behind (below),
// 2^(kBias + kLazy) = 2^15 is still in its range.
struct F16 : dsxg::F16 {
  static constexpr float kBias = 7.0f;
  static constexpr bool kScaled = true;
  static __device__ inline f16v mfma(s8v a, s8v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  }
};
struct BF16 : dsxg::BF16 {
  static constexpr float kBias = 0.0f;
  static constexpr bool kScaled = false;
  static __device__ inline f16v mfma(s8v a, s8v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  }
};
constexpr float kLazy = 8.0f;

constexpr int kRows = 128;   // of a block: four waves of 32
constexpr int kTile = 64;    // rows of the other side in shared memory
constexpr int kThreads = 256;

struct Rows {  // [tokens][heads][d], d contiguous
  const short* p;
  int64_t ld, head;  // strides in elements
};
struct Args {
  Rows q, k, v;
  const int4* tiles;  // first row, first and end row of its sequence
  int heads, kv_heads, group, d;
  int tokens, causal;
  float scale, scale2;  // scale2: scale log2(e)
};

// ---- tiles in shared memory --------------------------------------------------

// Of D features, a multiple of 32, in rows of HD, a power of two.
template <int D>
struct Tile {
  static constexpr int HD = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  static constexpr int kChunks = HD / 8;               // of 16 bytes, in a row
  static constexpr int kBytes = kTile * HD * 2;
  static constexpr int kLoads = kTile * kChunks / kThreads;
  static constexpr int kSteps = D / 16;                // matrix instructions along a row
  static constexpr int kBlocks = D / 32;               // of 32 features

  // Chunk c of row r lies at c ^ swizzle(r): the 16 rows of a fragment read, and
  // the 4 x 32 bytes that 16 lanes of a transposing read touch, then fall on
  // different banks (64 of 4 bytes).
  static __device__ inline int swizzle(int r) {
    return HD == 64 ? ((r >> 1) & 3) << 1 | ((r >> 3) & 1) : (r & 7) << 1 | ((r >> 3) & 1);
  }

  // Loads rows [0, left) of 64 straight to shared memory; a row past the end is
  // the last one again and a chunk past d the row's first (the products' other
  // operand holds zeros there).
  static __device__ inline void load(char* dst, const short* p, int64_t ld, int left, int d) {
    const int tid = threadIdx.x & (kThreads - 1), w = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const int at = j * kThreads + tid, r = at / kChunks;
      int c = (at % kChunks) ^ swizzle(r);
      c = c * 8 < d ? c : 0;
      const uint32_t off = (uint32_t)min(r, left - 1) * (uint32_t)(ld * 2) + c * 16;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)p + off),
                                       (__attribute__((address_space(3))) void*)(dst + j * kThreads * 16 + w * 1024), 16,
                                       0, 0);
    }
  }
  // Rows r0..r0+31 (r0 a multiple of 32), features 16 step..: one row a lane.
  static __device__ inline s8v rows(const char* tile, int r0, int step, int lane) {
    const int r = r0 + (lane & 31);
    return *(const s8v*)(tile + r * HD * 2 + (((step * 2 + (lane >> 5)) ^ swizzle(lane & 31)) << 4));
  }
  // Features f0..f0+31 (one a lane) of the 16 rows from r0: rows 4h..4h+3 and
  // 8+4h..8+4h+3 for the lane's half h.
  static __device__ inline s8v columns(const char* tile, int r0, int f0, int lane) {
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int c = f0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const char* row = tile + (r0 + r) * HD * 2 + (lane & 1) * 8;
    const s4v lo = read_transposed((LdsBlock*)(row + ((c ^ swizzle(r0 + r)) << 4)));
    const s4v hi = read_transposed((LdsBlock*)(row + 8 * HD * 2 + ((c ^ swizzle(r0 + r + 8)) << 4)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // The wave's own 32 rows as an operand in registers; zeros past d.
  static __device__ inline void own(s8v* f, const short* p, int64_t ld, int row, int d, int lane) {
    const short* at = p + row * ld;
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      const int c = (s * 2 + (lane >> 5)) * 8;
      f[s] = c < d ? *(const s8v*)(at + c) : s8v{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  // Their arrival is waited for here: left to their first use, inside a loop, the
  // wait would be for the tiles on their way as well, in every round.
  static __device__ inline void arrived(s8v* f) {
#pragma unroll
    for (int s = 0; s < kSteps; s++) asm volatile("" : "+v"(f[s]));
  }
};

// The same reads with three registers of addresses, for a kernel that has none
// to spare: the places of a row's chunks differ by an exclusive or. Two tiles,
// kBytes apart.
typedef __attribute__((address_space(3))) s8v LdsChunk;
__device__ inline s8v read_chunk(LdsChunk* __restrict__ p) { return *p; }
template <int D>
struct Reader {
  using L = Tile<D>;
  static constexpr int HD = L::HD;
  uint32_t row, lo, hi;
  __device__ inline void init(const char* lds, int lane) {
    const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
    const int r = lane & 31, half = lane >> 5;
    row = base + r * HD * 2 + ((half ^ L::swizzle(r)) << 4);
    const int k = 4 * half + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    lo = base + k * HD * 2 + ((c ^ L::swizzle(k)) << 4) + (lane & 1) * 8;
    hi = base + (k + 8) * HD * 2 + ((c ^ L::swizzle(k + 8)) << 4) + (lane & 1) * 8;
  }
  // For the rows from `at` bytes on.
  __device__ inline Reader from(int at) const {
    Reader r{row + at, lo + at, hi + at};
    asm volatile("" : "+v"(r.row), "+v"(r.lo), "+v"(r.hi));
    return r;
  }
  template <int TILE>
  __device__ inline s8v rows(int step) const {
    return read_chunk((LdsChunk*)(uintptr_t)((row ^ (step << 5)) + TILE * L::kBytes));
  }
  template <int TILE>
  __device__ inline s8v columns(int r0, int i) const {
    const uint32_t at = TILE * L::kBytes + r0 * HD * 2;
    const s4v x = read_transposed((LdsBlock*)(uintptr_t)((lo ^ (i << 6)) + at)), y = read_transposed((LdsBlock*)(uintptr_t)((hi ^ (i << 6)) + at));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Waits for this wave's direct loads and LDS reads, then for the other waves.
__device__ inline void sync_loads() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Values of 16 rows by 32 columns as the second operand of the next product.
template <class T>
__device__ inline s8v pack(const f16v& v, int half) {
  s8v r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = T::round(v[half * 8 + e]);
  return r;
}
// What pack lost of them, in the same type.
template <class T>
__device__ inline s8v pack_rest(const f16v& v, int half, const s8v& packed) {
  s8v r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = T::round(v[half * 8 + e] - T::widen(packed[e]));
  return r;
}
__device__ inline float other_half(float v) { return __shfl_xor(v, 32); }

// The row (of 32) that register r of a lane's half holds.
__device__ constexpr int row_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// Writes a wave's 32 rows of o (one a lane, features as row_of has them) by way
// of its part of shared memory. `rest`: what rounding to 16 bits loses instead.
template <class T, int D>
__device__ inline void store_rows(char* strip, const f16v* o, float factor, bool rest, short* out, int64_t ld,
                                  int rows, int d, int lane) {
  using L = Tile<D>;
  constexpr int HD = L::HD;
  const int r = lane & 31, half = lane >> 5;
#pragma unroll
  for (int i = 0; i < L::kBlocks; i++)
#pragma unroll
    for (int c = 0; c < 4; c++) {
      s4v w;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float v = o[i][c * 4 + e] * factor;
        w[e] = T::round(v);
        if (rest) {
          const float back = T::widen(w[e]);
          w[e] = T::round(__builtin_isfinite(back) ? v - back : 0.0f);
        }
      }
      *(s4v*)(strip + r * HD * 2 + (((i * 4 + c) ^ L::swizzle(r)) << 4) + half * 8) = w;
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int at = 0; at < 32 * L::kChunks; at += 64) {
    const int row = (at + lane) / L::kChunks, c = (at + lane) % L::kChunks;
    if (row < rows && c * 8 < d) *(s8v*)(out + row * ld + c * 8) = *(const s8v*)(strip + row * HD * 2 + ((c ^ L::swizzle(row)) << 4));
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A block's tile and heads: tile by tile in the table's order (of causal calls: the
// most work first), the heads of a key head eight blocks apart so that one XCD's L2
// serves them.
struct Place {
  int row0, start, end, head, kv;
  bool good;
};
__device__ inline Place place_of(const Args& a, int heads) {
  const int t = blockIdx.x / heads, h = blockIdx.x % heads;
  const int4 e = a.tiles[t];
  Place p{e.x, e.y, e.z, 0, 0, false};
  const int per = heads / a.kv_heads;
  p.kv = h % a.kv_heads;
  p.head = p.kv * per + h / a.kv_heads;
  p.good = p.start >= 0 && p.start <= p.row0 && p.row0 < p.end && p.end <= a.tokens;
  return p;
}

// A SIMD's waves: as many as the registers of a kernel of D features allow; of a
// block of eight, two or four. (16384
// rows, 16 heads of 64: k_attend with four 625 us, with three 635; both gradients
// with three 2.08 ms, with two 2.14.)
constexpr int dsx_waves(int d, int at_64, int groups) {
  return groups == 2 && at_64 == 3 ? 2 : d <= 32 ? 4 : d <= 64 ? at_64 : d <= 128 ? 2 : 1;
}
#define DSX_ATTENTION_KERNEL(D, WAVES, GROUPS)              \
  __launch_bounds__(kThreads * GROUPS) __attribute__((       \
      amdgpu_waves_per_eu(dsx_waves(D, WAVES, GROUPS), dsx_waves(D, WAVES, GROUPS))))

// v, as the compiler may not know it before this place: keeps what the masks of
// the few tiles at a sequence's edges need out of every tile's way.
__device__ inline int only_here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// N matrix instructions with READS LDS reads each: AHEAD instructions' reads are
// on their way before the first.
template <int N, int READS, int AHEAD>
__device__ inline void feed() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; i++) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// ---- forward -------------------------------------------------------------------

struct Forward {
  short* out;     // [tokens][heads][d]
  short* out_lo;  // what out lost in rounding, for delta (k_delta); NULL: not kept
  float* lse;     // [heads][tokens], base 2; NULL: not kept
};

// Two groups of four waves share a block's rows where there are few blocks: a
// group takes every other tile, and the second hands its sums to the first.
template <int D>
__device__ inline void hand_over(float* to, const f16v* o) {
#pragma unroll
  for (int i = 0; i < D / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) to[(i * 16 + r) * 64] = o[i][r];
}
template <int D>
__device__ inline void take_over(const float* from, f16v* o, float mine, float theirs) {
#pragma unroll
  for (int i = 0; i < D / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[i][r] = o[i][r] * mine + from[(i * 16 + r) * 64] * theirs;
}

template <class T, int D, int GROUPS>
__global__ DSX_ATTENTION_KERNEL(D, 4, GROUPS) void k_attend(Args a, Forward f) {
  using L = Tile<D>;
  constexpr int HD = L::HD;
  __shared__ __attribute__((aligned(1024))) char shared[GROUPS][2][2][L::kBytes];
  const Place p = place_of(a, a.heads);
  if (!p.good) return;
  const int lane = threadIdx.x & 63, half = lane >> 5, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  auto& lds = shared[group];
  const int w0 = p.row0 + 32 * w, row = w0 + (lane & 31);
  s8v qf[L::kSteps];
  L::own(qf, a.q.p + p.head * a.q.head, a.q.ld, min(row, p.end - 1), a.d, lane);
  const short* kp = a.k.p + p.kv * a.k.head + p.start * a.k.ld;
  const short* vp = a.v.p + p.kv * a.v.head + p.start * a.v.ld;
  const int hi = a.causal ? min(p.row0 + kRows, p.end) : p.end;
  const int wave_hi = w0 >= p.end ? p.start : a.causal ? min(w0 + 32, p.end) : p.end;
  const int last = a.causal ? min(row, p.end - 1) : p.end - 1;  // the row's last key
  const int nt = (hi - p.start + kTile - 1) / kTile;
  L::arrived(qf);
  auto load = [&](int t) {
    const int left = p.end - p.start - t * kTile;
    L::load(lds[(t / GROUPS) & 1][0], kp + (int64_t)t * kTile * a.k.ld, a.k.ld, left, a.d);
    L::load(lds[(t / GROUPS) & 1][1], vp + (int64_t)t * kTile * a.v.ld, a.v.ld, left, a.d);
  };
  f16v o[L::kBlocks];
#pragma unroll
  for (int i = 0; i < L::kBlocks; i++) o[i] = f16v{};
  float m = -INFINITY, l = 0;
  if (group < nt) load(group);
  for (int t = group; t - group < nt; t += GROUPS) {
    sync_loads();
    if (t + GROUPS < nt) load(t + GROUPS);
    const int j0 = p.start + t * kTile;
    if (j0 >= wave_hi) continue;
    const char *kt = lds[(t / GROUPS) & 1][0], *vt = lds[(t / GROUPS) & 1][1];
    f16v s[2] = {};
#pragma unroll
    for (int i = 0; i < L::kSteps; i++)
#pragma unroll
      for (int b = 0; b < 2; b++) s[b] = T::mfma(L::rows(kt, b * 32, i, lane), qf[i], s[b]);
    feed<2 * L::kSteps, 1, D <= 32 ? 2 : 6>();
    __builtin_amdgcn_sched_barrier(0);
    if (j0 + kTile - 1 > (a.causal ? min(w0, p.end - 1) : p.end - 1)) {
      const int left = only_here(last) - j0 - 4 * half;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) s[b][r] = b * 32 + row_of(r, 0) <= left ? s[b][r] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int r = 1; r < 32; r++) top = fmaxf(top, s[r >> 4][r & 15]);
    top = fmaxf(top, other_half(top)) * a.scale2;
    // The maximum that P is taken against may lag behind by kLazy: the sums are
    // the same, and most tiles need no scaling of o. (4096 rows, 32 heads of 128: 161
    // us, without it 172.)
    if (__any(top > m + kLazy || m == -INFINITY)) {
      // (finite, so that a row whose scores have all been -inf so far stays at zero)
      const float next = fmaxf(fmaxf(m, top), -0x1.fffffep127f), alpha = exp2f(m - next);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < L::kBlocks; i++) o[i] *= alpha;
      m = next;
    }
    const float shift = T::kBias - m;
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], a.scale2, shift));
        l += s[b][r];
      }
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const s8v pf = pack<T>(s[g >> 1], g & 1);
#pragma unroll
      for (int i = 0; i < L::kBlocks; i++) o[i] = T::mfma(L::columns(vt, g * 16, i * 32, lane), pf, o[i]);
    }
    // The first fragments are on their way while the vector unit works, and what
    // is left of its work goes between the matrix instructions.
    constexpr int kFrags = 4 * L::kBlocks, kAhead = kFrags > 4 ? 4 : 2;
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 40, 0);
#pragma unroll
    for (int i = 0; i < kFrags - kAhead; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 80 / (kFrags - kAhead), 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
  }
  l += other_half(l);
  const int rows = min(32, p.end - w0);
  __syncthreads();  // the tiles' place is free
  if (GROUPS == 2) {
    float* there = (float*)shared + w * 64 * (L::kBlocks * 16 + 2) + lane;
    if (group) {
      hand_over<D>(there, o);
      there[L::kBlocks * 16 * 64] = m;
      there[(L::kBlocks * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (!group) {
      const float m2 = there[L::kBlocks * 16 * 64], top = fmaxf(m, m2), mine = exp2f(m - top), theirs = exp2f(m2 - top);
      l = l * mine + there[(L::kBlocks * 16 + 1) * 64] * theirs;
      m = top;
      take_over<D>(there, o, mine, theirs);
    }
    __syncthreads();
    if (group) return;
  }
  if (rows <= 0) return;
  char* strip = (char*)shared + w * 32 * HD * 2;
  const int64_t ld = (int64_t)a.heads * a.d, at = w0 * ld + (int64_t)p.head * a.d;
  store_rows<T, D>(strip, o, 1.0f / l, false, f.out + at, ld, rows, a.d, lane);
  if (f.out_lo) store_rows<T, D>(strip, o, 1.0f / l, true, f.out_lo + at, ld, rows, a.d, lane);
  if (f.lse && half == 0 && row < p.end) f.lse[(int64_t)p.head * a.tokens + row] = m - T::kBias + log2f(l);
}

// ---- backward ------------------------------------------------------------------

struct Backward {
  Rows dout;
  const short* out;     // [tokens][heads][d]
  const short* out_lo;
  const float* lse;     // [heads][tokens]
  float* delta;         // [heads][tokens]: -delta
  short* dq;            // [tokens][heads][d]
  short* dk;            // [tokens][kv_heads][d]
  short* dv;
  float* part;          // where there are several parts: fp32 [2][parts][tokens][kv_heads][d]
  int parts;            // of a tile's work in k_key_grads
};
constexpr int kDeltaBlocks = 512;

// delta, 16 lanes a row, for calls without dq: k_query_grads forms it itself, beside
// the loads of other blocks (bf16, 9 sequences of 53 to 2048 rows, 32 heads of 128, all
// gradients: 518 us instead of 527; 8 x 1024 rows, 12 heads of 64: 81 instead of 89).
// Where few keys matter dP and delta nearly cancel, so that delta is taken from the
// output before its rounding: without what that lost, dq's and dk's errors over those
// of one rounding (64 features, bf16, rows of 2 to 12 keys) are 1.8 instead of 1.1, of
// 1000 keys 1.49 and 1.58 instead of 1.29 and 1.44.
template <class T>
__global__ __launch_bounds__(256) void k_delta(Args a, Backward b) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  const int per = 64 / 16;  // rows of a wave, 16 lanes each
  const int sub = lane & 15;
  for (int64_t i = ((int64_t)blockIdx.x * 4 + w) * per + (lane >> 4); i < rows; i += (int64_t)gridDim.x * 4 * per) {
    float s = 0;
    const int64_t t = i / a.heads;
    const int h = (int)(i - t * a.heads);
    const short* go = b.dout.p + t * b.dout.ld + h * b.dout.head;
    for (int c = sub * 8; c < a.d; c += 128) {
      const s8v x = *(const s8v*)(go + c), y = *(const s8v*)(b.out + i * a.d + c),
                z = *(const s8v*)(b.out_lo + i * a.d + c);
      float chunk = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) chunk = fmaf(T::widen(x[e]), T::widen(y[e]) + T::widen(z[e]), chunk);
      s += chunk;
    }
#pragma unroll
    for (int k = 8; k; k >>= 1) s += __shfl_xor(s, k);
    if (sub == 0) b.delta[(int64_t)h * a.tokens + t] = -s;
  }
}

// fp16 holds a row's dS (k_query_grads; a key's in k_key_grads) times a power of two
// of its own, whose place is a lane: it begins at 2^kLift and goes by the largest dS
// that the row has met, taken to [2^11, 2^12) where one passes 2^15, which scales the
// row's sums as well (exactly). What is below 2^-25 of a row's largest dS loses
// digits, to an error of 2^-36 of that one; a scale that rows share would lose those of
// small rows beside large ones. |dS| is below 2^41 (of finite inputs), so that
// nothing overflows at the start.
constexpr int kLift = 60;
template <class T, int N>
__device__ inline void fit(f16v& ds, f16v* sums, int& lift) {
  if constexpr (T::kScaled) {
    float top = fabsf(ds[0]);
#pragma unroll
    for (int r = 1; r < 16; r++) top = fmaxf(top, fabsf(ds[r]));
    if (!__any(top > 0x1p15f)) return;
    top = fmaxf(top, other_half(top));
    const int by = top > 0x1p15f && top < INFINITY ? 12 - __builtin_amdgcn_frexp_expf(top) : 0;
    const float down = ldexpf(1.0f, by);
    lift += by;
    ds *= down;
#pragma unroll
    for (int i = 0; i < N; i++) {
      // Above 128 features the sums live in the accumulation registers: said before and
      // behind, or they are moved out of them in every round (k_key_grads, 2 x 2048
      // rows, 16 heads of 256, both gradients: 722 us instead of 440).
      if (N > 4) asm volatile("" : "+a"(sums[i]));
      sums[i] *= down;
      if (N > 4) asm volatile("" : "+a"(sums[i]));
    }
  }
}

// dS is rounded to the inputs' type for its products with k and q, which adds an
// error to dq as large as that of dq's own rounding, and a larger one where the
// keys that matter have a direction in common (unrounded, dS adds up to zero along
// a row). What the rounding loses, in the same type, can go through the matrix
// unit as another operand. FEW (sequences of up to kFew rows, by a block's own, and
// small heads, where that effect is largest): all of it does, for dq and dk. Otherwise that of every other 16
// keys, for dq alone. The error of dq over that of one rounding (bf16, 64
// features, 2500 keys): 1.53 with none, 1.32 with every other 16, 1.13 with all; of
// dk with none 1.44; 60 keys, dq and dk: 1.65 with none, 1.07 with all. Time of dq
// for 16384 rows, 16 heads of 64: 0.77 ms with none, 0.89 with every other 16, 1.02
// with all.
constexpr int kFew = 256;
template <int D>
__device__ inline bool few(const Place& p) {
  return D <= 32 || p.end - p.start <= kFew;
}

template <class T, int D, bool FEW, int GROUPS>
__device__ __forceinline__ void query_grads(const Args& a, const Backward& b, const Place& p,
                                            char (&shared)[GROUPS][2][2][Tile<D>::kBytes]) {
  using L = Tile<D>;
  constexpr int HD = L::HD;
  const int lane = threadIdx.x & 63, half = lane >> 5, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  auto& lds = shared[group];
  const int w0 = p.row0 + 32 * w, row = w0 + (lane & 31), there = min(row, p.end - 1);
  s8v qf[L::kSteps], gf[L::kSteps];
  L::own(qf, a.q.p + p.head * a.q.head, a.q.ld, there, a.d, lane);
  L::own(gf, b.dout.p + p.head * b.dout.head, b.dout.ld, there, a.d, lane);
  // A row with one key has P = 1 whatever its score: dS is zero, not the
  // rounding errors of dP - delta.
  const bool one = a.causal ? row == p.start : p.end - p.start == 1;
  const float lse = one ? INFINITY : b.lse[(int64_t)p.head * a.tokens + there];
  float delta;
  int lift = T::kScaled ? kLift : 0;  // of the power of two in dS
  {
    const int64_t at = ((int64_t)there * a.heads + p.head) * a.d;
    s8v y[L::kSteps], z[L::kSteps];
    L::own(y, b.out + at, 0, 0, a.d, lane);
    L::own(z, b.out_lo + at, 0, 0, a.d, lane);
    float sum[L::kSteps];  // a chunk's, added in k_delta's order
#pragma unroll
    for (int i = 0; i < L::kSteps; i++) {
      sum[i] = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) sum[i] = fmaf(T::widen(gf[i][e]), T::widen(y[i][e]) + T::widen(z[i][e]), sum[i]);
    }
#pragma unroll
    for (int n = 8; n; n >>= 1)
#pragma unroll
      for (int i = 0; i < n; i++)
        if (i + n < L::kSteps) sum[i] += sum[i + n];
    delta = -(sum[0] + other_half(sum[0]));
    if (group == 0 && half == 0 && row < p.end) b.delta[(int64_t)p.head * a.tokens + row] = delta;
  }
  const short* kp = a.k.p + p.kv * a.k.head + p.start * a.k.ld;
  const short* vp = a.v.p + p.kv * a.v.head + p.start * a.v.ld;
  const int hi = a.causal ? min(p.row0 + kRows, p.end) : p.end;
  const int wave_hi = w0 >= p.end ? p.start : a.causal ? min(w0 + 32, p.end) : p.end;
  const int last = a.causal ? there : p.end - 1;
  const int nt = (hi - p.start + kTile - 1) / kTile;
  L::arrived(qf);
  L::arrived(gf);
  auto load = [&](int t) {
    const int left = p.end - p.start - t * kTile;
    L::load(lds[(t / GROUPS) & 1][0], kp + (int64_t)t * kTile * a.k.ld, a.k.ld, left, a.d);
    L::load(lds[(t / GROUPS) & 1][1], vp + (int64_t)t * kTile * a.v.ld, a.v.ld, left, a.d);
  };
  f16v dq[L::kBlocks];
#pragma unroll
  for (int i = 0; i < L::kBlocks; i++) dq[i] = f16v{};
  if (group < nt) load(group);
  for (int t = group; t - group < nt; t += GROUPS) {
    sync_loads();
    if (t + GROUPS < nt) load(t + GROUPS);
    const int j0 = p.start + t * kTile;
    if (j0 >= wave_hi) continue;
    const char *kt = lds[(t / GROUPS) & 1][0], *vt = lds[(t / GROUPS) & 1][1];
    const bool edge = j0 + kTile - 1 > (a.causal ? min(w0, p.end - 1) : p.end - 1);
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const float shift = (float)lift - lse;
      f16v s = {}, dp = {};
#pragma unroll
      for (int i = 0; i < L::kSteps; i++) {
        s = T::mfma(L::rows(kt, c * 32, i, lane), qf[i], s);
        dp = T::mfma(L::rows(vt, c * 32, i, lane), gf[i], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, shift));
        s[r] = e * (dp[r] + delta);
      }
      if (edge) {
        const int left = only_here(last) - j0 - c * 32 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = row_of(r, 0) <= left ? s[r] : 0.0f;
      }
      fit<T, L::kBlocks>(s, dq, lift);
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const s8v sf = pack<T>(s, g), rest = pack_rest<T>(s, g, sf);
#pragma unroll
        for (int i = 0; i < L::kBlocks; i++) {
          const s8v kf = L::columns(kt, c * 32 + g * 16, i * 32, lane);
          dq[i] = T::mfma(kf, sf, dq[i]);
          if (FEW || g == 0) dq[i] = T::mfma(kf, rest, dq[i]);
        }
      }
    }
  }
  const int rows = min(32, p.end - w0);
  __syncthreads();
  if (GROUPS == 2) {
    float* there = (float*)shared + w * 64 * (L::kBlocks * 16 + 1) + lane;
    if (group) {
      hand_over<D>(there, dq);
      there[L::kBlocks * 16 * 64] = (float)lift;
    }
    __syncthreads();
    if (!group) {  // to the smaller of the two powers of two
      const int other = (int)there[L::kBlocks * 16 * 64], least = min(lift, other);
      take_over<D>(there, dq, ldexpf(1.0f, least - lift), ldexpf(1.0f, least - other));
      lift = least;
    }
    __syncthreads();
    if (group) return;
  }
  if (rows <= 0) return;
  const int64_t ld = (int64_t)a.heads * a.d;
  store_rows<T, D>((char*)shared + w * 32 * HD * 2, dq, ldexpf(a.scale, -lift), false,
                    b.dq + w0 * ld + (int64_t)p.head * a.d, ld, rows, a.d, lane);
}

template <class T, int D, int GROUPS>
__global__ DSX_ATTENTION_KERNEL(D, 3, GROUPS) void k_query_grads(Args a, Backward b) {
  __shared__ __attribute__((aligned(1024))) char shared[GROUPS][2][2][Tile<D>::kBytes];
  const Place p = place_of(a, a.heads);
  if (!p.good) return;
  if (few<D>(p)) query_grads<T, D, true, GROUPS>(a, b, p, shared);
  else query_grads<T, D, false, GROUPS>(a, b, p, shared);
}

// Rows of fp32 partial sums, one a lane.
template <int D>
__device__ inline void store_part(float* out, const f16v* o, float factor, bool there, int d, int half) {
  if (!there) return;
#pragma unroll
  for (int i = 0; i < D / 32; i++)
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int f = i * 32 + c * 8 + half * 4;
      if (f < d) *(f4v*)(out + f) = f4v{o[i][c * 4], o[i][c * 4 + 1], o[i][c * 4 + 2], o[i][c * 4 + 3]} * factor;
    }
}

// `lds`: two pairs of tiles, then lse and delta of their rows. (One array: with two,
// the compiler waits for all direct loads in flight before each read.)
template <int D>
constexpr int kKeyGradsLds = 4 * Tile<D>::kBytes + 4 * kTile * 4;
template <class T, int D, bool FEW>
__device__ __forceinline__ void key_grads(const Args& a, const Backward& b, const Place& p,
                                          char (&lds)[kKeyGradsLds<D>]) {
  using L = Tile<D>;
  constexpr int HD = L::HD;
  float* stats = (float*)(lds + 4 * L::kBytes);
  const int lane = threadIdx.x & 63, half = lane >> 5, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w0 = p.row0 + 32 * w, key = w0 + (lane & 31), there = min(key, p.end - 1);
  s8v kf[L::kSteps], vf[L::kSteps];
  L::own(kf, a.k.p + p.kv * a.k.head, a.k.ld, there, a.d, lane);
  L::own(vf, a.v.p + p.kv * a.v.head, a.v.ld, there, a.d, lane);
  // The tiles of queries, head by head; the part's share of them. (place_of
  // numbers the parts of a key head as its heads.)
  const int first = a.causal ? p.row0 : p.start, part = p.head % b.parts;
  const int per = (p.end - first + kTile - 1) / kTile;
  const int step0 = (int)((int64_t)per * a.group * part / b.parts);
  const int nt = (int)((int64_t)per * a.group * (part + 1) / b.parts) - step0;
  L::arrived(kf);
  L::arrived(vf);
  float stat = 0;
  auto load = [&](int t, int head, int i0) {
    const int left = p.end - i0;
    L::load(lds + (t & 1) * 2 * L::kBytes, a.q.p + head * a.q.head + i0 * a.q.ld, a.q.ld, left, a.d);
    L::load(lds + ((t & 1) * 2 + 1) * L::kBytes, b.dout.p + head * b.dout.head + i0 * b.dout.ld, b.dout.ld, left, a.d);
    if (w < 2) stat = (w ? b.delta : b.lse)[(int64_t)head * a.tokens + i0 + min(lane, left - 1)];
  };
  Reader<D> reader;
  reader.init((const char*)lds, lane);
  f16v dk[L::kBlocks], dv[L::kBlocks];
#pragma unroll
  for (int i = 0; i < L::kBlocks; i++) dk[i] = dv[i] = f16v{};
  int lift = T::kScaled ? kLift : 0;
  int head = p.kv * a.group + step0 / per, i0 = first + step0 % per * kTile;
  if (nt > 0) load(0, head, i0);
  for (int t = 0; t < nt; t++) {
    if (w < 2) stats[((t & 1) * 2 + w) * kTile + lane] = stat;
    sync_loads();
    const int now = i0;
    i0 += kTile;
    if (i0 >= p.end) {
      i0 = first;
      head++;
    }
    if (t + 1 < nt) load(t + 1, head, i0);
    if (w0 >= p.end || (a.causal && now + kTile - 1 < w0)) continue;
    const bool edge = now + kTile > p.end || (a.causal && now < w0 + 31) || p.end - p.start == 1;
    constexpr int kUnroll = HD == 64 ? 2 : 1;
#pragma unroll kUnroll
    for (int c = 0; c < 2; c++) {
      const Reader<D> rd = reader.from((t & 1) * 2 * L::kBytes + c * 32 * HD * 2);
      const float ds_scale = ldexpf(1.0f, lift - (int)(2 * T::kBias));  // (P's 2^14 is taken off)
      f16v s = {}, dp;  // dP's sums begin at -delta
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const f4v delta = *(const f4v*)&stats[((t & 1) * 2 + 1) * kTile + c * 32 + q * 8 + half * 4];
#pragma unroll
        for (int e = 0; e < 4; e++) dp[q * 4 + e] = delta[e];
      }
#pragma unroll
      for (int i = 0; i < L::kSteps; i++) {
        s = T::mfma(rd.template rows<0>(i), kf[i], s);
        dp = T::mfma(rd.template rows<1>(i), vf[i], dp);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      feed<2 * L::kSteps, 1, D <= 32 ? 2 : 4>();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const f4v lse = *(const f4v*)&stats[(t & 1) * 2 * kTile + c * 32 + q * 8 + half * 4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int r = q * 4 + e;
          s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, 2.0f * T::kBias - lse[e]));
          dp[r] = s[r] * dp[r] * ds_scale;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (edge) {
        // rows [lo, hi) see the key; dS is zero for rows with one key, as in k_query_grads
        const int i0 = now + c * 32 + 4 * half;
        const int lo = only_here(a.causal ? key : p.start) - i0, hi = p.end - i0;
        const int more = (a.causal ? max(key, p.start + 1) : p.end - p.start == 1 ? p.end : p.start) - i0;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int i = row_of(r, 0);
          s[r] = i >= lo && i < hi ? s[r] : 0.0f;
          dp[r] = i >= more && i < hi ? dp[r] : 0.0f;
        }
      }
      fit<T, L::kBlocks>(dp, dk, lift);
      s8v pf[2], sf[2];
#pragma unroll
      for (int g = 0; g < 2; g++) {
        pf[g] = pack<T>(s, g);
        sf[g] = pack<T>(dp, g);
      }
      if (FEW) {
#pragma unroll
        for (int g = 0; g < 2; g++) {
          const s8v rest = pack_rest<T>(dp, g, sf[g]);
#pragma unroll
          for (int i = 0; i < L::kBlocks; i++) dk[i] = T::mfma(rd.template columns<0>(g * 16, i), rest, dk[i]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < 2; g++) {
#pragma unroll
        for (int i = 0; i < L::kBlocks; i++) {
          dv[i] = T::mfma(rd.template columns<1>(g * 16, i), pf[g], dv[i]);
          dk[i] = T::mfma(rd.template columns<0>(g * 16, i), sf[g], dk[i]);
        }
      }
      feed<4 * L::kBlocks, 2, 3>();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  const int rows = min(32, p.end - w0);
  __syncthreads();
  if (rows <= 0) return;
  const float fk = ldexpf(a.scale, -lift), fv = T::kScaled ? 0x1p-14f : 1.0f;
  const int64_t ld = (int64_t)a.kv_heads * a.d, at = w0 * ld + (int64_t)p.kv * a.d;
  if (b.parts > 1) {
    const int64_t plane = (int64_t)a.tokens * ld;
    float* out = b.part + part * plane + at + (lane & 31) * ld;
    store_part<D>(out, dk, fk, key < p.end, a.d, half);
    store_part<D>(out + b.parts * plane, dv, fv, key < p.end, a.d, half);
    return;
  }
  char* strip = (char*)lds + w * 32 * HD * 2;
  store_rows<T, D>(strip, dk, fk, false, b.dk + at, ld, rows, a.d, lane);
  store_rows<T, D>(strip, dv, fv, false, b.dv + at, ld, rows, a.d, lane);
}

template <class T, int D>
__global__ DSX_ATTENTION_KERNEL(D, 3, 1) void k_key_grads(Args a, Backward b) {
  __shared__ __attribute__((aligned(1024))) char lds[kKeyGradsLds<D>];
  const Place p = place_of(a, a.kv_heads * b.parts);
  if (!p.good) return;
  if (few<D>(p)) key_grads<T, D, true>(a, b, p, lds);
  else key_grads<T, D, false>(a, b, p, lds);
}

// The parts' sums, added in order: eight values a thread.
template <class T>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, short* __restrict__ dk,
                                              short* __restrict__ dv, int64_t n, int parts) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n) return;
  const float* p = part + (blockIdx.y ? parts * n : 0) + at;
  f4v x = {}, y = {};
  for (int s = 0; s < parts; s++) {
    x += *(const f4v*)(p + s * n);
    y += *(const f4v*)(p + s * n + 4);
  }
  s8v r;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    r[e] = T::round(x[e]);
    r[e + 4] = T::round(y[e]);
  }
  *(s8v*)((blockIdx.y ? dv : dk) + at) = r;
}

// ---- host ------------------------------------------------------------------

// Parts of k_key_grads' work on a tile: as many blocks as keep the CUs busy until
// the last of them ends, but no more, since the parts' sums go through memory (at
// most kPartBytes of them). In us: a CU takes a step (64 rows against a tile) in
// one per 64 features, where a block can go on with its own only after `alone`;
// what the parts add is written and read again. With one part and with those
// that the rule takes (dk and dv alone, bf16, causal, 128 features): 4096 rows,
// 32 heads (8 of keys) 660 us and 321 with 3; 2048 rows 337 and 114 with 6; of 64
// features, 16384 rows, 16 heads (2) 3321 and 1069 with 8; 8 x 1024 rows, 12 heads
// stay with one, 58, where two take 85. Over 17 shapes it is within 1% of the best
// of 1 to 32 parts on average, 7% at most.
constexpr int64_t kPartBytes = (int64_t)512 << 20;
int parts_of(const DsxAttention& q) {
  const double d = q.head_dim <= 64 ? (q.head_dim <= 32 ? 32 : 64) : round_up(q.head_dim, q.head_dim <= 128 ? 32 : 64);
  const double values = (double)q.tokens * q.kv_heads * q.head_dim;
  double steps = (double)q.pairs / (kRows * kTile);
  if (q.causal) steps = steps / 2 + q.tile_count;
  const double all = steps * q.heads * (d / 64) * (d > 128 ? 1.3 : 1.0) / kCus;
  const int64_t longest = ceil_div(q.longest, kTile) * (q.heads / q.kv_heads);
  const double alone = (double)longest * (1.2 + 0.0125 * d);
  double least = INFINITY;
  int parts = 1;
  for (int p = 1; p <= 64 && p <= longest && (p == 1 || 8.0 * p * values <= kPartBytes); p++) {
    const double us = fmax(all, alone / p) + 0.1 * fmin(all, alone / p) + (p > 1 ? 2.0 + 16.0 * p * values / 5e6 : 0.0);
    if (us < least) {
      least = us;
      parts = p;
    }
  }
  return parts;
}

struct Layout {
  int64_t delta, part, total;
};
Layout layout_of(const DsxAttention& q) {
  Layout l{};
  l.part = round_up(q.tokens * q.heads * 4, 256);
  const int parts = parts_of(q);
  l.total = l.part + (parts > 1 ? round_up(2 * parts * q.tokens * q.kv_heads * q.head_dim * 4, 256) : 0);
  return l;
}

Args args_of(const DsxAttention& q) {
  Args a{};
  a.q = {(const short*)q.q, q.ld_q, q.head_q};
  a.k = {(const short*)q.k, q.ld_k, q.head_k};
  a.v = {(const short*)q.v, q.ld_v, q.head_v};
  a.tiles = (const int4*)q.tiles;
  a.heads = q.heads;
  a.kv_heads = q.kv_heads;
  a.group = q.heads / q.kv_heads;
  a.d = q.head_dim;
  a.tokens = (int)q.tokens;
  a.causal = q.causal;
  a.scale = q.scale;
  a.scale2 = q.scale * 1.44269504088896340736f;
  return a;
}

// Whether a block's tiles are shared by two groups of waves: where the blocks
// leave CUs or half of them idle and have several tiles to share. k_attend (bf16,
// causal) with one and two: 96 blocks of 1024 rows, 64 features, 19.7 and 16.0 us;
// 512 of 4096 rows 69.1 and 55.9; 768 of 1024 rows 26.0 and 28.6; 512 of 256 rows 9.3
// and 10.2; 128 features, 512 of 2048 rows 55.9 and 48.2, 1024 of 2048 rows 86.2 and
// 97.2. k_delta and k_query_grads, 512 of 4096 rows of 64 features: 90.7 and 78.5.
// (Heads above 128 features have no registers for eight waves.)
bool two_groups(int64_t blocks, int64_t longest) { return blocks <= 2 * kCus && longest >= 8 * kTile; }

template <class T, int D>
void forward(const Args& a, const Forward& f, int64_t tiles, int64_t longest, hipStream_t s) {
  const dim3 grid((unsigned)(tiles * a.heads));
  if constexpr (D <= 128)
    if (two_groups(tiles * a.heads, longest)) {
      k_attend<T, D, 2><<<grid, 2 * kThreads, 0, s>>>(a, f);
      return;
    }
  k_attend<T, D, 1><<<grid, kThreads, 0, s>>>(a, f);
}

template <class T, int D>
void backward(Args a, const Backward& b, int64_t tiles, int64_t longest, hipStream_t s) {
  if (!b.dq) k_delta<T><<<kDeltaBlocks, 256, 0, s>>>(a, b);
  const dim3 grid((unsigned)(tiles * a.heads));
  bool two = false;
  if constexpr (D <= 128) {
    two = two_groups(tiles * a.heads, longest);
    if (b.dq && two) k_query_grads<T, D, 2><<<grid, 2 * kThreads, 0, s>>>(a, b);
  }
  if (b.dq && !two) k_query_grads<T, D, 1><<<grid, kThreads, 0, s>>>(a, b);
  if (!b.dk) return;
  a.tiles += tiles;  // by keys
  k_key_grads<T, D><<<dim3((unsigned)(tiles * a.kv_heads * b.parts)), kThreads, 0, s>>>(a, b);
  const int64_t n = (int64_t)a.tokens * a.kv_heads * a.d;
  if (b.parts > 1) k_join<T><<<dim3((unsigned)ceil_div(n, 2048), 2), 256, 0, s>>>(b.part, b.dk, b.dv, n, b.parts);
}

bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check(const char* what, const DsxAttention* q) {
  if (!q) return fail(DSX_EINVAL, "%s: the argument block is NULL", what);
  if (!dsxi::is16(q->dtype)) return fail(DSX_EINVAL, "%s: dtype must be DSX_F16 or DSX_BF16", what);
  if (q->tokens < 0 || q->tokens > DSX_ATTENTION_MAX_TOKENS)
    return fail(DSX_EINVAL, "%s: tokens in [0, %d]", what, DSX_ATTENTION_MAX_TOKENS);
  if (q->kv_heads < 1 || q->heads < q->kv_heads || q->heads % q->kv_heads || q->heads > DSX_ATTENTION_MAX_HEADS)
    return fail(DSX_EINVAL, "%s: heads must be a multiple of kv_heads, at most %d", what, DSX_ATTENTION_MAX_HEADS);
  if (q->head_dim < 8 || q->head_dim % 8 || q->head_dim > DSX_ATTENTION_MAX_HEAD_DIM)
    return fail(DSX_EINVAL, "%s: head_dim must be a multiple of 8 up to %d", what, DSX_ATTENTION_MAX_HEAD_DIM);
  if (q->tile_count < 0 || q->tile_count > q->tokens || (q->tokens && !q->tile_count))
    return fail(DSX_EINVAL, "%s: tile_count must lie in [1, tokens]", what);
  if (q->tile_count * q->heads >= 1 << 24)  // a launch's threads are counted in 32 bits
    return fail(DSX_EINVAL, "%s: tile_count times heads must be below 2^24", what);
  if (q->longest < 0 || q->longest > q->tokens) return fail(DSX_EINVAL, "%s: longest must lie in [0, tokens]", what);
  if (q->pairs < 0 || q->pairs > q->longest * q->tokens)
    return fail(DSX_EINVAL, "%s: pairs must lie in [0, longest * tokens]", what);
  if (!(q->scale > 0.0f) || !(q->scale < INFINITY)) return fail(DSX_EINVAL, "%s: scale must be positive and finite", what);
  return DSX_OK;
}

bool bad_rows(const void* p, int64_t ld, int64_t head, int64_t heads, int64_t d) {
  return !p || off16(p) || ld % 8 || head % 8 || ld < d || (heads > 1 && head < d) || ld > DSX_ATTENTION_MAX_STRIDE ||
         head > INT64_MAX / 4096;
}

int check_device(const char* what, const DsxAttention* q) {
  if (bad_rows(q->q, q->ld_q, q->head_q, q->heads, q->head_dim) ||
      bad_rows(q->k, q->ld_k, q->head_k, q->kv_heads, q->head_dim) ||
      bad_rows(q->v, q->ld_v, q->head_v, q->kv_heads, q->head_dim))
    return fail(DSX_EINVAL, "%s: q, k and v need 16-byte aligned rows, strides that are multiples of 8 and at least "
                "head_dim, row strides of at most %d", what, DSX_ATTENTION_MAX_STRIDE);
  if (!q->tiles || off16(q->tiles)) return fail(DSX_EINVAL, "%s: tiles is NULL or misaligned", what);
  return DSX_OK;
}

// The sizes between powers of two keep the rows of the next one in shared memory
// but leave its last products out. Forward and backward with them and in the next
// size's kernels (bf16, causal): 24 features, 16 heads of 2 x 4096 rows 79 + 304
// and 96 + 399 us; 96, 32 heads (8 of keys) of 4096 rows 139 + 454 and 161 + 534;
// 160, 16 heads (8) of 2 x 2048 rows 89 + 337 and 118 + 453.
#define DSX_BY_HEAD(CALL, T, ...)                                \
  do {                                                           \
    if (args->head_dim <= 32) CALL<T, 32>(__VA_ARGS__);          \
    else if (args->head_dim <= 64) CALL<T, 64>(__VA_ARGS__);     \
    else if (args->head_dim <= 96) CALL<T, 96>(__VA_ARGS__);     \
    else if (args->head_dim <= 128) CALL<T, 128>(__VA_ARGS__);   \
    else if (args->head_dim <= 192) CALL<T, 192>(__VA_ARGS__);   \
    else CALL<T, 256>(__VA_ARGS__);                              \
  } while (0)

}  // namespace

extern "C" {

int64_t dsx_attention_tiles(const int64_t* lengths, int64_t count, int32_t* tiles, int64_t capacity) {
  if (count < 0 || (count && !lengths)) return fail(-1, "dsx_attention_tiles: bad list of lengths");
  int64_t tokens = 0, n = 0;
  for (int64_t i = 0; i < count; i++) {
    if (lengths[i] < 0 || lengths[i] > DSX_ATTENTION_MAX_TOKENS - tokens)
      return fail(-1, "dsx_attention_tiles: lengths must be >= 0 and add up to at most %d", DSX_ATTENTION_MAX_TOKENS);
    tokens += lengths[i];
    n += ceil_div(lengths[i], kRows);
  }
  if (!tiles) return n;
  if (capacity < n) return fail(-1, "dsx_attention_tiles: %lld tiles do not fit", (long long)n);
  // Most work first for causal calls, by counting the tiles of each distance (in
  // tiles) from the sequence's first row, or from its end. Calls that are not causal
  // use the same order, where a tile's work is its whole sequence's: the first tile
  // of a long sequence behind many short ones then comes late.
  int64_t longest = 0;
  for (int64_t i = 0; i < count; i++)
    if (ceil_div(lengths[i], kRows) > longest) longest = ceil_div(lengths[i], kRows);
  int64_t* at = new (std::nothrow) int64_t[2 * (longest + 1)]();
  if (!at) return fail(-1, "dsx_attention_tiles: out of memory");
  for (int64_t i = 0; i < count; i++) at[ceil_div(lengths[i], kRows)]++;
  // at[k]: sequences of k tiles -> tiles at distance k - 1, which sequences of k
  // tiles and more have -> the first place of that distance, the farthest first.
  for (int64_t k = longest - 1; k >= 1; k--) at[k] += at[k + 1];
  int64_t place = 0;
  for (int64_t k = longest; k >= 1; k--) {
    const int64_t c = at[k];
    at[k] = at[longest + 1 + k - 1] = place;
    place += c;
  }
  int64_t row = 0;
  for (int64_t i = 0; i < count; i++) {
    const int64_t k = ceil_div(lengths[i], kRows);
    for (int64_t t = 0; t < k; t++) {
      const int32_t e[4] = {(int32_t)(row + t * kRows), (int32_t)row, (int32_t)(row + lengths[i]), 0};
      int32_t* by_query = tiles + 4 * at[t + 1]++;
      int32_t* by_key = tiles + 4 * (n + at[longest + 1 + (k - 1 - t)]++);
      for (int c = 0; c < 4; c++) by_query[c] = by_key[c] = e[c];
    }
    row += lengths[i];
  }
  delete[] at;
  return n;
}

int dsx_attention_forward(const DsxAttention* args, void* out, void* out_lo, float* lse, void* stream) {
  const char* what = "dsx_attention_forward";
  if (int rc = check(what, args)) return rc;
  if (!args->tokens) return DSX_OK;
  if (int rc = check_device(what, args)) return rc;
  if (!out || off16(out) || off16(out_lo) || ((uintptr_t)lse & 3) || !out_lo != !lse)
    return fail(DSX_EINVAL, "%s: NULL or misaligned output, or one of out_lo and lse alone", what);
  const Args a = args_of(*args);
  const Forward f{(short*)out, (short*)out_lo, lse};
  hipStream_t s = as_stream(stream);
  if (args->dtype == DSX_F16) DSX_BY_HEAD(forward, F16, a, f, args->tile_count, args->longest, s);
  else DSX_BY_HEAD(forward, BF16, a, f, args->tile_count, args->longest, s);
  return launch_status(what);
}

int64_t dsx_attention_workspace_bytes(const DsxAttention* args) {
  if (check("dsx_attention_workspace_bytes", args)) return -1;
  return layout_of(*args).total;
}

int dsx_attention_backward(const DsxAttention* args, const void* out, const void* out_lo, const float* lse,
                           const void* d_out, int64_t ld_dout, int64_t head_dout, void* dq, void* dk, void* dv,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "dsx_attention_backward";
  if (int rc = check(what, args)) return rc;
  if (!args->tokens) return DSX_OK;
  if (int rc = check_device(what, args)) return rc;
  if (!out || !out_lo || !lse || off16(out) || off16(out_lo) || ((uintptr_t)lse & 3))
    return fail(DSX_EINVAL, "%s: NULL or misaligned result of the forward", what);
  if (bad_rows(d_out, ld_dout, head_dout, args->heads, args->head_dim))
    return fail(DSX_EINVAL, "%s: bad gradient of the output", what);
  if (off16(dq) || off16(dk) || off16(dv) || !dk != !dv)
    return fail(DSX_EINVAL, "%s: misaligned gradient, or one of dk and dv alone", what);
  const Layout l = layout_of(*args);
  if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < l.total)
    return fail(DSX_EINVAL, "%s: the workspace must be 256-byte aligned and of %lld bytes", what, (long long)l.total);
  char* ws = (char*)workspace;
  Backward b{};
  b.dout = {(const short*)d_out, ld_dout, head_dout};
  b.out = (const short*)out;
  b.out_lo = (const short*)out_lo;
  b.lse = lse;
  b.delta = (float*)(ws + l.delta);
  b.part = (float*)(ws + l.part);
  b.dq = (short*)dq;
  b.dk = (short*)dk;
  b.dv = (short*)dv;
  b.parts = parts_of(*args);
  const Args a = args_of(*args);
  hipStream_t s = as_stream(stream);
  if (args->dtype == DSX_F16) DSX_BY_HEAD(backward, F16, a, b, args->tile_count, args->longest, s);
  else DSX_BY_HEAD(backward, BF16, a, b, args->tile_count, args->longest, s);
  return launch_status(what);
}

}  // extern "C"
