// dsx_gemm.h -- the matrix-product tile that the block and Muon kernels share.
//
// C (TM x TN) = sum over k of A(m, k) B(n, k), 16-bit inputs, fp32 sums in
// registers, on the 16x16x32 matrix instruction. Either operand may be stored
//   row:  element (i, k) at p[i * ld + k]   (k contiguous), or
//   col:  element (i, k) at p[k * ld + i]   (i contiguous),
// which covers all products of a layer and its gradients without a transposed
// copy: a col operand is transposed on the way from shared memory to the
// registers by the transposing LDS read (16 lanes read a 4 x 16 block, each
// lane gets one column of it).
//
// A block walks K in tiles of 64, two tiles in shared memory: while the waves
// multiply one, the other is filled by 16-byte loads that go straight to
// shared memory (no registers, no LDS store instructions). A tile is kept in
// 16-byte chunks at permuted places, so that the 16 lanes of a fragment read
// fall on different banks; a direct load writes lane after lane, so it is the
// global address that is permuted.
//
// Edges. A row or column of C past the end reads some valid element instead
// (clamped address) and its sums are not stored. A k past the end must add
// nothing: the places of the last tile that hold no k are written with zeros
// after the loads have landed. The direct loads need 16-byte aligned operands
// whose leading dimension and contiguous length are multiples of 8; anything
// else goes through registers (kRegs), element by element at the edges.
#ifndef DSX_GEMM_H_
#define DSX_GEMM_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsxg {

typedef short    s4v __attribute__((ext_vector_type(4)));
typedef short    s8v __attribute__((ext_vector_type(8)));
typedef short    s8u __attribute__((ext_vector_type(8), aligned(2)));  // any element address
typedef float    f4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16   b8v __attribute__((ext_vector_type(8)));

struct F16 {
  static __device__ inline f4v mfma(s8v a, s8v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  }
  static __device__ inline float widen(short v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ inline short round(float v) { return __builtin_bit_cast(short, (_Float16)v); }
};
struct BF16 {
  static __device__ inline f4v mfma(s8v a, s8v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  }
  static __device__ inline float widen(short v) { return __builtin_bit_cast(float, (uint32_t)(uint16_t)v << 16); }
  static __device__ inline short round(float v) { return __builtin_bit_cast(short, (__bf16)v); }
};

constexpr int kBK = 64;

// One operand of one K segment: `rows` is its extent along i, `k` along k.
struct Operand {
  const short* p;
  int64_t ld;
  int rows;
};

// XCD-aware order of a launch's blocks: block b runs on XCD b % 8, each with
// its own L2, so each XCD gets one contiguous run of tiles.
static __device__ inline int xcd_order(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7;
  return x * q + min(x, r) + (b >> 3);
}

// Tiles of an mt x nt grid in bands of `band` tile rows, column by column
// within a band: the tiles that run together share operands in L2.
static __device__ inline void band_order(int t, int mt, int nt, int band, int* tm, int* tn) {
  const int per = band * nt;
  const int b = t / per, r = t - b * per;
  const int h = min(band, mt - b * band);
  *tn = r / h;
  *tm = b * band + (r - *tn * h);
}

template <int ROWS, bool ROW, int THREADS>
struct Stage {
  static constexpr int kChunks = ROWS * kBK / 8;
  static constexpr int kInstr = (kChunks + THREADS - 1) / THREADS;  // 16-byte chunks per thread
  static constexpr bool kPart = kChunks % THREADS != 0;             // the last waves have none
  static constexpr int kBytes = ROWS * kBK * 2;
  static constexpr int kPerRow = ROW ? kBK / 8 : ROWS / 8;  // chunks in one stored row
  static constexpr bool kRow = ROW;
  static_assert(kChunks % THREADS == 0 || kChunks < THREADS, "whole loads");
  static_assert(kChunks % 64 == 0, "whole waves");

  // Swizzle of a stored row: row tiles permute their 8 chunks by the row pair;
  // col tiles permute 32-byte pairs of chunks by the k rows that one
  // transposing read touches (k%4 and k/8).
  static __device__ inline int chunk_of(int r, int slot) {
    if (ROW) return slot ^ ((r >> 1) & 7);
    const int g = (r & 3) + 4 * ((r >> 3) & 3);
    return (((slot >> 1) ^ (g & (ROWS / 16 - 1))) << 1) | (slot & 1);
  }
  // The stored row and the chunk of the thread's j-th load.
  static __device__ inline void place(int j, int tid, int* r, int* c) {
    const int at = j * THREADS + tid;
    *r = at / kPerRow;
    *c = chunk_of(*r, at % kPerRow);
  }

  // Byte offset from the tile's origin (row i0, first k) of a chunk, clamped
  // to valid elements: i within `rows` (left of the tile's origin: rows - i0),
  // k within `kleft`.
  static __device__ inline uint32_t offset(int r, int c, int64_t ld, int ileft, int kleft) {
    if (ROW) {
      const int rr = min(r, ileft - 1);
      const int k = c * 8 < kleft ? c * 8 : 0;
      return (uint32_t)(((int64_t)rr * ld + k) * 2);
    }
    const int i = c * 8 < ileft ? c * 8 : 0;
    const int kk = min(r, kleft - 1);
    return (uint32_t)(((int64_t)kk * ld + i) * 2);
  }

  // The chunk by elements, for operands off the direct loads' alignment.
  static __device__ inline s8v gather(const short* p, int r, int c, int64_t ld, int ileft, int kleft) {
    s8v v = {0, 0, 0, 0, 0, 0, 0, 0};
    const int i = ROW ? r : c * 8, k = ROW ? c * 8 : r;
    if (i >= ileft || k >= kleft) return v;
    const short* q = p + (ROW ? (int64_t)i * ld + k : (int64_t)k * ld + i);
    const int n = ROW ? kleft - k : ileft - i;
    if (n >= 8) return *(const s8u*)q;
    for (int e = 0; e < n; e++) v[e] = q[e];
    return v;
  }
};

// The product tile. NT = threads, WM x WN waves of (TM/WM) x (TN/WN).
// SPLIT: B's tile is two half tiles from two operands (the gate and the up
// projection), and a wave's columns are half of one and half of the other.
template <class T, int TM_, int TN_, int WM, int WN, bool RA, bool RB, bool DIRECT, bool SPLIT = false>
struct Gemm {
  static constexpr int TM = TM_, TN = TN_, THREADS = WM * WN * 64;
  static constexpr int WTM = TM / WM, WTN = TN / WN, MF = WTM / 16, NF = WTN / 16;
  static constexpr int BROWS = SPLIT ? TN / 2 : TN;
  using SA = Stage<TM, RA, THREADS>;
  using SB = Stage<BROWS, RB, THREADS>;
  static constexpr int NB = SPLIT ? 2 : 1;
  static constexpr int kTile = SA::kBytes + NB * SB::kBytes;
  static constexpr int kLds = 2 * kTile;

  f4v acc[MF][NF];
  int tid, lane, wm, wn;

  __device__ inline void init() {
    tid = threadIdx.x;
    lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    wm = w / WN;
    wn = w % WN;
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
      for (int j = 0; j < NF; j++) acc[i][j] = f4v{0, 0, 0, 0};
  }

  // Row of C within the tile that this lane's fragment (mf) holds, and the
  // first of the four consecutive columns of fragment nf.
  __device__ inline int row_of(int mf) const { return wm * WTM + mf * 16 + (lane & 15); }
  __device__ inline int col_of(int nf) const { return wn * WTN + nf * 16 + (lane >> 4) * 4; }
  // SPLIT: the column within a half tile; fragments nf < NF/2 are the first
  // operand's, the others the second's at the same columns.
  __device__ inline int half_col(int nf) const { return wn * (WTN / 2) + nf * 16 + (lane >> 4) * 4; }

  template <class S>
  static __device__ inline s8v frag(const char* tile, int i0, int kk, int lane) {
    if (S::kRow) {
      const int r = i0 + (lane & 15);
      return *(const s8v*)(tile + r * 128 + (((kk * 4 + (lane >> 4)) ^ ((r >> 1) & 7)) << 4));
    }
    constexpr int rb = S::kPerRow * 16;  // bytes of a stored row
    const int k = kk * 32 + (lane >> 4) * 8 + ((lane & 15) >> 2);
    const int g = ((k & 3) + 4 * ((k >> 3) & 3)) & (S::kPerRow / 2 - 1);
    const char* q = tile + k * rb + (((i0 >> 4) ^ g) << 5) + (lane & 3) * 8;
    typedef __attribute__((address_space(3))) s4v* lp;
    const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q);
    const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 4 * rb));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  __device__ inline void compute(const char* tile) {
    const char* ta = tile;
    const char* tb = tile + SA::kBytes;
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      s8v a[MF], b[NF];
#pragma unroll
      for (int j = 0; j < NF; j++) {
        if (SPLIT)
          b[j] = frag<SB>(tb + (j < NF / 2 ? 0 : SB::kBytes), wn * (WTN / 2) + (j % (NF / 2)) * 16, kk, lane);
        else
          b[j] = frag<SB>(tb, wn * WTN + j * 16, kk, lane);
      }
#pragma unroll
      for (int i = 0; i < MF; i++) a[i] = frag<SA>(ta, wm * WTM + i * 16, kk, lane);
      // B's fragment first: D's lane is then the row of C and its four values
      // are consecutive columns.
#pragma unroll
      for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) acc[i][j] = T::mfma(b[j], a[i], acc[i][j]);
    }
  }

  // Whether this thread's wave loads a part of a tile smaller than the block.
  template <class S>
  __device__ inline bool has() const {
    return !S::kPart || __builtin_amdgcn_readfirstlane(tid >> 6) < S::kChunks / 64;
  }
  template <class S>
  __device__ inline void load_direct(char* dst, const short* p, const uint32_t* off) {
    if (!has<S>()) return;
#pragma unroll
    for (int j = 0; j < S::kInstr; j++) {
      const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)((const char*)p + off[j]),
          (__attribute__((address_space(3))) void*)(dst + j * THREADS * 16 + w * 1024), 16, 0, 0);
    }
  }
  template <class S>
  __device__ inline void offsets(uint32_t* off, const Operand& o, int i0, int kleft) {
#pragma unroll
    for (int j = 0; j < S::kInstr; j++) {
      int r, c;
      S::place(j, tid, &r, &c);
      off[j] = S::offset(r, c, o.ld, o.rows - i0, kleft);
    }
  }
  // Zeros where the last tile holds no k.
  template <class S>
  __device__ inline void zero_tail(char* dst, bool row, int kleft) {
    if (!has<S>()) return;
#pragma unroll
    for (int j = 0; j < S::kInstr; j++) {
      int r, c;
      S::place(j, tid, &r, &c);
      if ((row ? c * 8 : r) >= kleft) *(s8v*)(dst + (j * THREADS + tid) * 16) = s8v{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  template <class S>
  __device__ inline void load_regs(s8v* v, const short* p, int64_t ld, int ileft, int kleft) {
    if (!has<S>()) return;
#pragma unroll
    for (int j = 0; j < S::kInstr; j++) {
      int r, c;
      S::place(j, tid, &r, &c);
      v[j] = S::gather(p, r, c, ld, ileft, kleft);
    }
  }
  template <class S>
  __device__ inline void store_regs(char* dst, const s8v* v) {
    if (!has<S>()) return;
#pragma unroll
    for (int j = 0; j < S::kInstr; j++) *(s8v*)(dst + (j * THREADS + tid) * 16) = v[j];
  }

  // acc += A[m0.., k] B[n0.., k] for k in [0, K). For SPLIT, b0 and b1 are the
  // two half tiles' operands, both at row n0.
  __device__ inline void run(char* lds, const Operand& a, const Operand& b0, const Operand& b1, int m0, int n0,
                             int K) {
    const int nt = (K + kBK - 1) / kBK;
    if (nt <= 0) return;
    const int64_t sa = RA ? kBK : kBK * a.ld, sb = RB ? kBK : kBK * b0.ld, sb1 = RB ? kBK : kBK * b1.ld;
    const short* pa = a.p + (RA ? m0 * a.ld : m0);
    const short* pb = b0.p + (RB ? n0 * b0.ld : n0);
    const short* pb1 = SPLIT ? b1.p + (RB ? n0 * b1.ld : n0) : pb;
    if constexpr (DIRECT) {
      uint32_t oa[SA::kInstr], ob[SB::kInstr], ob1[SPLIT ? SB::kInstr : 1];
      auto set = [&](int kleft) {
        offsets<SA>(oa, a, m0, kleft);
        offsets<SB>(ob, b0, n0, kleft);
        if (SPLIT) offsets<SB>(ob1, b1, n0, kleft);
      };
      auto load = [&](char* dst) {
        load_direct<SA>(dst, pa, oa);
        load_direct<SB>(dst + SA::kBytes, pb, ob);
        if (SPLIT) load_direct<SB>(dst + SA::kBytes + SB::kBytes, pb1, ob1);
        pa += sa;
        pb += sb;
        pb1 += sb1;
      };
      set(K);
      load(lds);
      for (int t = 0; t < nt; t++) {
        char* cur = lds + (t & 1) * kTile;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + 1 < nt) {
          const int left = K - (t + 1) * kBK;
          if (left < kBK) set(left);
          load(lds + ((t + 1) & 1) * kTile);
        } else if (K - t * kBK < kBK) {
          const int left = K - t * kBK;
          zero_tail<SA>(cur, RA, left);
          zero_tail<SB>(cur + SA::kBytes, RB, left);
          if (SPLIT) zero_tail<SB>(cur + SA::kBytes + SB::kBytes, RB, left);
          __syncthreads();
        }
        compute(cur);
      }
    } else {
      s8v va[SA::kInstr], vb[SB::kInstr], vb1[SPLIT ? SB::kInstr : 1];
      auto load = [&](int left) {
        load_regs<SA>(va, pa, a.ld, a.rows - m0, left);
        load_regs<SB>(vb, pb, b0.ld, b0.rows - n0, left);
        if (SPLIT) load_regs<SB>(vb1, pb1, b1.ld, b1.rows - n0, left);
        pa += sa;
        pb += sb;
        pb1 += sb1;
      };
      auto store = [&](char* dst) {
        store_regs<SA>(dst, va);
        store_regs<SB>(dst + SA::kBytes, vb);
        if (SPLIT) store_regs<SB>(dst + SA::kBytes + SB::kBytes, vb1);
      };
      load(K);
      store(lds);
      for (int t = 0; t < nt; t++) {
        __syncthreads();
        if (t + 1 < nt) load(K - (t + 1) * kBK);
        compute(lds + (t & 1) * kTile);
        if (t + 1 < nt) store(lds + ((t + 1) & 1) * kTile);
      }
    }
    __syncthreads();  // the tiles may be filled again
  }
};

}  // namespace dsxg

#endif  // DSX_GEMM_H_
