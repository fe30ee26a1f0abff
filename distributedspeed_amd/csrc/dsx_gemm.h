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
// A block walks K in tiles of 64, two of them in shared memory (four for few
// small tiles, see Gemm): while the waves multiply one, the others are filled by
// 16-byte loads that go straight to shared memory (no registers, no LDS store
// instructions). A tile is kept in
// 16-byte chunks at permuted places, so that the 16 lanes of a fragment read
// fall on different banks; a direct load writes lane after lane, so it is the
// global address that is permuted.
//
// Edges. A row or column of C past the end reads some valid element instead
// (clamped address) and its sums are not stored. A k past the end must add
// nothing: the places of the last tile that hold no k are written with zeros
// after the loads have landed, by whole chunks. The direct loads need 16-byte
// aligned operands whose leading dimension is a multiple of 8 and whose rows
// are either as long or hold zeros up to there; anything else goes through
// registers (DIRECT = false), element by element at the edges.
#ifndef DSX_GEMM_H_
#define DSX_GEMM_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsxg {

typedef short    s4v __attribute__((ext_vector_type(4)));
typedef short    s8v __attribute__((ext_vector_type(8)));
typedef short    s8u __attribute__((ext_vector_type(8), aligned(2)));  // any element address
typedef float    f4v __attribute__((ext_vector_type(4)));
typedef float    f4u __attribute__((ext_vector_type(4), aligned(4)));
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

struct Nothing {};  // of an epilogue that reads nothing

// A kernel of tile G. Two waves a SIMD for the square tiles, which is what
// their shared memory allows: left to itself the compiler aims at more, puts
// the sums into the accumulation registers and moves them back and forth
// within the loop (128-tiles, 4096 x 14336 x 4096: 990 and 1144 TFLOP/s).
#define DSX_TILE_KERNEL(G) \
  __launch_bounds__(G::THREADS) __attribute__((amdgpu_waves_per_eu(G::kWavesPerSimd, G::kWavesPerSimd)))

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
  static constexpr int kGroupMask = ROWS % 256 == 0 ? 15 : ROWS % 128 == 0 ? 7 : 3;  // stays within ROWS / 16 pairs
  static_assert(kChunks % THREADS == 0 || kChunks < THREADS, "whole loads");
  static_assert(kChunks % 64 == 0, "whole waves");

  // Swizzle of a stored row: row tiles permute their 8 chunks by the row pair;
  // col tiles permute 32-byte pairs of chunks by the k rows that one
  // transposing read touches (k%4 and k/8).
  static __device__ inline int chunk_of(int r, int slot) {
    if (ROW) return slot ^ ((r >> 1) & 7);
    const int g = (r & 3) + 4 * ((r >> 3) & 3);
    return (((slot >> 1) ^ (g & kGroupMask)) << 1) | (slot & 1);
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

// The transposing LDS read. `restrict` carries alias information to the
// instruction: without any, the compiler waits for every direct load in flight
// before each such read (tile t + 1's loads before tile t is multiplied),
// although the loads fill the other tile and are waited for at the barrier.
// 256-tiles of col operands, 8192^3: 1122 TFLOP/s so, 1277 with it.
typedef __attribute__((address_space(3))) s4v LdsBlock;
static __device__ inline s4v read_transposed(LdsBlock* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
}

// The product tile: WM x WN waves of (TM/WM) x (TN/WN).
// SPLIT: B's tile is two half tiles from two operands (the gate and the up
// projection), and a wave's columns are half of one and half of the other.
// STAGES: K tiles in shared memory. Two suffice where the tile's products, or
// other blocks on the CU, cover the next one's loads; where a launch has at most
// two blocks of 64-tiles a CU each K tile waits for its loads, and four of them
// hide that: A A of 1024 x 1024 with 784 (227 tiles) 12.3 us with two, 9.7 with
// four; beyond two blocks a CU their shared memory costs more than it gives
// (1001 x 2731, 688 tiles: 17.0 and 20.9).
template <class T, int TM_, int TN_, int WM, int WN, bool RA, bool RB, bool DIRECT, bool SPLIT = false,
          int STAGES = 2>
struct Gemm {
  static constexpr int TM = TM_, TN = TN_, THREADS = WM * WN * 64;
  static constexpr int WTM = TM / WM, WTN = TN / WN, MF = WTM / 16, NF = WTN / 16;
  static constexpr int BROWS = SPLIT ? TN / 2 : TN;
  template <int S>
  using Staged = Gemm<T, TM_, TN_, WM, WN, RA, RB, DIRECT, SPLIT, S>;
  using SA = Stage<TM, RA, THREADS>;
  using SB = Stage<BROWS, RB, THREADS>;
  static constexpr int NB = SPLIT ? 2 : 1;
  static constexpr int kTile = SA::kBytes + NB * SB::kBytes;
  static constexpr int kLds = STAGES * kTile;
  static_assert((STAGES & (STAGES - 1)) == 0 && (DIRECT || STAGES == 2), "slots by a mask; registers hold one tile");
  static constexpr int kWavesFit = 163840 / kLds * (WM * WN) / 4;
  static constexpr int kWavesPerSimd = kWavesFit < 4 ? kWavesFit : 4;

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

  // Hands out C, eight consecutive columns at a time: f(row, col, v, w, raw),
  // both within the tile (within a half tile, v of the first operand and w of
  // the second, for SPLIT). A fragment holds four columns of a row in a lane, 32
  // bytes of 16-bit output a row and instruction; by way of a strip of 16 rows
  // in the wave's own part of shared memory (the tiles' place, free by now) the
  // lanes of a row write 128 bytes together. raw is what pre(row, col) loaded
  // for the same place, two strips ahead.
  // Where COLUMNS, f's v (which it may change) is handed out again by columns:
  // t(col, row0, v), 16 consecutive rows of one column.
  static constexpr int kStripLd = WTN + 4;  // floats: 16 rows fall on different banks
  template <bool COLUMNS, class P, class F, class U>
  __device__ inline void emit(char* lds, P&& pre, F&& f, U&& t) {
    static_assert(WM * WN * 16 * kStripLd * 4 <= kLds, "the strips fit the tiles' place");
    static_assert(!(COLUMNS && SPLIT), "one operand");
    float* strip = (float*)lds + (wm * WN + wn) * 16 * kStripLd;
    constexpr int COLS = SPLIT ? WTN / 2 : WTN, PER = COLS / 8, PASSES = (16 * PER + 63) / 64, AHEAD = 2;
    decltype(pre(0, 0)) raw[AHEAD + 1][PASSES];
    auto at = [&](int q, int* r, int* c) {
      const int p = q * 64 + lane;
      *r = p / PER;
      *c = p % PER * 8;
      return 16 * PER % 64 == 0 || p < 16 * PER;
    };
    auto fetch = [&](int i) {
#pragma unroll
      for (int q = 0; q < PASSES; q++) {
        int r, c;
        if (at(q, &r, &c)) raw[i % (AHEAD + 1)][q] = pre(wm * WTM + i * 16 + r, wn * COLS + c);
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD && i < MF; i++) fetch(i);
#pragma unroll
    for (int i = 0; i < MF; i++) {
      if (i + AHEAD < MF) fetch(i + AHEAD);
#pragma unroll
      for (int j = 0; j < NF; j++) *(f4v*)(strip + (lane & 15) * kStripLd + j * 16 + (lane >> 4) * 4) = acc[i][j];
      wave_sync();
#pragma unroll
      for (int q = 0; q < PASSES; q++) {
        int r, c;
        if (!at(q, &r, &c)) continue;
        float v[8], w[8];
        get8(strip + r * kStripLd + c, v);
        if (SPLIT) get8(strip + r * kStripLd + COLS + c, w);
        f(wm * WTM + i * 16 + r, wn * COLS + c, v, w, raw[i % (AHEAD + 1)][q]);
        if (COLUMNS) put8(strip + r * kStripLd + c, v);
      }
      wave_sync();
      if (COLUMNS) {
#pragma unroll
        for (int c0 = 0; c0 < WTN; c0 += 64) {
          const int c = c0 + lane;
          if (WTN % 64 && c >= WTN) continue;
          float v[16];
#pragma unroll
          for (int r = 0; r < 16; r++) v[r] = strip[r * kStripLd + c];
          t(wn * WTN + c, wm * WTM + i * 16, v);
        }
        wave_sync();
      }
    }
  }
  static __device__ inline void put8(float* p, const float* v) {
    *(f4v*)p = f4v{v[0], v[1], v[2], v[3]};
    *(f4v*)(p + 4) = f4v{v[4], v[5], v[6], v[7]};
  }
  static __device__ inline void get8(const float* p, float* v) {
    const f4v a = *(const f4v*)p, b = *(const f4v*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[e] = a[e];
      v[e + 4] = b[e];
    }
  }
  // Orders a wave's own LDS accesses across its lanes.
  static __device__ inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  template <class S>
  static __device__ inline s8v frag(const char* tile, int i0, int kk, int lane) {
    if (S::kRow) {
      const int r = i0 + (lane & 15);
      return *(const s8v*)(tile + r * 128 + (((kk * 4 + (lane >> 4)) ^ ((r >> 1) & 7)) << 4));
    }
    constexpr int rb = S::kPerRow * 16;  // bytes of a stored row
    const int k = kk * 32 + (lane >> 4) * 8 + ((lane & 15) >> 2);
    const int g = ((k & 3) + 4 * ((k >> 3) & 3)) & S::kGroupMask;
    const char* q = tile + k * rb + (((i0 >> 4) ^ g) << 5) + (lane & 3) * 8;
    const s4v lo = read_transposed((LdsBlock*)q), hi = read_transposed((LdsBlock*)(q + 4 * rb));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  // Waits until all but the last LEFT of this wave's direct loads have landed
  // (they land in order) and its LDS reads are done.
  template <int LEFT>
  static __device__ inline void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
  }
  // A barrier after such a wait for the next tile, `after` more tiles being on
  // their way behind it. The STAGES - 2 last of them may stay so.
  __device__ inline void sync_loads(int after) const {
    constexpr int ahead = STAGES - 2;
    static_assert(STAGES == 2 || !(SA::kPart || SB::kPart), "as many loads in every wave");
    if (ahead && after >= ahead) wait_loads<ahead * (SA::kInstr + NB * SB::kInstr)>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  struct Frags {
    s8v a[MF], b[NF];
  };
  // The fragments of half a K tile (32 of its 64 k).
  __device__ inline void read(Frags& f, const char* tile, int kk) const {
    const char* tb = tile + SA::kBytes;
#pragma unroll
    for (int j = 0; j < NF; j++) {
      if (SPLIT)
        f.b[j] = frag<SB>(tb + (j < NF / 2 ? 0 : SB::kBytes), wn * (WTN / 2) + (j % (NF / 2)) * 16, kk, lane);
      else
        f.b[j] = frag<SB>(tb, wn * WTN + j * 16, kk, lane);
    }
#pragma unroll
    for (int i = 0; i < MF; i++) f.a[i] = frag<SA>(tile, wm * WTM + i * 16, kk, lane);
  }
  // B's fragment first: D's lane is then the row of C and its four values are
  // consecutive columns.
  __device__ inline void multiply(const Frags& f) {
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
      for (int j = 0; j < NF; j++) acc[i][j] = T::mfma(f.b[j], f.a[i], acc[i][j]);
  }
  // Reads of one half tile spread over the products of the other, so that
  // neither unit waits for a burst of the other's (256-tiles, 8192^3, operands
  // row/row, row/col and col/col: 1318, 1294 and 1277 TFLOP/s in the compiler's
  // order, 1316, 1320 and 1332 in this one).
  static __device__ inline void interleave() {
    constexpr int reads = MF * (RA ? 1 : 2) + NF * (RB ? 1 : 2), per = MF * NF / reads > 0 ? MF * NF / reads : 1;
#pragma unroll
    for (int i = 0; i < reads; i++) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // an LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, per, 0);  // matrix instructions
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
      Frags f0, f1;
      auto fill = [&](int t) {
        const int left = K - t * kBK;
        if (left < kBK) set(left);
        load(lds + (t & (STAGES - 1)) * kTile);
      };
      set(K);
      fill(0);
      if (STAGES == 2) sync_loads(0);
#pragma unroll
      for (int t = 1; t < STAGES; t++)
        if (t < nt) fill(t);
      if (STAGES > 2) sync_loads(nt >= STAGES ? nt : 0);
      auto tail = [&](int t) {
        const int left = K - t * kBK;
        if (left >= kBK) return;
        char* cur = lds + (t & (STAGES - 1)) * kTile;
        zero_tail<SA>(cur, RA, left);
        zero_tail<SB>(cur + SA::kBytes, RB, left);
        if (SPLIT) zero_tail<SB>(cur + SA::kBytes + SB::kBytes, RB, left);
        __syncthreads();
      };
      if (nt == 1) tail(0);
      read(f0, lds, 0);
      for (int t = 0; t + 1 < nt; t++) {
        char* cur = lds + (t & (STAGES - 1)) * kTile;
        char* nxt = lds + ((t + 1) & (STAGES - 1)) * kTile;
        read(f1, cur, 1);
        multiply(f0);
        interleave();
        sync_loads(nt - t - 2);  // all of this tile is in registers, all of the next in shared memory
        if (t + STAGES < nt) fill(t + STAGES);
        if (t + 2 >= nt) tail(t + 1);
        read(f0, nxt, 0);
        multiply(f1);
        interleave();
      }
      read(f1, lds + ((nt - 1) & (STAGES - 1)) * kTile, 1);
      multiply(f0);
      multiply(f1);
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
        Frags f;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
          read(f, lds + (t & 1) * kTile, kk);
          multiply(f);
        }
        if (t + 1 < nt) store(lds + ((t + 1) & 1) * kTile);
      }
    }
    __syncthreads();  // the tiles may be filled again
  }
};

}  // namespace dsxg

#endif  // DSX_GEMM_H_
