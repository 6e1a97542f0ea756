// bcfft_dense_tile.h — the tile kernel of the dense products (bcfft_dense.hip).
#pragma once
#include "bcfft_dense.h"

#include <type_traits>

namespace bcfft {

// ------------------------------------------------------------------ matrix-core step
// frag: 16 bytes of k per lane: row lane & 15, 16-byte piece lane >> 4 of 64 bytes. D's rows are a's
// rows, four per lane; D's columns b's rows.
template <int DT>
__device__ __forceinline__ f32x4 mma(uint4 a, uint4 b, f32x4 c) {
  if constexpr (DT == BCFFT_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == BCFFT_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    // lane group g holds k = 4 g .. 4 g + 3: step j multiplies k = 4 g + j of both sides
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}

// ------------------------------------------------------------------ operand tiles
// A tile holds R rows of 128 bytes of k (64 16-bit or 32 fp32 elements), R * 8 pieces of 16 bytes. Piece q
// of the tile lies at LDS byte 16 q (what the direct-to-LDS loads require: lane order), and which global
// piece it is carries the bank swizzle:
//   by rows:    q = 8 row + c holds piece c ^ (row & 7) of the row's 128 bytes
//   by columns: q = CPR krow + c holds piece c ^ swizzle(krow) of the k-row's R elements (CPR = R E / 16)
template <int DT, int R, bool COL, int NT>
struct Operand {
  static constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  static constexpr int EPC = 16 / E;                  // elements per piece
  static constexpr int BK = 128 / E;                  // k per tile
  static constexpr int CPR = R * E / 16;              // pieces per k-row (by columns)
  static constexpr int PER = R * 8 / NT;              // pieces per thread
  static_assert(R * 8 % NT == 0 && NT % 64 == 0, "whole pieces per thread");

  __device__ static __forceinline__ int swizzle(int krow) {
    if constexpr (DT == BCFFT_F32) return ((krow >> 2 & 3) << 2) & (CPR - 1);
    else return (((krow & 3) | (krow >> 3 & 3) << 2) << 1) & (CPR - 1);
  }
  // tile row (or k-row) and global piece of this thread's i-th piece
  __device__ static __forceinline__ void place(int i, int& row, int& piece) {
    const int q = i * NT + (int)threadIdx.x;
    if constexpr (COL) {
      row = q / CPR;
      piece = (q % CPR) ^ swizzle(row);
    } else {
      row = q >> 3;
      piece = (q & 7) ^ (row & 7);
    }
  }
  // byte offsets from the tile's first element, rows (columns) past `dim` repeating the last valid ones:
  // they only reach output rows that are not stored
  __device__ static __forceinline__ void offsets(uint32_t (&off)[PER], int64_t dim, int64_t ld) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, piece;
      place(i, row, piece);
      if constexpr (COL) {
        const int last = (int)(dim / EPC) - 1;
        off[i] = (uint32_t)(row * ld * E) + (uint32_t)(piece < last ? piece : last) * 16u;
      } else {
        const int64_t r = row < dim ? row : dim - 1;
        off[i] = (uint32_t)(r * ld * E) + (uint32_t)piece * 16u;
      }
    }
  }
  // any address and any size: a piece that is not whole inside (dim, kleft) is put together by element,
  // zero outside
  __device__ static __forceinline__ uint4 fetch(const char* base, int64_t dim, int64_t ld, int64_t kleft, int i) {
    int row, piece;
    place(i, row, piece);
    const int64_t r = COL ? piece * EPC : row, k = COL ? row : piece * EPC;
    const int64_t along = COL ? dim - r : kleft - k, across = COL ? kleft - k : dim - r;
    const char* p = base + (COL ? k * ld + r : r * ld + k) * E;
    if (across <= 0 || along <= 0) return make_uint4(0, 0, 0, 0);
    if (along >= EPC) {
      const Unaligned16<E> u = *reinterpret_cast<const Unaligned16<E>*>(p);
      return make_uint4(u.w[0], u.w[1], u.w[2], u.w[3]);
    }
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < EPC - 1; ++j) {
      if (j < along) {
        if constexpr (E == 4) w[j] = ((const uint32_t*)p)[j];
        else w[j / 2] |= (uint32_t)((const uint16_t*)p)[j] << 16 * (j & 1);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Fragment reads: rows base .. base + 15 of a tile for the kk-th 64 bytes of k
template <int DT, int R, bool COL>
struct Fragments {
  static constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  static constexpr int CPR = R * E / 16;
  static constexpr int RB = R * E;
  int lane_off, key;                                   // by columns: the row part, and the swizzle

  __device__ __forceinline__ void init(int lane) {
    const int g = lane >> 4, l = lane & 15;
    if constexpr (!COL) {
      lane_off = l * 128 + ((g ^ (l & 7)) << 4);
      key = 0;
    } else if constexpr (DT == BCFFT_F32) {
      lane_off = 4 * g * RB + (l & 3) * 4;
      key = ((g << 2) & (CPR - 1)) ^ (l >> 2);
    } else {
      const int q4 = l >> 2, p4 = l & 3;
      lane_off = (8 * g + q4) * RB + (p4 & 1) * 8;
      key = (((q4 | g << 2) << 1) & (CPR - 1)) ^ (p4 >> 1);
    }
  }
  __device__ __forceinline__ uint4 read(const char* tile, int base, int kk) const {
    if constexpr (!COL) {
      return *reinterpret_cast<const uint4*>(tile + base * 128 + (lane_off ^ (kk << 6)));
    } else if constexpr (DT == BCFFT_F32) {
      const char* p = tile + lane_off + (((base / 4) ^ key) << 4) + 16 * kk * RB;
      return make_uint4(*(const uint32_t*)p, *(const uint32_t*)(p + RB), *(const uint32_t*)(p + 2 * RB),
                        *(const uint32_t*)(p + 3 * RB));
    } else {
      // a 16-lane group's transposed read: rows 4 of k, each lane receives one column's four values
      const char* p = tile + lane_off + (((base / 8) ^ key) << 4) + 32 * kk * RB;
      using V = __attribute__((address_space(3))) s16x4*;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((V)(p));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((V)(p + 4 * RB));
      const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
      return make_uint4(a.x, a.y, b.x, b.y);
    }
  }
};

// LDS[lds + 16 lane] <- 16 bytes at base + off (per lane). The compiler does not count these loads: the
// loop's own waits and barriers order them.
__device__ __forceinline__ void dma16_base(const char* base, uint32_t off, uint32_t lds) {
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(off), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// this wave's LDS accesses complete and at most N of its loads into LDS outstanding, then the rendezvous
template <int N>
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// this wave's LDS reads complete, then the rendezvous
__device__ __forceinline__ void tile_reuse() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ------------------------------------------------------------------ the tile kernel
// WM x WN waves, each (BM / WM) x (BN / WN) of the BM x BN tile in accumulators. A tile of k is 2 FM steps,
// one row fragment against all column fragments each. What keeps the matrix cores fed:
//  - Two tiles of k are in flight behind the one that is read, at every moment (8192 x 4096 x 4096 bf16: 1188
//    TFLOP/s with one). 256 x 128 tiles have three LDS buffers of A and of B. 256 x 256 tiles fill the 160 KB
//    with three of A and two of B (RB = 2): B's second fragments are in registers before half of a tile's
//    steps are done, a barrier there (HALF) frees its buffer, and the tile after the next goes into it
//    (operands from HBM: 1257 -> 1367 TFLOP/s against loads that wait for the end of the tile; 8192 x 2 (11008) x
//    4096, gated: 1150 -> 1053 us).
//  - The loads of later tiles are issued one per step or two. In one burst after the barrier they hold all
//    waves at the address unit.
//  - k tiles of 128 bytes: 64-byte pieces of rows fetch every 128-byte cache line twice (1101 -> 1025
//    TFLOP/s with 256 x 128 tiles).
//  - Fragments are read two steps ahead of their products, and the barrier to the next tile stands two
//    steps before the current one's end, when its last fragment is in a register: the first reads of the
//    next tile run under the last products of this one.
//  - No branch in the loop: past a run's end the last tile is loaded again and never read.
// 8 waves: with 4 of twice the size the single wave of a SIMD leaves its gaps open (1321 -> 1043).
// Matrix cores busy (gated 8192 x 2 (11008) x 4096): 61 % of the cycles with loads that wait, 74 % so; the clock
// under that load falls from 2.0 to 1.8 GHz, which is what bounds it now.
// GLU: B's tile is BN / 2 rows of the gate weight and BN / 2 of the up weight, and a wave holds the same
// columns of both, so the product of the two needs no exchange.
// Both operands' rows start on 16 bytes (by columns: and hold a multiple of 16 bytes).
template <int DT, bool CA, bool CB, int BM, int BN, int WM, int WN, int RA, int RB, bool GLU>
__global__ __launch_bounds__(64 * WM * WN, 1) void bc_dense_tile_kernel(DenseArgs a) {
  constexpr int NT = 64 * WM * WN, E = DT == BCFFT_F32 ? 4 : 2, BK = 128 / E;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int NB = GLU ? 2 : 1, BR = BN / NB;        // B's sources and rows of each
  constexpr int ABYTES = BM * 128, BBYTES = BN * 128;
  using OA = Operand<DT, BM, CA, NT>;
  using OB = Operand<DT, BR, CB, NT>;
  constexpr int LA = OA::PER, LB = NB * OB::PER;       // loads per thread and tile
  static_assert(!GLU || !CB, "the gated form reads weights by rows");
  constexpr bool REUSE = RB == 2;
  static_assert(RA == 3 && (RB == 3 || RB == 2), "two tiles in flight behind the one that is read");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN, wn = wave % WN;

  // workgroups of one XCD (round-robin by id) take a contiguous run of tiles; within it, columns of GROUP
  // row tiles, so that the operands of the tiles in flight fit the XCD's L2
  const int mt = (int)((a.m + BM - 1) / BM), nt = (int)((a.n + BR - 1) / BR);
  const int total = mt * nt;
  int id = blockIdx.x;
  {
    const int per = total / 8, extra = total % 8, xcd = id % 8, slot = id / 8;
    id = xcd * per + (xcd < extra ? xcd : extra) + slot;
  }
  constexpr int GROUP = 8;
  const int band = id / (GROUP * nt), first = band * GROUP;
  const int high = mt - first < GROUP ? mt - first : GROUP;
  const int tm = first + (id - band * GROUP * nt) % high, tn = (id - band * GROUP * nt) / high;
  const int64_t m0 = (int64_t)uniform(tm) * BM, n0 = (int64_t)uniform(tn) * BR;
  const int64_t mleft = a.m - m0, nleft = a.n - n0;

  uint32_t offa[OA::PER], offb[OB::PER];
  OA::offsets(offa, CA ? a.am - m0 : mleft, a.lda);
  OB::offsets(offb, CB ? a.bn - n0 : nleft, a.ldb);
  const uint32_t lds0 = lds_addr(lds) + (uint32_t)uniform(wave) * 1024u;
  char* const lds_b = lds + RA * ABYTES;               // A's buffers, then B's
  const int64_t step_a = CA ? (int64_t)BK * a.lda * E : 128, step_b = CB ? (int64_t)BK * a.ldb * E : 128;

  Fragments<DT, BM, CA> fa;
  Fragments<DT, BR, CB> fb;
  fa.init(lane);
  fb.init(lane);
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int STEPS = 2 * FM, HALF = FN + (FM > FN ? 2 : 0);
  constexpr int PER_STEP = FN > FM ? FN / FM : 1;      // B's second fragments, read in the first FM steps
  static_assert(FN <= FM * PER_STEP && (!REUSE || (PER_STEP == 1 && HALF < STEPS - 2)), "and before its buffer is loaded anew");
  uint4 va[4], vb[2][FN];
  auto read_a = [&](const char* tile, int s) { return fa.read(tile, wm * TM + s % FM * 16, s / FM); };
  auto read_b = [&](const char* tile, int j, int kk) {
    if constexpr (GLU)
      return fb.read(tile + (j < FN / 2 ? 0 : BR * 128), wn * (TN / 2) + (j % (FN / 2)) * 16, kk);
    else
      return fb.read(tile, wn * TN + j * 16, kk);
  };
  auto first_reads = [&](const char* ta, const char* tb) {
#pragma unroll
    for (int j = 0; j < FN; ++j) vb[0][j] = read_b(tb, j, 0);
    va[0] = read_a(ta, 0);
    va[1] = read_a(ta, 1);
  };

  // this slice's run of k tiles, segment by segment
  const int tps = (int)((a.k + BK - 1) / BK), full = (int)(a.k / BK);   // tiles of a segment, whole ones
  const int tiles = tps * a.segs;
  const int t0 = uniform((int)((int64_t)tiles * blockIdx.y / a.kz));
  const int t1 = uniform((int)((int64_t)tiles * (blockIdx.y + 1) / a.kz));
  for (int seg = 0; seg < a.segs; ++seg) {
    const int s0 = t0 - seg * tps > 0 ? t0 - seg * tps : 0;
    const int s1 = t1 - seg * tps < tps ? t1 - seg * tps : tps;
    if (s0 >= s1) continue;
    const int run = (s1 < full ? s1 : full) - s0;      // whole tiles of this run
    const char* pa = (const char*)(seg ? a.a[1] : a.a[0]) + (CA ? m0 : m0 * a.lda) * E + s0 * step_a;
    const char* pb[NB];
#pragma unroll
    for (int s = 0; s < NB; ++s)
      pb[s] = (const char*)((GLU ? s : seg) ? a.b[1] : a.b[0]) + (CB ? n0 : n0 * a.ldb) * E + s0 * step_b;

    if (run > 0) {
      int left_a = run - 1, left_b = run - 1;          // tiles after the ones that pa, pb point at
      int wa = 0, wb = RA * ABYTES, ra = 0, rb = 0;    // buffers written and read next
      auto load_a = [&](int i) { dma16_base(pa, offa[i], lds0 + wa + i * NT * 16); };
      auto load_b = [&](int i) {
        const int s = i / OB::PER, q = i % OB::PER;
        dma16_base(pb[s], offb[q], lds0 + wb + s * BR * 128 + q * NT * 16);
      };
      // past the run's end the last tile again, never read
      auto next_a = [&]() {
        pa += left_a > 0 ? step_a : 0;
        --left_a;
        wa = wa + ABYTES == RA * ABYTES ? 0 : wa + ABYTES;
      };
      auto next_b = [&]() {
#pragma unroll
        for (int s = 0; s < NB; ++s) pb[s] += left_b > 0 ? step_b : 0;
        --left_b;
        wb = wb + BBYTES == RA * ABYTES + RB * BBYTES ? RA * ABYTES : wb + BBYTES;
      };
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < LA; ++i) load_a(i);
        next_a();
#pragma unroll
        for (int i = 0; i < LB; ++i) load_b(i);
        next_b();
      }
      constexpr int YOUNG = LA + LB;                   // loads of the tile after the next one
      tile_barrier<YOUNG>();
      first_reads(lds, lds_b);
      for (int t = 0; t < run; ++t) {
        const char* ta = lds + ra;
        const char* tb = lds_b + rb;
        ra = ra + ABYTES == RA * ABYTES ? 0 : ra + ABYTES;
        rb = rb + BBYTES == RB * BBYTES ? 0 : rb + BBYTES;
        constexpr int ISSUE = STEPS - 2, SHARE = ISSUE * LA / (LA + LB), FIRST = REUSE ? HALF : SHARE > 0 ? SHARE : 1;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int kk = s / FM, i = s % FM;
          if (REUSE && s == HALF) tile_reuse();        // every wave holds B's fragments
          if (s + 2 < STEPS) va[(s + 2) % 4] = read_a(ta, s + 2);
#pragma unroll
          for (int j = s * PER_STEP; j < (s + 1) * PER_STEP; ++j)
            if (j < FN) vb[1][j] = read_b(tb, j, 1);
          if (s < FIRST) {
#pragma unroll
            for (int q = s * LA / FIRST; q < (s + 1) * LA / FIRST; ++q) load_a(q);
          } else if (s < ISSUE) {
#pragma unroll
            for (int q = (s - FIRST) * LB / (ISSUE - FIRST); q < (s + 1 - FIRST) * LB / (ISSUE - FIRST); ++q) load_b(q);
          }
          if (s == STEPS - 2) {
            next_b();
            next_a();
            tile_barrier<YOUNG>();
            first_reads(lds + ra, lds_b + rb);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mma<DT>(vb[kk][j], va[s % 4], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      tile_barrier<0>();                               // nothing in flight, nobody reading
    }
    if (s1 > full) {                                   // the rest of k, copied: zero past its end
      const int64_t kleft = a.k - (int64_t)full * BK;
      if (run > 0) {
        pa += step_a;
#pragma unroll
        for (int s = 0; s < NB; ++s) pb[s] += step_b;
      }
#pragma unroll
      for (int i = 0; i < LA; ++i) *reinterpret_cast<uint4*>(lds + (tid + i * NT) * 16) = OA::fetch(pa, CA ? a.am - m0 : mleft, a.lda, kleft, i);
#pragma unroll
      for (int s = 0; s < NB; ++s)
#pragma unroll
        for (int i = 0; i < OB::PER; ++i)
          *reinterpret_cast<uint4*>(lds_b + s * BR * 128 + (tid + i * NT) * 16) = OB::fetch(pb[s], CB ? a.bn - n0 : nleft, a.ldb, kleft, i);
      tile_barrier<0>();
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int j = 0; j < FN; ++j) vb[0][j] = read_b(lds_b, j, kk);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const uint4 v = read_a(lds, kk * FM + i);
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mma<DT>(vb[0][j], v, acc[i][j]);
        }
      }
      tile_barrier<0>();
    }
  }

  // The accumulators of 16 rows at a time through the wave's own piece of LDS (its buffers are free, and a
  // wave's LDS accesses are in order), so that a lane finishes eight consecutive columns and a row's columns of
  // this wave are stored as whole lines (16 rows x 64 columns: 8 rows of 128 bytes per store; as they lie in
  // the accumulators 16 rows of 32 bytes: 256 x 256 tiles of k = 64 took 19.1 us, 12.7 so)
  constexpr int OC = TN / NB, PITCH = TN + 4, LPR = OC / 8, RPP = 64 / LPR;
  static_assert(WM * WN * 16 * PITCH * 4 <= RA * ABYTES + RB * BBYTES && 16 % RPP == 0, "the waves' pieces of LDS");
  float* const st = (float*)lds + wave * 16 * PITCH;
  const int r0 = lane / LPR, c0 = lane % LPR * 8;
  const int64_t n = n0 + wn * OC + c0;
  const int cnt = n < a.n ? (a.n - n < 8 ? (int)(a.n - n) : 8) : 0;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j) *reinterpret_cast<f32x4*>(st + (lane & 15) * PITCH + j * 16 + 4 * (lane >> 4)) = acc[i][j];
    asm volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < 16 / RPP; ++p) {
      const int r = p * RPP + r0;
      const int64_t m = m0 + wm * TM + i * 16 + r;
      float v[8], u[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(st + r * PITCH + c0 + 4 * q);
        const f32x4 y = *reinterpret_cast<const f32x4*>(st + r * PITCH + (GLU ? OC : 0) + c0 + 4 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = x[j], u[4 * q + j] = y[j];
      }
      if (m < a.m && cnt > 0) {
        if (a.kz > 1) {
          store_partial(a, blockIdx.y, m, n, v, cnt);
          if constexpr (GLU) store_partial(a, blockIdx.y, m, a.n + n, u, cnt);
        } else if constexpr (GLU) {
          finish_glu<DT>(a, m, n, v, u, cnt);
        } else {
          finish_linear<DT>(a, m, n, v, cnt);
        }
      }
    }
    asm volatile("" ::: "memory");
  }
}

}  // namespace bcfft
