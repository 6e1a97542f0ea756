// bcfft_dense.hip — the dense projections that a partly patched model keeps (patch_llama_fft.py:343-394
// replaces some layers' projections; the others stay nn.Linear), on the matrix cores:
//   linear     y = act(x W^T + b) + r                    forward and backward
//   glu        h = act(x Wg^T) * (x Wu^T)                both projections and the product in one kernel
// and their gradients dz W, dz^T x, (dg Wg + du Wu), (dg, du)^T x with dz = dy act'(z), dg = dh u act'(g),
// du = dh act(g).
//
// One tile kernel computes C[m][n] = sum_k A(m, k) B(n, k) for all of them. Either operand lies "by rows"
// (k contiguous) or "by columns" (m or n contiguous): forward by rows / by rows, dx by rows / by columns,
// dw by columns / by columns. Products of 16-bit operands are exact in the fp32 accumulators of the
// matrix cores (v_mfma_f32_16x16x32), fp32 operands use v_mfma_f32_16x16x4; one rounding at the end.
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
// loop's own wait and barrier order them.
__device__ __forceinline__ void dma16_base(const char* base, uint32_t off, uint32_t lds) {
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(off), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// every load into LDS and every LDS access of this wave complete, then the workgroup's rendezvous
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ------------------------------------------------------------------ the tile kernel
// WM x WN waves, each (BM / WM) x (BN / WN) of the BM x BN tile in accumulators; two LDS buffers, the next
// tile on its way while the current one is multiplied, one barrier per tile.
// GLU: B's tile is BN / 2 rows of the gate weight and BN / 2 of the up weight, and a wave holds the same
// columns of both, so the product of the two needs no exchange.
// ASYNC: operands whose rows start 16-byte aligned go to LDS directly; else through registers.
template <int DT, bool CA, bool CB, int BM, int BN, int WM, int WN, bool ASYNC, bool GLU>
__global__ __launch_bounds__(64 * WM * WN, 1) void bc_dense_tile_kernel(DenseArgs a) {
  constexpr int NT = 64 * WM * WN, E = DT == BCFFT_F32 ? 4 : 2, BK = 128 / E;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int NB = GLU ? 2 : 1, BR = BN / NB;        // B's sources and rows of each
  constexpr int ABYTES = BM * 128, BBYTES = BN * 128, BUF = ABYTES + BBYTES;
  using OA = Operand<DT, BM, CA, NT>;
  using OB = Operand<DT, BR, CB, NT>;
  static_assert(!GLU || !CB, "the gated form reads weights by rows");
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

  // this slice's run of k tiles
  const int tps = (int)((a.k + BK - 1) / BK);          // tiles per segment
  const int tiles = tps * a.segs;
  const int t0 = uniform((int)((int64_t)tiles * blockIdx.y / a.kz));
  const int t1 = uniform((int)((int64_t)tiles * (blockIdx.y + 1) / a.kz));

  uint32_t offa[OA::PER], offb[OB::PER];
  if constexpr (ASYNC) {
    OA::offsets(offa, mleft, a.lda);
    OB::offsets(offb, nleft, a.ldb);
  }
  auto base_a = [&](int seg, int64_t k) {
    return (const char*)(seg ? a.a[1] : a.a[0]) + (CA ? k * a.lda + m0 : m0 * a.lda + k) * E;
  };
  auto base_b = [&](int src, int64_t k) {
    return (const char*)(src ? a.b[1] : a.b[0]) + (CB ? k * a.ldb + n0 : n0 * a.ldb + k) * E;
  };
  uint4 ra[ASYNC ? 1 : OA::PER], rb[ASYNC ? 1 : NB * OB::PER];
  const uint32_t lds0 = lds_addr(lds);
  const uint32_t wave_lds = (uint32_t)__builtin_amdgcn_readfirstlane(wave) * 1024u;
  int seg = uniform(t0 / tps);                         // where the next tile of k lies
  int64_t at = (int64_t)(t0 - seg * tps) * BK;
  // the next tile on its way into buffer `buf`
  auto stage = [&](int buf) {
    const int64_t k = at;
    const int sg = seg;
    at += BK;
    if (at >= a.k) at = 0, ++seg;
    if constexpr (ASYNC) {
      if (k + BK <= a.k) {
        const uint32_t l = lds0 + buf * BUF + wave_lds;
        const char* pa = base_a(sg, k);
#pragma unroll
        for (int i = 0; i < OA::PER; ++i) dma16_base(pa, offa[i], l + i * NT * 16);
#pragma unroll
        for (int s = 0; s < NB; ++s) {
          const char* pb = base_b(GLU ? s : sg, k);
#pragma unroll
          for (int i = 0; i < OB::PER; ++i) dma16_base(pb, offb[i], l + ABYTES + s * BR * 128 + i * NT * 16);
        }
        return;
      }
    }
    // the last, partial tile of k, or operands that are not 16-byte aligned
    char* out = lds + buf * BUF + tid * 16;
#pragma unroll
    for (int i = 0; i < OA::PER; ++i) {
      const uint4 v = OA::fetch(base_a(sg, k), mleft, a.lda, a.k - k, i);
      if constexpr (ASYNC) *reinterpret_cast<uint4*>(out + i * NT * 16) = v;
      else ra[i] = v;
    }
#pragma unroll
    for (int s = 0; s < NB; ++s) {
#pragma unroll
      for (int i = 0; i < OB::PER; ++i) {
        const uint4 v = OB::fetch(base_b(GLU ? s : sg, k), nleft, a.ldb, a.k - k, i);
        if constexpr (ASYNC) *reinterpret_cast<uint4*>(out + ABYTES + s * BR * 128 + i * NT * 16) = v;
        else rb[s * OB::PER + i] = v;
      }
    }
  };
  auto commit = [&](int buf) {                         // registers -> LDS (not ASYNC)
    char* out = lds + buf * BUF + tid * 16;
    if constexpr (!ASYNC) {
#pragma unroll
      for (int i = 0; i < OA::PER; ++i) *reinterpret_cast<uint4*>(out + i * NT * 16) = ra[i];
#pragma unroll
      for (int s = 0; s < NB; ++s)
#pragma unroll
        for (int i = 0; i < OB::PER; ++i)
          *reinterpret_cast<uint4*>(out + ABYTES + s * BR * 128 + i * NT * 16) = rb[s * OB::PER + i];
    }
  };

  Fragments<DT, BM, CA> fa;
  Fragments<DT, BR, CB> fb;
  fa.init(lane);
  fb.init(lane);
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (t0 < t1) {
    stage(0);
    commit(0);
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    tile_barrier();
    if (t + 1 < t1) stage(buf ^ 1);
    const char* ta = lds + buf * BUF;
    const char* tb = ta + ABYTES;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 vb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (GLU)
          vb[j] = fb.read(tb + (j < FN / 2 ? 0 : BR * 128), wn * (TN / 2) + (j % (FN / 2)) * 16, kk);
        else
          vb[j] = fb.read(tb, wn * TN + j * 16, kk);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const uint4 va = fa.read(ta, wm * TM + i * 16, kk);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mma<DT>(vb[j], va, acc[i][j]);
      }
    }
    if (t + 1 < t1) commit(buf ^ 1);
  }

  // lane: row m0 + .. + (lane & 15), four consecutive columns from 4 (lane >> 4)
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + wm * TM + i * 16 + (lane & 15);
    if (m >= a.m) continue;
#pragma unroll
    for (int j = 0; j < FN / NB; ++j) {
      const int64_t n = n0 + wn * (TN / NB) + j * 16 + 4 * (lane >> 4);
      if (n >= a.n) continue;
      const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
      if constexpr (GLU) {
        if (a.kz > 1) {
          store_partial(a, blockIdx.y, m, n, acc[i][j], cnt);
          store_partial(a, blockIdx.y, m, a.n + n, acc[i][j + FN / 2], cnt);
        } else {
          finish_glu<DT>(a, m, n, acc[i][j], acc[i][j + FN / 2], cnt);
        }
      } else {
        if (a.kz > 1) store_partial(a, blockIdx.y, m, n, acc[i][j], cnt);
        else finish_linear<DT>(a, m, n, acc[i][j], cnt);
      }
    }
  }
}

// sums the slices of a split k in order and finishes the output
template <int DT, bool GLU>
__global__ __launch_bounds__(256) void bc_dense_finish_kernel(DenseArgs a) {
  const int64_t quads = (a.n + 3) / 4, total = quads * a.m;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t m = q / quads, n = (q - m * quads) * 4;
    const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
    f32x4 g = load_partials(a, m, n, cnt);
    if constexpr (GLU) finish_glu<DT>(a, m, n, g, load_partials(a, m, a.n + n, cnt), cnt);
    else finish_linear<DT>(a, m, n, g, cnt);
  }
}

// ------------------------------------------------------------------ few rows
// Up to 16 MT rows of x (decode): bound by the weights' single read. A workgroup takes 16 rows of W (and 16
// of the other weight, GLU), its KW waves a part of k each, straight from memory into the fragments; x comes
// out of L2. The waves' sums meet in LDS.
template <int DT, int MT, int KW, bool GLU>
__global__ __launch_bounds__(64 * KW) void bc_dense_rows_kernel(DenseArgs a) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2, EPC = 16 / E, BK = 128 / E, NB = GLU ? 2 : 1;
  constexpr int UNROLL = 4;
  __shared__ f32x4 part[KW][NB * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t wrow = n0 + l < a.n ? n0 + l : a.n - 1;       // repeated rows are not stored
  const char* pw[NB];
#pragma unroll
  for (int s = 0; s < NB; ++s) pw[s] = (const char*)a.b[s] + wrow * a.ldb * E;
  const char* px[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) px[i] = (const char*)a.a[0] + (16 * i + l < a.m ? 16 * i + l : a.m - 1) * a.lda * E;
  const int64_t tiles = (a.k + BK - 1) / BK;
  const int64_t t0 = tiles * wave / KW, t1 = tiles * (wave + 1) / KW;

  f32x4 acc[NB][MT];
#pragma unroll
  for (int s = 0; s < NB; ++s)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[s][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [&](const char* p, int64_t k) {          // 16 bytes of k, whatever the address
    const Unaligned16<E> u = *reinterpret_cast<const Unaligned16<E>*>(p + k * E);
    return make_uint4(u.w[0], u.w[1], u.w[2], u.w[3]);
  };
  auto step = [&](const uint4 (&w)[NB], const uint4 (&x)[MT]) {
#pragma unroll
    for (int s = 0; s < NB; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[s][i] = mma<DT>(w[s], x[i], acc[s][i]);
  };
  int64_t t = t0;
  for (; t + UNROLL <= t1 && (t + UNROLL) * BK <= a.k; t += UNROLL) {
    uint4 w[UNROLL][2][NB], x[UNROLL][2][MT];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int64_t k = (t + u) * BK + (g + 4 * kk) * EPC;
#pragma unroll
        for (int s = 0; s < NB; ++s) w[u][kk][s] = load(pw[s], k);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[u][kk][i] = load(px[i], k);
      }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) step(w[u][kk], x[u][kk]);
  }
  for (; t < t1; ++t) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int64_t k = t * BK + (g + 4 * kk) * EPC;
      uint4 w[NB], x[MT];
#pragma unroll
      for (int s = 0; s < NB; ++s) w[s] = load_part<E>(pw[s], k, a.k);
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i] = load_part<E>(px[i], k, a.k);
      step(w, x);
    }
  }
#pragma unroll
  for (int s = 0; s < NB; ++s)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][s * MT + i][lane] = acc[s][i];
  __syncthreads();
  for (int i = wave; i < MT; i += KW) {
    const int64_t m = 16 * i + l, n = n0 + 4 * g;
    if (m >= a.m || n >= a.n) continue;
    f32x4 v[NB];
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      v[s] = part[0][s * MT + i][lane];
#pragma unroll
      for (int w = 1; w < KW; ++w) v[s] += part[w][s * MT + i][lane];
    }
    const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
    if constexpr (GLU) finish_glu<DT>(a, m, n, v[0], v[NB - 1], cnt);
    else finish_linear<DT>(a, m, n, v[0], cnt);
  }
}

// ------------------------------------------------------------------ elementwise part of the backward
// dz = dy act'(z) as the next products' operand, rounded once to dtype, and each column's sum over 64 rows
// of the unrounded dz (fp32) for the bias gradient. Thread: 4 columns; workgroup: 1024 columns x 64 rows.
constexpr int DZ_ROWS = 64;
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_dz_kernel(DzArgs a) {
  const int64_t n = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 4;
  if (n >= a.n) return;
  const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
  const int64_t m0 = (int64_t)blockIdx.x * DZ_ROWS, m1 = m0 + DZ_ROWS < a.m ? m0 + DZ_ROWS : a.m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t m = m0; m < m1; ++m) {
    float d[4], z[4];
    load4_at<DT>(a.dy, m * a.ldd + n, cnt, d);
    if (a.z) {
      load4_at<BCFFT_F32>(a.z, m * a.n + n, cnt, z);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float s, v;
        act_both(a.act, z[j], v, s);
        d[j] *= s;
      }
    }
    if (a.dz) store4_at<DT>(a.dz, m * a.n + n, cnt, d);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += d[j];
  }
  if (a.part)
    for (int j = 0; j < cnt; ++j) a.part[(int64_t)blockIdx.x * a.n + n + j] = sum[j];
}
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_db_kernel(const float* __restrict__ part, int64_t slices, int64_t n,
                                                          void* __restrict__ db) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  double s = 0.0;
  for (int64_t k = 0; k < slices; ++k) s += part[k * n + i];
  const float v[4] = {(float)s, 0.f, 0.f, 0.f};
  store4_at<DT>(db, i, 1, v);
}
// dg = dh u act'(g) and du = dh act(g), side by side in rows of 2 n
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_dgu_kernel(DzArgs a) {
  const int64_t quads = (a.n + 3) / 4, total = quads * a.m;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t m = q / quads, n = (q - m * quads) * 4;
    const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
    float d[4], g[4], u[4], dg[4], du[4];
    load4_at<DT>(a.dy, m * a.ldd + n, cnt, d);
    load4_at<BCFFT_F32>(a.z, m * a.n + n, cnt, g);
    load4_at<BCFFT_F32>(a.z + a.m * a.n, m * a.n + n, cnt, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float s, v;
      act_both(a.act, g[j], v, s);
      dg[j] = d[j] * u[j] * s;
      du[j] = d[j] * v;
    }
    store4_at<DT>(a.dz, m * 2 * a.n + n, cnt, dg);
    store4_at<DT>(a.dz, m * 2 * a.n + a.n + n, cnt, du);
  }
}

// ------------------------------------------------------------------ launches
struct Shape {                                         // how a product is cut: tile kind, slices of k
  int kind, kz;                                        // kind 0: few rows; 1: 128 x 128; 2: 256 x 128; 3: 256 x 256
};

static bool aligned_operand(const void* p, int64_t ld, int64_t dim, bool col, int e) {
  return ((uintptr_t)p & 15) == 0 && ld * e % 16 == 0 && (!col || dim * e % 16 == 0);
}

template <int DT, bool CA, bool CB, int BM, int BN, int WM, int WN, bool ASYNC, bool GLU>
static void launch_tile(const DenseArgs& a, hipStream_t s) {
  constexpr int BR = GLU ? BN / 2 : BN;
  constexpr unsigned lds = 2 * (BM + BN) * 128;
  auto kern = bc_dense_tile_kernel<DT, CA, CB, BM, BN, WM, WN, ASYNC, GLU>;
  if constexpr (lds > 65536) (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  const unsigned tiles = (unsigned)(((a.m + BM - 1) / BM) * ((a.n + BR - 1) / BR));
  hipLaunchKernelGGL(kern, dim3(tiles, (unsigned)a.kz), dim3(64 * WM * WN), lds, s, a);
}

template <int DT, bool CA, bool CB, bool GLU>
static void launch_product_as(const DenseArgs& a, Shape sh, hipStream_t s) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  bool async = true;
  for (int i = 0; i < a.segs; ++i) async = async && aligned_operand(a.a[i], a.lda, a.m, CA, E);
  for (int i = 0; i < (GLU ? 2 : a.segs); ++i) async = async && aligned_operand(a.b[i], a.ldb, a.n, CB, E);
  if (!async) launch_tile<DT, CA, CB, 128, 128, 2, 2, false, GLU>(a, s);
  else if (sh.kind == 1) launch_tile<DT, CA, CB, 128, 128, 2, 2, true, GLU>(a, s);
  else if (sh.kind == 2) launch_tile<DT, CA, CB, 256, 128, 4, 2, true, GLU>(a, s);
  else launch_tile<DT, CA, CB, 256, 256, 2, 4, true, GLU>(a, s);
  if (a.kz > 1) {
    const int64_t quads = (a.n + 3) / 4 * a.m;
    const unsigned blocks = (unsigned)((quads + 255) / 256 < 16384 ? (quads + 255) / 256 : 16384);
    hipLaunchKernelGGL((bc_dense_finish_kernel<DT, GLU>), dim3(blocks), dim3(256), 0, s, a);
  }
}

template <int DT, bool GLU>
static void launch_rows(const DenseArgs& a, hipStream_t s) {
  const unsigned groups = (unsigned)((a.n + 15) / 16);
  auto go = [&](auto mt, auto kw) {
    hipLaunchKernelGGL((bc_dense_rows_kernel<DT, mt.value, kw.value, GLU>), dim3(groups), dim3(64 * kw.value), 0, s, a);
  };
  using std::integral_constant;
  if (a.m <= 16 && groups <= 512) go(integral_constant<int, 1>(), integral_constant<int, 8>());
  else if (a.m <= 16) go(integral_constant<int, 1>(), integral_constant<int, 4>());
  else if (groups <= 512) go(integral_constant<int, 2>(), integral_constant<int, 8>());
  else go(integral_constant<int, 2>(), integral_constant<int, 4>());
}

// Tile and slices for an m x n product over k of `parts` column blocks per output (2: gated): the cheapest by
// an estimate in units of one 128 x 128 x 128-byte step: workgroup rounds over the CUs times steps, and for
// slices the partial sums' way through memory.
static Shape choose(int64_t m, int64_t n, int64_t ksteps, int parts, bool forward) {
  if (forward && m <= 32) return {0, 1};
  const int64_t cus = device_cu_count();
  Shape best{1, 1};
  double least = 1e300;
  struct Kind { int kind, bm, bn, slots; double step; };
  const Kind kinds[3] = {{1, 128, 128, 2, 1.15}, {2, 256, 128, 1, 1.9}, {3, 256, 256, 1, 3.4}};
  for (const Kind& q : kinds) {
    const int64_t tiles = ((m + q.bm - 1) / q.bm) * ((n + q.bn / parts - 1) / (q.bn / parts));
    for (int64_t kz = 1; kz <= 16 && (kz == 1 || ksteps / kz >= 8); kz *= 2) {
      const int64_t groups = tiles * kz;
      // groups per CU, and the share of the CU's rate they reach when fewer than `slots` run there
      const int64_t rounds = (groups + cus * q.slots - 1) / (cus * q.slots);
      const double per = groups >= cus * q.slots ? (double)rounds * q.slots : (double)((groups + cus - 1) / cus);
      double cost = per * ((double)(ksteps + kz - 1) / kz + 3.0) * q.step;
      if (kz > 1) cost += 12.0 + (double)(kz + 1) * m * n * parts * 4.0 / 2.2e6;
      if (cost < least) {
        least = cost;
        best = {q.kind, (int)kz};
      }
    }
  }
  return best;
}

template <bool CA, bool CB, bool GLU>
static void launch_product(int dt, const DenseArgs& a, Shape sh, hipStream_t s) {
  if constexpr (!CA && !CB) {
    if (sh.kind == 0) {
      if (dt == BCFFT_F32) launch_rows<BCFFT_F32, GLU>(a, s);
      else if (dt == BCFFT_F16) launch_rows<BCFFT_F16, GLU>(a, s);
      else launch_rows<BCFFT_BF16, GLU>(a, s);
      return;
    }
  }
  if (dt == BCFFT_F32) launch_product_as<BCFFT_F32, CA, CB, GLU>(a, sh, s);
  else if (dt == BCFFT_F16) launch_product_as<BCFFT_F16, CA, CB, GLU>(a, sh, s);
  else launch_product_as<BCFFT_BF16, CA, CB, GLU>(a, sh, s);
}

static bool valid_dt(int d) { return d == BCFFT_F32 || d == BCFFT_F16 || d == BCFFT_BF16; }
static int elem(int d) { return d == BCFFT_F32 ? 4 : 2; }
static int64_t round16(int64_t b) { return (b + 15) / 16 * 16; }
static int64_t ksteps(int64_t k, int dt) { return (k * elem(dt) + 127) / 128; }
static bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
// a tile's byte offsets are 32-bit (256 rows of a stride of up to 2^20 elements), a grid has fewer than 2^31 tiles
static bool valid_sizes(int64_t n, int64_t k, int64_t m) {
  return n >= 0 && n <= (1 << 23) && k >= 1 && k <= (1 << 20) && m >= 1 && m <= (1 << 20);
}
static int64_t partial_bytes(int64_t m, int64_t n, Shape sh) { return sh.kz > 1 ? round16((int64_t)sh.kz * m * n * 4) : 0; }

struct BackwardPlan {                                  // workspace of a backward call
  Shape dx, dw;
  int64_t dz_bytes, part_bytes, slices, ws_dx, ws_dw, total;
};
static BackwardPlan backward_plan(int64_t n, int64_t k, int64_t m, int dt, int parts, int act) {
  BackwardPlan p;
  p.dx = choose(n, k, parts * ksteps(m, dt), 1, false);
  p.dw = choose(parts * m, k, ksteps(n, dt), 1, false);
  p.dz_bytes = parts == 2 || act != BCFFT_ACT_NONE ? round16(n * parts * m * elem(dt)) : 0;
  p.slices = (n + DZ_ROWS - 1) / DZ_ROWS;
  p.part_bytes = parts == 1 ? round16(p.slices * m * 4) : 0;
  p.ws_dx = partial_bytes(n, k, p.dx);
  p.ws_dw = partial_bytes(parts * m, k, p.dw);
  p.total = p.dz_bytes + p.part_bytes + (p.ws_dx > p.ws_dw ? p.ws_dx : p.ws_dw);
  return p;
}

template <class F>
static void by_dtype(int dt, F&& f) {
  if (dt == BCFFT_F32) f(std::integral_constant<int, BCFFT_F32>());
  else if (dt == BCFFT_F16) f(std::integral_constant<int, BCFFT_F16>());
  else f(std::integral_constant<int, BCFFT_BF16>());
}

// dx = [dz] W (parts 1) or dg Wg + du Wu (parts 2: dz holds both, rows of 2 m)
static void launch_dx(int dt, const void* dz, int64_t ldz, const void* w0, const void* w1, int64_t n, int64_t k, int64_t m,
                      Shape sh, void* dx, float* ws, hipStream_t s) {
  DenseArgs a{};
  a.a[0] = dz;
  a.a[1] = (const char*)dz + m * elem(dt);
  a.b[0] = w0;
  a.b[1] = w1;
  a.lda = ldz;
  a.ldb = k;
  a.k = m;
  a.segs = w1 ? 2 : 1;
  a.m = n;
  a.n = k;
  a.y = dx;
  a.ws = ws;
  a.kz = sh.kz;
  launch_product<false, true, false>(dt, a, sh, s);
}
// dw[m][k] = sum over tokens of dz[token][m] x[token][k]
static void launch_dw(int dt, const void* dz, int64_t ldz, const void* x, int64_t ldx, int64_t n, int64_t k, int64_t m,
                      Shape sh, void* dw, float* ws, hipStream_t s) {
  DenseArgs a{};
  a.a[0] = dz;
  a.b[0] = x;
  a.lda = ldz;
  a.ldb = ldx;
  a.k = n;
  a.segs = 1;
  a.m = m;
  a.n = k;
  a.y = dw;
  a.ws = ws;
  a.kz = sh.kz;
  launch_product<true, true, false>(dt, a, sh, s);
}

}  // namespace bcfft

using namespace bcfft;

extern "C" {

int64_t bcfft_dense_workspace_bytes(int op, int64_t n_tokens, int64_t in_features, int64_t out_features, int dtype,
                                    int act) {
  if (!valid_dt(dtype) || !valid_sizes(n_tokens, in_features, out_features) || act < 0 || act > BCFFT_ACT_GELU) return -1;
  if (n_tokens == 0) return 0;
  switch (op) {
    case BCFFT_DENSE_LINEAR:
      return partial_bytes(n_tokens, out_features, choose(n_tokens, out_features, ksteps(in_features, dtype), 1, true));
    case BCFFT_DENSE_GLU:
      return partial_bytes(n_tokens, 2 * out_features, choose(n_tokens, out_features, ksteps(in_features, dtype), 2, true));
    case BCFFT_DENSE_LINEAR_BACKWARD: return backward_plan(n_tokens, in_features, out_features, dtype, 1, act).total;
    case BCFFT_DENSE_GLU_BACKWARD: return backward_plan(n_tokens, in_features, out_features, dtype, 2, act).total;
    default: return -1;
  }
}

int bcfft_dense_linear(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                       int64_t out_features, const void* w, const void* bias, const void* residual, int64_t r_stride,
                       int act, void* y, float* z, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n_tokens, in_features, out_features) || x_stride < in_features || x_stride > (1 << 20) ||
      (residual && r_stride < out_features))
    return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU) return BCFFT_ERR_ARG;
  if (n_tokens == 0) return BCFFT_OK;
  if (!x || !w || !y) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if (!aligned_to(x, e) || !aligned_to(w, e) || !aligned_to(bias, e) || !aligned_to(residual, e) || !aligned_to(y, e) ||
      !aligned_to(z, 4) || !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  Shape sh = choose(n_tokens, out_features, ksteps(in_features, dtype), 1, true);
  const int64_t need = partial_bytes(n_tokens, out_features, sh);
  if (need > 0 && (!workspace || workspace_bytes < need)) sh.kz = 1;
  DenseArgs a{};
  a.a[0] = x;
  a.b[0] = w;
  a.lda = x_stride;
  a.ldb = in_features;
  a.k = in_features;
  a.segs = 1;
  a.m = n_tokens;
  a.n = out_features;
  a.bias = bias;
  a.res = residual;
  a.ldr = r_stride;
  a.y = y;
  a.z = z;
  a.act = act;
  a.ws = (float*)workspace;
  a.kz = sh.kz;
  launch_product<false, false, false>(dtype, a, sh, (hipStream_t)stream);
  return record_launch_status();
}

int bcfft_dense_glu(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                    int64_t out_features, const void* w_gate, const void* w_up, int act, void* h, float* gu,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n_tokens, in_features, out_features) || x_stride < in_features || x_stride > (1 << 20)) return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU) return BCFFT_ERR_ARG;
  if (n_tokens == 0) return BCFFT_OK;
  if (!x || !w_gate || !w_up || !h) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if (!aligned_to(x, e) || !aligned_to(w_gate, e) || !aligned_to(w_up, e) || !aligned_to(h, e) || !aligned_to(gu, 4) ||
      !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  Shape sh = choose(n_tokens, out_features, ksteps(in_features, dtype), 2, true);
  const int64_t need = partial_bytes(n_tokens, 2 * out_features, sh);
  if (need > 0 && (!workspace || workspace_bytes < need)) sh.kz = 1;
  DenseArgs a{};
  a.a[0] = x;
  a.b[0] = w_gate;
  a.b[1] = w_up;
  a.lda = x_stride;
  a.ldb = in_features;
  a.k = in_features;
  a.segs = 1;
  a.m = n_tokens;
  a.n = out_features;
  a.y = h;
  a.z = gu;
  a.act = act;
  a.ws = (float*)workspace;
  a.kz = sh.kz;
  launch_product<false, false, true>(dtype, a, sh, (hipStream_t)stream);
  return record_launch_status();
}

int bcfft_dense_linear_backward(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                                int64_t out_features, const void* w, const void* dy, int64_t dy_stride, const float* z,
                                int act, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n_tokens, in_features, out_features) || x_stride < in_features || x_stride > (1 << 20) ||
      dy_stride < out_features || dy_stride > (1 << 20))
    return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU || n_tokens == 0) return BCFFT_ERR_ARG;
  if (!dy || (act != BCFFT_ACT_NONE && !z) || (dx && !w) || (dw && !x)) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if (!aligned_to(x, e) || !aligned_to(w, e) || !aligned_to(dy, e) || !aligned_to(z, 4) || !aligned_to(dx, e) ||
      !aligned_to(dw, e) || !aligned_to(db, e) || !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  const BackwardPlan p = backward_plan(n_tokens, in_features, out_features, dtype, 1, act);
  if (p.total > 0 && (!workspace || workspace_bytes < p.total)) return BCFFT_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  void* dz = act != BCFFT_ACT_NONE ? ws : nullptr;
  float* part = (float*)(ws + p.dz_bytes);
  float* sums = (float*)(ws + p.dz_bytes + p.part_bytes);
  if (dz || db) {
    const DzArgs d{dy, dy_stride, dz ? z : nullptr, (dx || dw) ? dz : nullptr, db ? part : nullptr, n_tokens, out_features, act};
    by_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL(bc_dense_dz_kernel<dt.value>, dim3((unsigned)p.slices, (unsigned)((out_features + 1023) / 1024)),
                         dim3(256), 0, s, d);
      if (db)
        hipLaunchKernelGGL(bc_dense_db_kernel<dt.value>, dim3((unsigned)((out_features + 255) / 256)), dim3(256), 0, s, part,
                           p.slices, out_features, db);
    });
  }
  const void* g = dz ? dz : dy;
  const int64_t ldg = dz ? out_features : dy_stride;
  if (dx) launch_dx(dtype, g, ldg, w, nullptr, n_tokens, in_features, out_features, p.dx, dx, sums, s);
  if (dw) launch_dw(dtype, g, ldg, x, x_stride, n_tokens, in_features, out_features, p.dw, dw, sums, s);
  return record_launch_status();
}

int bcfft_dense_glu_backward(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                             int64_t out_features, const void* w_gate, const void* w_up, const void* dh,
                             int64_t dh_stride, const float* gu, int act, void* dx, void* dw, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n_tokens, in_features, out_features) || 2 * out_features > (1 << 20) || x_stride < in_features ||
      x_stride > (1 << 20) || dh_stride < out_features)
    return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU || n_tokens == 0) return BCFFT_ERR_ARG;
  if (!dh || !gu || (dx && (!w_gate || !w_up)) || (dw && !x)) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if (!aligned_to(x, e) || !aligned_to(w_gate, e) || !aligned_to(w_up, e) || !aligned_to(dh, e) || !aligned_to(gu, 4) ||
      !aligned_to(dx, e) || !aligned_to(dw, e) || !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  const BackwardPlan p = backward_plan(n_tokens, in_features, out_features, dtype, 2, act);
  if (!workspace || workspace_bytes < p.total) return BCFFT_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  float* sums = (float*)(ws + p.dz_bytes);
  const DzArgs d{dh, dh_stride, gu, ws, nullptr, n_tokens, out_features, act};
  const int64_t quads = (out_features + 3) / 4 * n_tokens;
  const unsigned blocks = (unsigned)((quads + 255) / 256 < 65536 ? (quads + 255) / 256 : 65536);
  by_dtype(dtype, [&](auto dt) { hipLaunchKernelGGL(bc_dense_dgu_kernel<dt.value>, dim3(blocks), dim3(256), 0, s, d); });
  if (dx) launch_dx(dtype, ws, 2 * out_features, w_gate, w_up, n_tokens, in_features, out_features, p.dx, dx, sums, s);
  if (dw) launch_dw(dtype, ws, 2 * out_features, x, x_stride, n_tokens, in_features, 2 * out_features, p.dw, dw, sums, s);
  return record_launch_status();
}

}  // extern "C"
