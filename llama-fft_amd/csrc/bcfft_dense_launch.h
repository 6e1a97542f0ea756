// bcfft_dense_launch.h — the dense products' kernels of one dtype and their launch, included by
// bcfft_dense_{f32,f16,bf16}.hip (one translation unit each).
#pragma once
#include "bcfft_dense_tile.h"

#include <atomic>

namespace bcfft {

// sums the slices of a split k in order and finishes the output
template <int DT, bool GLU>
__global__ __launch_bounds__(256) void bc_dense_finish_kernel(DenseArgs a) {
  const int64_t quads = (a.n + 3) / 4, total = quads * a.m;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t m = q / quads, n = (q - m * quads) * 4;
    const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
    float g[4], u[4];
    load_partials(a, m, n, cnt, g);
    if constexpr (GLU) {
      load_partials(a, m, a.n + n, cnt, u);
      finish_glu<DT>(a, m, n, g, u, cnt);
    } else {
      finish_linear<DT>(a, m, n, g, cnt);
    }
  }
}

// ------------------------------------------------------------------ few rows
// 16 MT rows of x (decode; more rows: one block of them per grid row): bound by the weights' single read. A workgroup takes 16 rows of W (and 16
// of the other weight, GLU), its KW waves a part of k each, straight from memory into the fragments; x comes
// out of L2. The waves' sums meet in LDS.
// Past 32 rows x's traffic out of L2 outweighs W's, and two tiles of k at a time fill the registers.
// A wave with few 128-byte tiles of k (8 for 4096 16-bit values) loads four at a time; with more (STREAM) it
// loads one while it multiplies the last: 1 x 4096 -> 2 x 11008 36.9 us against 34.1 from HBM (5.3 TB/s), 1 x
// 11008 -> 4096 22.7 against 20.3, but 1 x 4096 -> 4096 6.6 against 7.0 and every two-row-tile form.
template <int DT, int MT, int KW, bool STREAM, bool GLU>
__global__ __launch_bounds__(64 * KW) void bc_dense_rows_kernel(DenseArgs a) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2, EPC = 16 / E, BK = 128 / E, NB = GLU ? 2 : 1;
  constexpr int UNROLL = MT > 2 ? 2 : 4;
  __shared__ f32x4 part[KW][NB * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
  const int64_t wrow = n0 + l < a.n ? n0 + l : a.n - 1;       // repeated rows are not stored
  const char* pw[NB];
#pragma unroll
  for (int s = 0; s < NB; ++s) pw[s] = (const char*)a.b[s] + wrow * a.ldb * E;
  const char* px[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) px[i] = (const char*)a.a[0] + (m0 + 16 * i + l < a.m ? m0 + 16 * i + l : a.m - 1) * a.lda * E;
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
  if constexpr (STREAM) {
    const int64_t whole = a.k / BK < t1 ? a.k / BK : t1;
    uint4 w[2][2][NB], x[2][2][MT];
    auto fill = [&](int buf, int64_t tile) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int64_t k = tile * BK + (g + 4 * kk) * EPC;
#pragma unroll
        for (int s = 0; s < NB; ++s) w[buf][kk][s] = load(pw[s], k);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[buf][kk][i] = load(px[i], k);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto use = [&](int buf) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) step(w[buf][kk], x[buf][kk]);
      __builtin_amdgcn_sched_barrier(0);
    };
    if (t < whole) {
      fill(0, t);
      for (; t + 2 <= whole; t += 2) {
        fill(1, t + 1);
        use(0);
        fill(0, t + 2 < whole ? t + 2 : whole - 1);    // past the end the last one again, unused
        use(1);
      }
      if (t < whole) {
        use(0);
        ++t;
      }
    }
  } else {
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
    const int64_t m = m0 + 16 * i + l, n = n0 + 4 * g;
    if (m >= a.m || n >= a.n) continue;
    float v[NB][4];
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      f32x4 sum = part[0][s * MT + i][lane];
#pragma unroll
      for (int w = 1; w < KW; ++w) sum += part[w][s * MT + i][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[s][j] = sum[j];
    }
    const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
    if constexpr (GLU) finish_glu<DT>(a, m, n, v[0], v[NB - 1], cnt);
    else finish_linear<DT>(a, m, n, v[0], cnt);
  }
}

// ------------------------------------------------------------------ few tokens' weight gradient
// dw[m][k] = sum over up to 32 tokens of dz[token][m] x[token][k]: bound by the writing of dw. A workgroup takes
// 256 columns, 64 per wave, and `rows` rows; x's fragments stay in registers, dz's lie in LDS by m. D's rows are
// the columns k, so a lane holds runs of them: tile c's row r is column 32 (c / 2) + 8 (r / 4) + 4 (c % 2) + r % 4
// for 16-bit outputs (fp32: 16 c + r), which makes every store 16 bytes of a row's 64. Against tiles that
// stage 64 tokens and their outputs in LDS: 1 token, 22016 x 4096 bf16 71 -> 35 us (the writes' own time), 17024 x
// 8100 fp32 235 -> 130; 16 tokens, 4096 x 4096 fp16 16.6 -> 11.6.
constexpr int FEW_TOKENS = 32;
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_outer_kernel(DenseArgs a, int rows) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2, Q = DT == BCFFT_F32 ? 2 : 1;      // MFMA steps of 32 tokens
  constexpr int EPC = 16 / E, PITCH = FEW_TOKENS * E + 16;
  __shared__ __attribute__((aligned(16))) char dz[256 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l = lane & 15;
  const int tokens = (int)a.k;
  const int64_t k0 = (int64_t)blockIdx.x * 256 + (tid >> 6) * 64, m0 = (int64_t)blockIdx.y * rows;
  // tokens t0 .. of one column, zero past the last: no branch between the loads (past the end the last token's
  // again), so all are in flight together
  auto column = [&](const void* p, int64_t ld, int64_t at, int t0) {
    uint32_t v[EPC];
#pragma unroll
    for (int j = 0; j < EPC; ++j) {
      const int64_t i = (t0 + j < tokens ? t0 + j : tokens - 1) * ld + at;
      if constexpr (DT == BCFFT_F32) v[j] = ((const uint32_t*)p)[i];
      else v[j] = ((const uint16_t*)p)[i];
    }
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < EPC; ++j) w[j * E / 4] |= (t0 + j < tokens ? v[j] : 0u) << (E == 4 ? 0 : 16 * (j & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  uint4 xf[4][Q];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int64_t k = k0 + (DT == BCFFT_F32 ? 16 * c + l : 32 * (c / 2) + 8 * (l / 4) + 4 * (c % 2) + l % 4);
    const int64_t at = k < a.n ? k : a.n - 1;          // columns that are not stored
#pragma unroll
    for (int q = 0; q < Q; ++q) xf[c][q] = column(a.b[0], a.ldb, at, (q * 4 + g) * EPC);
  }
  if (tid < rows) {
    const int64_t m = m0 + tid < a.m ? m0 + tid : a.m - 1;
#pragma unroll
    for (int p = 0; p < FEW_TOKENS / EPC; ++p)
      *reinterpret_cast<uint4*>(dz + tid * PITCH + p * 16) = column(a.a[0], a.lda, m, p * EPC);
  }
  __syncthreads();
  const int64_t left = a.m - m0;
  const int count = left < rows ? (int)left : rows;
  for (int i = 0; i < count; i += 16) {
    uint4 zf[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) zf[q] = *reinterpret_cast<const uint4*>(dz + (i + l) * PITCH + (q * 4 + g) * 16);
    f32x4 d[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      d[c] = mma<DT>(xf[c][0], zf[0], f32x4{0.f, 0.f, 0.f, 0.f});
      if constexpr (Q > 1) d[c] = mma<DT>(xf[c][Q - 1], zf[Q - 1], d[c]);
    }
    if (i + l >= count) continue;
    const int64_t row = (m0 + i + l) * a.n;
    constexpr int N = EPC, STORES = 16 / N;            // columns per store
#pragma unroll
    for (int s = 0; s < STORES; ++s) {
      const int64_t k = k0 + (DT == BCFFT_F32 ? 16 * s + 4 * g : 32 * s + 8 * g);
      float v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = d[s * N / 4 + j / 4][j % 4];
      if (k < a.n) store_at<DT>(a.y, row + k, a.n - k < N ? (int)(a.n - k) : N, v);
    }
  }
}

template <int DT, bool CA, bool CB, int BM, int BN, int WM, int WN, int RA, int RB, bool GLU>
static void launch_tile(const DenseArgs& a, hipStream_t s) {
  constexpr int BR = GLU ? BN / 2 : BN;
  constexpr unsigned lds = (RA * BM + RB * BN) * 128;
  auto kern = bc_dense_tile_kernel<DT, CA, CB, BM, BN, WM, WN, RA, RB, GLU>;
  // once per device: the attribute call costs the host as much as the launch
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  (void)hipGetDevice(&dev);
  if (dev > 63 || !(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (dev <= 63) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const unsigned tiles = (unsigned)(((a.m + BM - 1) / BM) * ((a.n + BR - 1) / BR));
  hipLaunchKernelGGL(kern, dim3(tiles, (unsigned)a.kz), dim3(64 * WM * WN), lds, s, a);
}

template <int DT, bool CA, bool CB, bool GLU>
static void launch_tiles(const DenseArgs& a, int kind, hipStream_t s) {
  if (kind == 1) launch_tile<DT, CA, CB, 128, 128, 2, 2, 3, 2, GLU>(a, s);
  if constexpr (DT != BCFFT_F32)
    if (kind == 2) launch_tile<DT, CA, CB, 256, 128, 4, 2, 3, 3, GLU>(a, s);
  if (kind == 3) launch_tile<DT, CA, CB, 256, 256, 2, 4, 3, 2, GLU>(a, s);
  if constexpr (!CA)
    if (kind == 4) launch_tile<DT, CA, CB, 64, 128, 2, 2, 3, 3, GLU>(a, s);
  if constexpr (DT == BCFFT_F32 && CB && !CA)
    if (kind == 5) launch_tile<DT, CA, CB, 32, 128, 1, 4, 3, 3, GLU>(a, s);
  if constexpr (!CA && !GLU)
    if (kind == 6) launch_tile<DT, CA, CB, 64, 64, 2, 2, 3, 3, GLU>(a, s);
  if (a.kz > 1) {
    const int64_t quads = (a.n + 3) / 4 * a.m;
    const unsigned blocks = (unsigned)((quads + 255) / 256 < 16384 ? (quads + 255) / 256 : 16384);
    hipLaunchKernelGGL((bc_dense_finish_kernel<DT, GLU>), dim3(blocks), dim3(256), 0, s, a);
  }
}

template <int DT, bool GLU>
static void launch_rows(const DenseArgs& a, hipStream_t s) {
  const unsigned groups = (unsigned)((a.n + 15) / 16);
  const int64_t tiles = (a.k * (DT == BCFFT_F32 ? 4 : 2) + 127) / 128;
  auto go = [&](auto mt, auto kw, auto stream) {
    hipLaunchKernelGGL((bc_dense_rows_kernel<DT, mt.value, kw.value, stream.value, GLU>), dim3(groups, (unsigned)((a.m + 16 * mt.value - 1) / (16 * mt.value))),
                       dim3(64 * kw.value), 0, s, a);
  };
  using std::integral_constant;
  using std::bool_constant;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  const integral_constant<int, 3> three;
  const integral_constant<int, 4> four;
  // 8 waves per 16 rows of W while that leaves no more than two workgroups per CU, 4 beyond
  auto with = [&](auto kw) {
    if (a.m > 48) go(four, kw, bool_constant<false>());
    else if (a.m > 32) go(three, kw, bool_constant<false>());
    else if (a.m > 16) go(two, kw, bool_constant<false>());
    else if (tiles >= 12 * kw.value) go(one, kw, bool_constant<true>());
    else go(one, kw, bool_constant<false>());
  };
  if (groups <= 512) with(integral_constant<int, 8>());
  else with(integral_constant<int, 4>());
}

template <int DT>
static void launch_outer(const DenseArgs& a, hipStream_t s) {
  const int64_t across = (a.n + 255) / 256;
  // 256 rows per workgroup where that makes four per CU, else 64
  const int rows = across * ((a.m + 255) / 256) >= 4 * device_cu_count() ? 256 : 64;
  hipLaunchKernelGGL(bc_dense_outer_kernel<DT>, dim3((unsigned)across, (unsigned)((a.m + rows - 1) / rows)), dim3(256), 0, s, a, rows);
}

template <int DT>
static void launch_product_dt(const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s) {
  switch (layout) {
    case DENSE_ROWS: return sh.kind == 0 ? launch_rows<DT, false>(a, s) : launch_tiles<DT, false, false, false>(a, sh.kind, s);
    case DENSE_GLU: return sh.kind == 0 ? launch_rows<DT, true>(a, s) : launch_tiles<DT, false, false, true>(a, sh.kind, s);
    case DENSE_ROWS_COLS: return launch_tiles<DT, false, true, false>(a, sh.kind, s);
    case DENSE_COLS: return sh.kind == 0 ? launch_outer<DT>(a, s) : launch_tiles<DT, true, true, false>(a, sh.kind, s);
  }
}

}  // namespace bcfft
