// bcfft_dense.h — arguments and output stages of the dense-product kernels (bcfft_dense.hip).
#pragma once
#include "bcfft_device.h"

namespace bcfft {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;

struct DenseArgs {
  const void* a[2];                      // operand of the output's rows, per segment of k
  const void* b[2];                      // operand of the output's columns, per segment; GLU: gate and up
  int64_t lda, ldb;                      // elements between rows (by rows) or between k-rows (by columns)
  int64_t k;                             // elements of k per segment
  int64_t m, n;                          // output rows and columns (GLU: columns of h)
  int64_t am, bn;                        // by columns: elements that may be read of a k-row of a, b (>= m, n)
  const void* bias;                      // (n) or null
  const void* res;                       // (m, n) with stride ldr, or null
  int64_t ldr;
  void* y;                               // (m, n) contiguous
  float* z;                              // what the backward needs: x W^T + b (m, n); GLU: g then u (2, m, n); or null
  float* ws;                             // (kz, m, n or 2 n) partial sums
  int segs, kz, act;
};

struct DzArgs {
  const void* dy;
  int64_t ldd;
  const float* z;                        // pre-activation, or g and u
  void* dz;                              // rows of dz, ldz elements apart; or rows of dg and, ldz / 2 further, du
  int64_t ldz;
  float* part;                           // column sums per slice of rows, or null
  int64_t m, n;
  int act, rows;                         // rows per workgroup (dz)
};

// how a product is cut: tile kind (0: few rows or tokens, 1: 128 x 128, 2: 256 x 128 of 16 bits, 3: 256 x 256, 4: 64 x
// 128 with A by rows, 5: 32 x 128 of fp32 with A by rows and B by columns, 6: 64 x 64 with A by rows but for the gated
// form) and slices of k
struct Shape {
  int kind, kz;
};
// C = A B^T of one dtype; A and B by rows or by columns (bcfft_dense_{f32,f16,bf16}.hip)
enum DenseLayout { DENSE_ROWS, DENSE_GLU, DENSE_ROWS_COLS, DENSE_COLS };
void launch_product_f32(const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s);
void launch_product_f16(const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s);
void launch_product_bf16(const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s);

// 16 bytes at an address aligned to the element only (gfx950 serves unaligned global accesses)
template <int E>
struct __attribute__((packed, aligned(E))) Unaligned16 {
  uint32_t w[4];
};
template <int E>
struct __attribute__((packed, aligned(E))) Unaligned8 {
  uint32_t w[2];
};

// elements k .. of a row of kend elements, 16 bytes, zero past the end
template <int E>
__device__ __forceinline__ uint4 load_part(const char* row, int64_t k, int64_t kend) {
  constexpr int EPC = 16 / E;
  uint32_t w[4] = {0, 0, 0, 0};
  if (k + EPC <= kend) {
    const Unaligned16<E> u = *reinterpret_cast<const Unaligned16<E>*>(row + k * E);
    return make_uint4(u.w[0], u.w[1], u.w[2], u.w[3]);
  }
#pragma unroll
  for (int j = 0; j < EPC - 1; ++j) {
    if (k + j < kend) {
      if constexpr (E == 4) w[j] = ((const uint32_t*)row)[k + j];
      else w[j / 2] |= (uint32_t)((const uint16_t*)row)[k + j] << 16 * (j & 1);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// elements i .. i + cnt (cnt <= N, N = 1, 4 or 8) of an array of DT as fp32, 0 past cnt
template <int DT, int N>
__device__ __forceinline__ void load_at(const void* p, int64_t i, int cnt, float (&v)[N]) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  if (N > 1 && cnt == N) {
    uint32_t w[N * E / 4 > 0 ? N * E / 4 : 1];
    if constexpr (N * E >= 16) {
#pragma unroll
      for (int q = 0; q < N * E / 16; ++q) {
        const Unaligned16<E> u = *reinterpret_cast<const Unaligned16<E>*>((const char*)p + i * E + 16 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * q + j] = u.w[j];
      }
    } else if constexpr (N * E == 8) {
      const Unaligned8<E> u = *reinterpret_cast<const Unaligned8<E>*>((const char*)p + i * E);
      w[0] = u.w[0], w[1] = u.w[1];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (DT == BCFFT_F32) {
        v[j] = __uint_as_float(w[j]);
      } else if (j % 2 == 0) {
        const float2 f = unpack16<DT>(w[j / 2]);
        v[j] = f.x;
        if (j + 1 < N) v[j + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < cnt ? load_scalar(p, i + j, DT) : 0.f;
  }
}
template <int DT, int N>
__device__ __forceinline__ void store_at(void* p, int64_t i, int cnt, const float (&v)[N]) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  uint32_t w[(N * E + 3) / 4];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (DT == BCFFT_F32) w[j] = __float_as_uint(v[j]);
    else if (j % 2 == 0) w[j / 2] = pack16<DT>(v[j], j + 1 < N ? v[j + 1] : 0.f);
  }
  if (N > 1 && cnt == N) {
    if constexpr (N * E >= 16) {
#pragma unroll
      for (int q = 0; q < N * E / 16; ++q) {
        Unaligned16<E> u;
#pragma unroll
        for (int j = 0; j < 4; ++j) u.w[j] = w[4 * q + j];
        *reinterpret_cast<Unaligned16<E>*>((char*)p + i * E + 16 * q) = u;
      }
    } else if constexpr (N * E == 8) {
      Unaligned8<E> u;
      u.w[0] = w[0], u.w[1] = w[1];
      *reinterpret_cast<Unaligned8<E>*>((char*)p + i * E) = u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < cnt) {
        if constexpr (DT == BCFFT_F32) ((uint32_t*)p)[i + j] = w[j];
        else ((uint16_t*)p)[i + j] = (uint16_t)(w[j / 2] >> 16 * (j & 1));
      }
    }
  }
}

// ------------------------------------------------------------------ activations (fp32)
// The normal distribution function Phi(z) = erfc(-z / sqrt 2) / 2: for x = |z| / sqrt 2 and t = 1 / (1 + 0.45 x),
// erfc(x) = t exp(-x^2 + p(t)), p the degree 9 Chebyshev fit to log(erfcx(x) / t) over x in [0, 10] (fit error
// 1.3e-8; in fp32 within 2.3e-7 of Phi, 5e-6 relative down to z = -6). A third of the instructions of the
// library's erfc: with that one the epilogue of 2048 x 4096 outputs took half as long as their product.
__device__ __forceinline__ float normal_cdf(float z) {
  const float x = fabsf(z) * 0.70710678f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.45f, x, 1.f));
  float p = 0.183369572f;
  p = fmaf(p, t, -1.043303666f);
  p = fmaf(p, t, 2.375441185f);
  p = fmaf(p, t, -2.667089331f);
  p = fmaf(p, t, 1.544028557f);
  p = fmaf(p, t, -0.7029624839f);
  p = fmaf(p, t, 0.3095381628f);
  p = fmaf(p, t, 0.3691916272f);
  p = fmaf(p, t, 1.002771143f);
  p = fmaf(p, t, -1.370984761f);
  const float q = 0.5f * t * __expf(fmaf(-x, x, p));
  return z < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float act_value(int act, float z) {
  switch (act) {
    case BCFFT_ACT_RELU: return z > 0.f || z != z ? z : 0.f;
    case BCFFT_ACT_SILU: return silu(z);
    case BCFFT_ACT_GELU: return z * normal_cdf(z);
    default: return z;
  }
}
// act(z) and act'(z)
__device__ __forceinline__ void act_both(int act, float z, float& v, float& slope) {
  switch (act) {
    case BCFFT_ACT_RELU:
      v = z > 0.f || z != z ? z : 0.f;
      slope = z > 0.f ? 1.f : z != z ? z : 0.f;
      break;
    case BCFFT_ACT_SILU: {
      const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
      v = z * s;
      slope = s * (1.f + z * (1.f - s));
      break;
    }
    case BCFFT_ACT_GELU: {
      const float phi = normal_cdf(z);
      v = z * phi;
      slope = phi + z * 0.39894228f * __expf(-0.5f * z * z);
      break;
    }
    default:
      v = z;
      slope = 1.f;
  }
}

// ------------------------------------------------------------------ output stages
// N consecutive columns n .. n + cnt of row m, accumulated in fp32; one rounding
template <int DT, int N>
__device__ __forceinline__ void finish_linear(const DenseArgs& a, int64_t m, int64_t n, float (&v)[N], int cnt) {
  if (a.bias) {
    float b[N];
    load_at<DT>(a.bias, n, cnt, b);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += b[j];
  }
  if (a.z) store_at<BCFFT_F32>(a.z, m * a.n + n, cnt, v);
  if (a.act != BCFFT_ACT_NONE) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = act_value(a.act, v[j]);
  }
  if (a.res) {
    float r[N];
    load_at<DT>(a.res, m * a.ldr + n, cnt, r);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += r[j];
  }
  store_at<DT>(a.y, m * a.n + n, cnt, v);
}
template <int DT, int N>
__device__ __forceinline__ void finish_glu(const DenseArgs& a, int64_t m, int64_t n, const float (&g)[N], const float (&u)[N], int cnt) {
  if (a.z) {
    store_at<BCFFT_F32>(a.z, m * a.n + n, cnt, g);
    store_at<BCFFT_F32>(a.z + a.m * a.n, m * a.n + n, cnt, u);
  }
  float h[N];
#pragma unroll
  for (int j = 0; j < N; ++j) h[j] = act_value(a.act, g[j]) * u[j];
  store_at<DT>(a.y, m * a.n + n, cnt, h);
}

// partial sums of a slice of k: rows of 2 n for the gated form, whose `n` here counts both halves
__device__ __forceinline__ int64_t partial_width(const DenseArgs& a) { return a.b[1] && a.segs == 1 ? 2 * a.n : a.n; }
template <int N>
__device__ __forceinline__ void store_partial(const DenseArgs& a, int slice, int64_t m, int64_t n, const float (&v)[N], int cnt) {
  store_at<BCFFT_F32>(a.ws, ((int64_t)slice * a.m + m) * partial_width(a) + n, cnt, v);
}
template <int N>
__device__ __forceinline__ void load_partials(const DenseArgs& a, int64_t m, int64_t n, int cnt, float (&s)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) s[j] = 0.f;
  for (int k = 0; k < a.kz; ++k) {
    float v[N];
    load_at<BCFFT_F32>(a.ws, ((int64_t)k * a.m + m) * partial_width(a) + n, cnt, v);
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] += v[j];
  }
}

}  // namespace bcfft
