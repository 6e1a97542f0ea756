// bcfft_dense.hip — the dense projections that a partly patched model keeps (patch_llama_fft.py:343-394
// replaces some layers' projections; the others stay nn.Linear), on the matrix cores:
//   linear     y = act(x W^T + b) + r                    forward and backward
//   glu        h = act(x Wg^T) * (x Wu^T)                both projections and the product in one kernel
// and their gradients dz W, dz^T x, (dg Wg + du Wu), (dg, du)^T x with dz = dy act'(z), dg = dh u act'(g),
// du = dh act(g).
//
// The products run in bcfft_dense_{f32,f16,bf16}.hip; here are the elementwise kernels between them, the choice
// of tiles and the C entry points.
#include "bcfft_dense.h"

#include <cmath>
#include <type_traits>

namespace bcfft {

// ------------------------------------------------------------------ elementwise part of the backward
// dz = dy act'(z) as the next products' operand, rounded once to dtype, and each column's sum over a.rows rows
// of the unrounded dz (fp32) for the bias gradient. Workgroup: 256 columns x a.rows rows.
// Both are bound by memory: 4 rows of 64 column quads per pass, the row lanes' sums joined in LDS.
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_dz_kernel(DzArgs a) {
  __shared__ float sums[4][64][5];
  const int quad = threadIdx.x & 63, lane = threadIdx.x >> 6;
  const int64_t n = ((int64_t)blockIdx.y * 64 + quad) * 4;
  const int64_t m0 = (int64_t)blockIdx.x * a.rows;
  const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (n < a.n) {
#pragma unroll 4
    for (int r = 0; r < a.rows / 4; ++r) {
      const int64_t m = m0 + 4 * r + lane;
      if (m >= a.m) break;
      float d[4], z[4];
      load_at<DT>(a.dy, m * a.ldd + n, cnt, d);
      if (a.z) {
        load_at<BCFFT_F32>(a.z, m * a.n + n, cnt, z);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float s, v;
          act_both(a.act, z[j], v, s);
          d[j] *= s;
        }
      }
      if (a.dz) store_at<DT>(a.dz, m * a.ldz + n, cnt, d);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += d[j];
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) sums[lane][quad][j] = sum[j];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (col < a.n) {
    const int q = threadIdx.x >> 2, j = threadIdx.x & 3;
    a.part[(int64_t)blockIdx.x * a.n + col] = (sums[0][q][j] + sums[1][q][j]) + (sums[2][q][j] + sums[3][q][j]);
  }
}
// 32 columns, 8 lanes of slices each
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_db_kernel(const float* __restrict__ part, int64_t slices, int64_t n,
                                                          void* __restrict__ db) {
  __shared__ double sums[8][32];
  const int c = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + c;
  double s = 0.0;
  if (i < n) {
#pragma unroll 4
    for (int64_t k = lane; k < slices; k += 8) s += part[k * n + i];
  }
  sums[lane][c] = s;
  __syncthreads();
  if (lane == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sums[k][c];
    const float v[1] = {(float)s};
    store_at<DT>(db, i, 1, v);
  }
}
// dg = dh u act'(g) and du = dh act(g), side by side in a row
template <int DT>
__global__ __launch_bounds__(256) void bc_dense_dgu_kernel(DzArgs a) {
  const int64_t quads = (a.n + 3) / 4, total = quads * a.m;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t m = q / quads, n = (q - m * quads) * 4;
    const int cnt = a.n - n < 4 ? (int)(a.n - n) : 4;
    float d[4], g[4], u[4], dg[4], du[4];
    load_at<DT>(a.dy, m * a.ldd + n, cnt, d);
    load_at<BCFFT_F32>(a.z, m * a.n + n, cnt, g);
    load_at<BCFFT_F32>(a.z + a.m * a.n, m * a.n + n, cnt, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float s, v;
      act_both(a.act, g[j], v, s);
      dg[j] = d[j] * u[j] * s;
      du[j] = d[j] * v;
    }
    store_at<DT>(a.dz, m * a.ldz + n, cnt, dg);
    store_at<DT>(a.dz, m * a.ldz + a.ldz / 2 + n, cnt, du);
  }
}

// rows of `cols` elements, 16-byte aligned and padded with zeros to whole 16-byte pieces: operands whose rows
// do not start on 16 bytes run the same direct-to-LDS kernels (one copy of the operand at memory speed,
// against products at a third of the rate with loads through registers)
template <int E>
__global__ __launch_bounds__(256) void bc_dense_pack_kernel(const char* __restrict__ src, int64_t ld, int64_t rows,
                                                            int64_t cols, char* __restrict__ dst) {
  constexpr int EPC = 16 / E;
  const int64_t pieces = (cols + EPC - 1) / EPC, total = pieces * rows;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t r = q / pieces, c = q - r * pieces;
    *reinterpret_cast<uint4*>(dst + q * 16) = load_part<E>(src + r * ld * E, c * EPC, cols);
  }
}

// ------------------------------------------------------------------ launches
// Tile and slices for an m x n product over ksteps tiles of k, with `parts` products per output (2: gated):
// the least estimated time in microseconds. A CU's time for one tile of k of one workgroup is
//   idle + busy u     u: the part of the chip's slots taken over the call; the clock and the caches give way
//                     under load (256 x 256 tiles: 1.22 us at u = 0.59, 1.29 at 0.78, 1.46 at 1)
//   + alone           where every CU runs one workgroup: all wait for the same k from HBM, none fills in
//   + 0.06 cols       operands that lie by columns (by the tile's side)
// and fixed a workgroup's start and its outputs. 16-bit values are fitted with weights out of HBM, as a model's
// are (four to fourteen sets of operands in turn; 1700 and 2048 x 4096 x 4096 and 11008, 1700 x 11008 x 4096,
// 1700 x 5120 x 13824, 8192 x 4096 x 4096, 1700 x 2 (11008) x 4096): most within 5 %, single rounds of half a
// chip within 15 %. fp32: 2048 x 4096 x 64 and 1024, 4096 x 4096 x 1024, 5963 x 6240 x 128. Slices pay their
// partial sums' way through memory and the finishing launch (1700 x 4096 x 11008 in two 142 + 12 us, whole 162).
// Small tiles spread small products: 128 x 1024 -> 4096 takes 12.0 us in 128 x 128 tiles, 9.3 in 64 x 128, 7.4 in 64
// x 64 (fp32 65.7, 36.8, 21.3); 1024 x 4096 -> 4096 43.3, 50.5, 65.3.
// Few rows leave most of a 128-row tile's products empty, which fp32 pays for (4096 -> 4096, by columns: 20 rows
// 38.6 us, 24.0 in 64-row tiles, 19.6 in 32-row tiles).
// Not built: fp32 256 x 128 (two 128 x 128 tiles take 3.70 a step against 3.72) and 16-bit 32 x 128 (as many tiles as
// 64 x 128, a step of 0.38 + 0.16 u against 0.37 + 0.09 u): the estimate never takes them.
// Up to 32 rows run the few-rows kernel; more, 64 at a time, where that takes less than tiles with `pack`, the
// packing of their operands: all of x passes through every CU that has a workgroup, 16 rows of W at a time
// (16-bit 48 x 4096 -> 4096: 20.6 us against 16.8, with 4954 features, packed, 30.4 against 36.8; 512 x 512 -> 512
// 5.0 against 8.6; fp32 48 x 4954 -> 4096 56.9 against 80.9, 512 x 512 -> 512 7.5 against 18.1).
static Shape choose(int64_t m, int64_t n, int64_t ksteps, int parts, int dt, int cols, double pack = 0.0) {
  if (cols == 0 && m <= 32) return {0, 1};
  const int64_t cus = device_cu_count();
  struct Kind { int kind, bm, bn; double idle, busy, alone, fixed, step32, alone32, fixed32; };
  const Kind kinds[6] = {{1, 128, 128, 0.30, 0.20, 0.12, 3.0, 1.85, 0.15, 4.7}, {2, 256, 128, 0.46, 0.40, 0.10, 3.0, 0.0, 0.0, 0.0},
                         {3, 256, 256, 0.90, 0.56, 0.06, 6.0, 7.3, 0.0, 16.0}, {4, 64, 128, 0.25, 0.09, 0.12, 2.0, 0.95, 0.12, 3.2},
                         {5, 32, 128, 0.0, 0.0, 0.0, 0.0, 0.50, 0.45, 3.0}, {6, 64, 64, 0.16, 0.08, 0.19, 1.3, 0.47, 0.08, 2.5}};
  constexpr double START = 2.0;                        // of a tile launch beyond the few-rows kernel's
  Shape best{1, 1};
  double least = 1e300;
  if (cols == 0 && (m + 63) / 64 <= 65535) {           // blocks of rows are the grid's second dimension
    const int64_t rounds = ((n + 15) / 16 * ((m + 63) / 64) + cus - 1) / cus;
    const double rows = m < 64 ? (double)m : 64.0;
    least = (double)(rounds * ksteps) * (0.09 + 0.0044 * rows + 0.05 * (parts - 1)) + 1.5 - pack - START;
    best = {0, 1};
  }
  for (const Kind& q : kinds) {
    if ((dt == BCFFT_F32 ? q.step32 : q.idle) == 0.0) continue;          // not built for the type
    if ((q.kind == 4 && cols == 2) || (q.kind == 5 && (cols != 1 || m > 32)) || (q.kind == 6 && (cols == 2 || parts == 2))) continue;
    const int64_t tiles = ((m + q.bm - 1) / q.bm) * ((n * parts + q.bn - 1) / q.bn);
    for (int64_t kz = 1; kz <= 16 && (kz == 1 || ksteps / kz >= 4); ++kz) {
      const int64_t groups = tiles * kz;
      const int64_t per_cu = (groups + cus - 1) / cus;                   // the fullest CU's workgroups
      const double used = (double)groups / (double)(per_cu * cus);
      double step = dt == BCFFT_F32 ? q.step32 : q.idle + q.busy * used + 0.06 * cols * sqrt(q.bm * q.bn / 65536.0);
      if (per_cu == 1) step += dt == BCFFT_F32 ? q.alone32 : q.alone;
      double cost = (double)per_cu * ((double)((ksteps + kz - 1) / kz) * step + (dt == BCFFT_F32 ? q.fixed32 : q.fixed));
      if (kz > 1) cost += 6.0 + (double)(2 * kz) * m * n * parts * 4.0 / 5e6;
      if (cost < least) {
        least = cost;
        best = {q.kind, (int)kz};
      }
    }
  }
  return best;
}

static void launch_product(int dt, const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s) {
  if (dt == BCFFT_F32) launch_product_f32(a, layout, sh, s);
  else if (dt == BCFFT_F16) launch_product_f16(a, layout, sh, s);
  else launch_product_bf16(a, layout, sh, s);
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
static bool valid_stride(int64_t stride, int64_t features) { return stride >= features && stride <= (1 << 20); }
// rows start on 16 bytes, or are packed because their features are no whole number of 16-byte pieces
static bool aligned_stride(int64_t stride, int64_t rows, int64_t features, int dt) {
  return rows <= 1 || stride * elem(dt) % 16 == 0 || features * elem(dt) % 16 != 0;
}
static int64_t partial_bytes(int64_t m, int64_t n, Shape sh) { return sh.kz > 1 ? round16((int64_t)sh.kz * m * n * 4) : 0; }
// elements of a row padded to whole 16-byte pieces
static int64_t padded(int64_t cols, int dt) { return round16(cols * elem(dt)) / elem(dt); }
static bool whole(int64_t cols, int dt) { return cols * elem(dt) % 16 == 0; }
static int64_t packed_bytes(int64_t rows, int64_t cols, int dt) { return rows * round16(cols * elem(dt)); }
static const void* pack(int dt, const void* src, int64_t ld, int64_t rows, int64_t cols, char*& ws, hipStream_t s) {
  const int64_t total = rows * padded(cols, dt) * elem(dt) / 16;
  const unsigned blocks = (unsigned)((total + 255) / 256 < 16384 ? (total + 255) / 256 : 16384);
  if (elem(dt) == 4) hipLaunchKernelGGL(bc_dense_pack_kernel<4>, dim3(blocks), dim3(256), 0, s, (const char*)src, ld, rows, cols, ws);
  else hipLaunchKernelGGL(bc_dense_pack_kernel<2>, dim3(blocks), dim3(256), 0, s, (const char*)src, ld, rows, cols, ws);
  const void* at = ws;
  ws += packed_bytes(rows, cols, dt);
  return at;
}

struct ForwardPlan {
  Shape shape;
  bool packed;                                         // x and the weights are copied to 16-byte rows
  int64_t pack_bytes, total;
};
static ForwardPlan forward_plan(int64_t n, int64_t k, int64_t m, int dt, int parts) {
  ForwardPlan p;
  // two launches, and the operands read and written once more
  const double pack = whole(k, dt) ? 0.0 : 5.0 + (double)(2 * packed_bytes(n + parts * m, k, dt)) / 4.6e6;
  p.shape = choose(n, m, ksteps(k, dt), parts, dt, 0, pack);
  p.packed = p.shape.kind != 0 && !whole(k, dt);       // the few-rows kernel reads any address
  p.pack_bytes = p.packed ? packed_bytes(n + parts * m, k, dt) : 0;
  p.total = p.pack_bytes + partial_bytes(n, parts * m, p.shape);
  return p;
}
struct BackwardPlan {                                  // workspace of a backward call, in this order
  Shape dx, dw;
  int64_t dz_bytes, part_bytes, slices, pack_bytes, total;
  int rows;
};
static BackwardPlan backward_plan(int64_t n, int64_t k, int64_t m, int dt, int parts, int act) {
  BackwardPlan p;
  const bool split = parts == 2 && !whole(m, dt);      // dg and du are not adjacent columns
  p.dx = choose(n, k, parts * ksteps(m, dt), 1, dt, 1);
  p.dw = n <= 32 ? Shape{0, 1} : choose(split ? m : parts * m, k, ksteps(n, dt), 1, dt, 2);
  p.dz_bytes = parts == 2 || act != BCFFT_ACT_NONE || !whole(m, dt) ? parts * packed_bytes(n, m, dt) : 0;
  // 64 rows per workgroup of dz where that makes four workgroups per CU, else 16 (2048 x 4096: 25 -> 18 us, 1362 x 448: 18 -> 6 us)
  p.rows = (n + 63) / 64 * ((m + 255) / 256) >= 4 * device_cu_count() ? 64 : 16;
  p.slices = (n + p.rows - 1) / p.rows;
  p.part_bytes = parts == 1 ? round16(p.slices * m * 4) : 0;
  p.pack_bytes = whole(k, dt) ? 0 : packed_bytes(n + parts * m, k, dt);
  const int64_t sx = partial_bytes(n, k, p.dx), sw = partial_bytes(split ? m : parts * m, k, p.dw);
  p.total = p.dz_bytes + p.part_bytes + p.pack_bytes + (sx > sw ? sx : sw);
  return p;
}

template <class F>
static void by_dtype(int dt, F&& f) {
  if (dt == BCFFT_F32) f(std::integral_constant<int, BCFFT_F32>());
  else if (dt == BCFFT_F16) f(std::integral_constant<int, BCFFT_F16>());
  else f(std::integral_constant<int, BCFFT_BF16>());
}

// The forwards share their operands' preparation; what differs is set by the caller
static int run_forward(int dt, DenseArgs a, const void* w1, const ForwardPlan& p, void* workspace, int64_t bytes,
                       hipStream_t s) {
  if (p.total > 0 && (!workspace || bytes < p.total)) return BCFFT_ERR_ARG;
  char* ws = (char*)workspace;
  a.b[1] = w1;
  a.segs = 1;
  a.am = a.m;
  a.bn = a.n;
  if (p.packed) {
    a.a[0] = pack(dt, a.a[0], a.lda, a.m, a.k, ws, s);
    a.b[0] = pack(dt, a.b[0], a.ldb, a.n, a.k, ws, s);
    if (w1) a.b[1] = pack(dt, w1, a.ldb, a.n, a.k, ws, s);
    a.k = a.lda = a.ldb = padded(a.k, dt);             // the padding is zero
  }
  a.ws = (float*)ws;
  a.kz = p.shape.kz;
  launch_product(dt, a, w1 ? DENSE_GLU : DENSE_ROWS, p.shape, s);
  return record_launch_status();
}

// dx = dz W, or dg Wg + du Wu with du `apart` elements behind dg; W's rows of kp elements
static void launch_dx(int dt, const void* dz, int64_t ldz, int64_t apart, const void* w0, const void* w1, int64_t n,
                      int64_t k, int64_t kp, int64_t m, Shape sh, void* dx, float* ws, hipStream_t s) {
  DenseArgs a{};
  a.a[0] = dz;
  a.a[1] = (const char*)dz + apart * elem(dt);
  a.b[0] = w0;
  a.b[1] = w1;
  a.lda = ldz;
  a.ldb = kp;
  a.k = m;
  a.segs = w1 ? 2 : 1;
  a.m = a.am = n;
  a.n = k;
  a.bn = kp;
  a.y = dx;
  a.ws = ws;
  a.kz = sh.kz;
  launch_product(dt, a, DENSE_ROWS_COLS, sh, s);
}
// dw[m][k] = sum over tokens of dz[token][m] x[token][k]; mp, kp: readable elements of their rows
static void launch_dw(int dt, const void* dz, int64_t ldz, int64_t mp, const void* x, int64_t ldx, int64_t kp, int64_t n,
                      int64_t k, int64_t m, Shape sh, void* dw, float* ws, hipStream_t s) {
  DenseArgs a{};
  a.a[0] = dz;
  a.b[0] = x;
  a.lda = ldz;
  a.ldb = ldx;
  a.k = n;
  a.segs = 1;
  a.m = m;
  a.am = mp;
  a.n = k;
  a.bn = kp;
  a.y = dw;
  a.ws = ws;
  a.kz = sh.kz;
  launch_product(dt, a, DENSE_COLS, sh, s);
}

}  // namespace bcfft

using namespace bcfft;

extern "C" {

int64_t bcfft_dense_workspace_bytes(int op, int64_t n_tokens, int64_t in_features, int64_t out_features, int dtype,
                                    int act) {
  if (!valid_dt(dtype) || !valid_sizes(n_tokens, in_features, out_features) || act < 0 || act > BCFFT_ACT_GELU) return -1;
  if (op < BCFFT_DENSE_LINEAR || op > BCFFT_DENSE_GLU_BACKWARD) return -1;
  if (n_tokens == 0) return 0;
  const int parts = op == BCFFT_DENSE_GLU || op == BCFFT_DENSE_GLU_BACKWARD ? 2 : 1;
  if (op == BCFFT_DENSE_LINEAR || op == BCFFT_DENSE_GLU) return forward_plan(n_tokens, in_features, out_features, dtype, parts).total;
  return backward_plan(n_tokens, in_features, out_features, dtype, parts, act).total;
}

int bcfft_dense_plan(int op, int product, int64_t n_tokens, int64_t in_features, int64_t out_features, int dtype, int* kind,
                     int* slices) {
  const int64_t n = n_tokens, k = in_features, m = out_features;
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n, k, m) || n == 0) return BCFFT_ERR_SHAPE;
  const bool backward = op == BCFFT_DENSE_LINEAR_BACKWARD || op == BCFFT_DENSE_GLU_BACKWARD;
  if (op < BCFFT_DENSE_LINEAR || op > BCFFT_DENSE_GLU_BACKWARD || product < 0 || product > (backward ? 1 : 0) || !kind || !slices)
    return BCFFT_ERR_ARG;
  const int parts = op == BCFFT_DENSE_GLU || op == BCFFT_DENSE_GLU_BACKWARD ? 2 : 1;
  Shape sh;
  if (backward) {
    const BackwardPlan p = backward_plan(n, k, m, dtype, parts, BCFFT_ACT_NONE);
    sh = product ? p.dw : p.dx;
  } else {
    sh = forward_plan(n, k, m, dtype, parts).shape;
  }
  *kind = sh.kind;
  *slices = sh.kz;
  return BCFFT_OK;
}

int bcfft_dense_linear(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                       int64_t out_features, const void* w, const void* bias, const void* residual, int64_t r_stride,
                       int act, void* y, float* z, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n_tokens, in_features, out_features) || !valid_stride(x_stride, in_features) ||
      (residual && r_stride < out_features))
    return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU) return BCFFT_ERR_ARG;
  if (n_tokens == 0) return BCFFT_OK;
  if (!x || !w || !y) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if (!aligned_to(x, 16) || !aligned_to(w, 16) || !aligned_stride(x_stride, n_tokens, in_features, dtype) ||
      !aligned_to(bias, e) || !aligned_to(residual, e) || !aligned_to(y, e) || !aligned_to(z, 4) || !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  DenseArgs a{};
  a.a[0] = x;
  a.b[0] = w;
  a.lda = x_stride;
  a.ldb = a.k = in_features;
  a.m = n_tokens;
  a.n = out_features;
  a.bias = bias;
  a.res = residual;
  a.ldr = r_stride;
  a.y = y;
  a.z = z;
  a.act = act;
  return run_forward(dtype, a, nullptr, forward_plan(n_tokens, in_features, out_features, dtype, 1), workspace,
                     workspace_bytes, (hipStream_t)stream);
}

int bcfft_dense_glu(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                    int64_t out_features, const void* w_gate, const void* w_up, int act, void* h, float* gu,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n_tokens, in_features, out_features) || !valid_stride(x_stride, in_features)) return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU) return BCFFT_ERR_ARG;
  if (n_tokens == 0) return BCFFT_OK;
  if (!x || !w_gate || !w_up || !h) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if (!aligned_to(x, 16) || !aligned_to(w_gate, 16) || !aligned_to(w_up, 16) ||
      !aligned_stride(x_stride, n_tokens, in_features, dtype) || !aligned_to(h, e) || !aligned_to(gu, 4) ||
      !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  DenseArgs a{};
  a.a[0] = x;
  a.b[0] = w_gate;
  a.lda = x_stride;
  a.ldb = a.k = in_features;
  a.m = n_tokens;
  a.n = out_features;
  a.y = h;
  a.z = gu;
  a.act = act;
  return run_forward(dtype, a, w_up, forward_plan(n_tokens, in_features, out_features, dtype, 2), workspace,
                     workspace_bytes, (hipStream_t)stream);
}

int bcfft_dense_linear_backward(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                                int64_t out_features, const void* w, const void* dy, int64_t dy_stride, const float* z,
                                int act, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  const int64_t n = n_tokens, k = in_features, m = out_features;
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n, k, m) || !valid_stride(x_stride, k) || !valid_stride(dy_stride, m)) return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU || n == 0) return BCFFT_ERR_ARG;
  if (!dy || (act != BCFFT_ACT_NONE && !z) || (dx && !w) || (dw && !x)) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if ((dw && (!aligned_to(x, 16) || !aligned_stride(x_stride, n, k, dtype))) || (dx && !aligned_to(w, 16)) ||
      !aligned_to(dy, 16) || !aligned_stride(dy_stride, n, m, dtype) || !aligned_to(z, 4) || !aligned_to(dx, e) ||
      !aligned_to(dw, e) || !aligned_to(db, e) || !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  const BackwardPlan p = backward_plan(n, k, m, dtype, 1, act);
  if (p.total > 0 && (!workspace || workspace_bytes < p.total)) return BCFFT_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  void* dz = p.dz_bytes ? ws : nullptr;                // dy itself where it needs neither slope nor padding
  float* part = (float*)(ws + p.dz_bytes);
  ws += p.dz_bytes + p.part_bytes;
  const int64_t mp = padded(m, dtype), kp = padded(k, dtype);
  if ((dz && (dx || dw)) || db) {
    const DzArgs d{dy, dy_stride, act != BCFFT_ACT_NONE ? z : nullptr, dx || dw ? dz : nullptr, mp, db ? part : nullptr,
                   n, m, act, p.rows};
    by_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL(bc_dense_dz_kernel<dt.value>, dim3((unsigned)p.slices, (unsigned)((m + 255) / 256)), dim3(256), 0, s, d);
      if (db)
        hipLaunchKernelGGL(bc_dense_db_kernel<dt.value>, dim3((unsigned)((m + 31) / 32)), dim3(256), 0, s, part, p.slices, m, db);
    });
  }
  const void* g = dz ? dz : dy;
  const int64_t ldg = dz ? mp : dy_stride;
  const bool packed = p.pack_bytes > 0;
  const void* wp = packed && dx ? pack(dtype, w, k, m, k, ws, s) : w;
  const bool xpacked = packed && p.dw.kind != 0;       // few tokens' weight gradient reads any address
  const void* xp = xpacked && dw ? pack(dtype, x, x_stride, n, k, ws, s) : x;
  if (dx) launch_dx(dtype, g, ldg, 0, wp, nullptr, n, k, packed ? kp : k, m, p.dx, dx, (float*)ws, s);
  if (dw) launch_dw(dtype, g, ldg, dz ? mp : m, xp, xpacked ? kp : x_stride, xpacked ? kp : k, n, k, m, p.dw, dw, (float*)ws, s);
  return record_launch_status();
}

int bcfft_dense_glu_backward(const void* x, int dtype, int64_t n_tokens, int64_t x_stride, int64_t in_features,
                             int64_t out_features, const void* w_gate, const void* w_up, const void* dh,
                             int64_t dh_stride, const float* gu, int act, void* dx, void* dw, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const int64_t n = n_tokens, k = in_features, m = out_features;
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (!valid_sizes(n, k, m) || 2 * m > (1 << 20) || !valid_stride(x_stride, k) || dh_stride < m) return BCFFT_ERR_SHAPE;
  if (act < 0 || act > BCFFT_ACT_GELU || n == 0) return BCFFT_ERR_ARG;
  if (!dh || !gu || (dx && (!w_gate || !w_up)) || (dw && !x)) return BCFFT_ERR_ARG;
  const int e = elem(dtype);
  if ((dw && (!aligned_to(x, 16) || !aligned_stride(x_stride, n, k, dtype))) ||
      (dx && (!aligned_to(w_gate, 16) || !aligned_to(w_up, 16))) || !aligned_to(dh, e) || !aligned_to(gu, 4) ||
      !aligned_to(dx, e) || !aligned_to(dw, e) || !aligned_to(workspace, 16))
    return BCFFT_ERR_ALIGN;
  const BackwardPlan p = backward_plan(n, k, m, dtype, 2, act);
  if (!workspace || workspace_bytes < p.total) return BCFFT_ERR_ARG;
  if (!dx && !dw) return BCFFT_OK;
  hipStream_t s = (hipStream_t)stream;
  char* dz = (char*)workspace;
  char* ws = dz + p.dz_bytes + p.part_bytes;
  const int64_t mp = padded(m, dtype), kp = padded(k, dtype);
  const DzArgs d{dh, dh_stride, gu, dz, 2 * mp, nullptr, n, m, act, 0};
  const int64_t quads = (m + 3) / 4 * n;
  const unsigned blocks = (unsigned)((quads + 255) / 256 < 65536 ? (quads + 255) / 256 : 65536);
  by_dtype(dtype, [&](auto dt) { hipLaunchKernelGGL(bc_dense_dgu_kernel<dt.value>, dim3(blocks), dim3(256), 0, s, d); });
  const bool packed = p.pack_bytes > 0;
  const void* wgp = packed && dx ? pack(dtype, w_gate, k, m, k, ws, s) : w_gate;
  const void* wup = packed && dx ? pack(dtype, w_up, k, m, k, ws, s) : w_up;
  const bool xpacked = packed && p.dw.kind != 0;       // few tokens' weight gradient reads any address
  const void* xp = xpacked && dw ? pack(dtype, x, x_stride, n, k, ws, s) : x;
  const int64_t ldx = xpacked ? kp : x_stride, kr = xpacked ? kp : k;
  if (dx) launch_dx(dtype, dz, 2 * mp, mp, wgp, wup, n, k, packed ? kp : k, m, p.dx, dx, (float*)ws, s);
  if (dw && mp == m) {
    launch_dw(dtype, dz, 2 * mp, 2 * mp, xp, ldx, kr, n, k, 2 * m, p.dw, dw, (float*)ws, s);
  } else if (dw) {
    launch_dw(dtype, dz, 2 * mp, mp, xp, ldx, kr, n, k, m, p.dw, dw, (float*)ws, s);
    launch_dw(dtype, dz + mp * e, 2 * mp, mp, xp, ldx, kr, n, k, m, p.dw, (char*)dw + m * k * e, (float*)ws, s);
  }
  return record_launch_status();
}

}  // extern "C"
