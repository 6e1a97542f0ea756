// bcfft_distill.hip — distillation from a teacher's top logits: the teacher's k largest logits per row
// (bc_topk_logits_kernel) and the KL divergence from them to a student's softmax, forward and backward
// (bc_distill_kernel, bc_distill_backward_kernel). The teacher cache and loss of calibrate_bc.py:192-299
// in compressed form.
//
// Per row, T the temperature, t_j and i_j the teacher's k entries, rest the log of the teacher's mass
// outside them (or none), s the student's logits:
//   P = softmax([t_1/T .. t_k/T, rest]),  q = softmax(s / T),  q_rest = sum of q outside the i_j
//   loss = w (sum_j P_j (log P_j - log q_{i_j}) + P_rest (log P_rest - log q_rest))
//   dloss/ds_v = (w g / T) (q_v - sum_{j: i_j = v} P_j)   for v among the i_j
//                (w g / T) (q_v - P_rest q_v / q_rest)    else
//
// One workgroup per row. Bound by HBM: a row is read once, into registers (HOLD 16-byte pieces per
// thread, up to 131072 16-bit logits), and every further pass (maxima, sums, gradients) runs on them;
// longer rows are read again, out of L2 / the memory-side cache. A 1024-thread workgroup may use 128
// VGPRs per thread, 64 of them hold the row, so two workgroups of 512 threads (32000 16-bit logits)
// share a CU and one's arithmetic runs under the other's loads.
//
// The loss is a small difference of logarithms: a thread's part of a sum is kept in fp32 (at most a few
// hundred terms of one sign), the sums over threads, the teacher's softmax and the logarithms in fp64.
#include "bcfft_device.h"

#include <type_traits>

namespace bcfft {

constexpr int TOPK_MAX = 1024;          // entries per row
constexpr int TOPK_CAND = 2048;         // candidates ranked in LDS
constexpr int DISTILL_VOCAB_MAX = 1 << 18;   // the entries' bitmap: 32 KB of LDS

// exp(x / T) as exp2(x c + x lo): c + lo = log2(e) / T to 48 bits, so the constant's own rounding
// (up to 3e-8 relative, times x: the same sign in every term) does not shift the whole sum.
// c is rounded down and lo > 0: for x = -inf both products are -inf, never inf - inf.
struct ExpScale {
  float c, lo;
};
__device__ __forceinline__ float exp_scaled(float x, ExpScale e) {
  return __builtin_amdgcn_exp2f(fmaf(x, e.c, x * e.lo));
}

template <int DT> struct RowType {
  static constexpr int VEC = 8;        // elements per 16 bytes
};
template <> struct RowType<BCFFT_F32> {
  static constexpr int VEC = 4;
};

// 16 bytes at any element-aligned address (gfx950 serves unaligned global accesses)
template <int DT>
struct __attribute__((packed, aligned(DT == BCFFT_F32 ? 4 : 2))) Raw16 {
  uint32_t w[4];
};
template <int DT>
__device__ __forceinline__ uint4 load16(const void* row, int64_t at) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  const Raw16<DT> r = *reinterpret_cast<const Raw16<DT>*>((const char*)row + at * E);
  return make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
}
template <int DT>
__device__ __forceinline__ void unpack(uint4 u, float (&v)[RowType<DT>::VEC]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == BCFFT_F32) {
      v[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = unpack16<DT>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
// The row as every pass sees it: HOLD whole 16-byte pieces per thread in registers, or (HOLD = 0) read
// again; the elements behind the last whole piece one per thread. The held pieces' loads have no branch
// between them (past the end they repeat the last piece, unused), so all are in flight together.
template <int DT, int NT, int HOLD>
struct Row {
  static constexpr int VEC = RowType<DT>::VEC;
  uint4 held[HOLD > 0 ? HOLD : 1];
  const void* row;
  int64_t pieces;
  int tail;
  float last;

  __device__ __forceinline__ void open(const void* r, int64_t vocab) {
    row = r;
    pieces = vocab / VEC;
    tail = (int)(vocab - pieces * VEC);
    if constexpr (HOLD > 0) {
      if (pieces > 0) {
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
          const int p = i * NT + (int)threadIdx.x;
          held[i] = load16<DT>(row, (p < (int)pieces ? p : (int)pieces - 1) * VEC);
        }
      }
    }
    if ((int)threadIdx.x < tail) last = load_scalar(row, pieces * VEC + threadIdx.x, DT);
  }
  // f(first element's index, values): float[VEC] of a piece, float[1] behind the last one
  template <class F>
  __device__ __forceinline__ void each(F&& f) {
    if constexpr (HOLD > 0) {
#pragma unroll
      for (int i = 0; i < HOLD; ++i) {
        const int p = i * NT + (int)threadIdx.x;
        if (p < (int)pieces) {
          uint4 h = held[i];             // opaque: each pass widens its own values instead of keeping an
          asm volatile("" : "+v"(h.x), "+v"(h.y), "+v"(h.z), "+v"(h.w));   // earlier pass's (2x the registers)
          float v[VEC];
          unpack<DT>(h, v);
          f(p * VEC, v);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      for (int64_t p = threadIdx.x; p < pieces; p += NT) {
        float v[VEC];
        unpack<DT>(load16<DT>(row, p * VEC), v);
        f((int)(p * VEC), v);
      }
    }
    if ((int)threadIdx.x < tail) {
      float v[1] = {last};
      f((int)(pieces * VEC) + (int)threadIdx.x, v);
    }
  }
};
template <class A> constexpr int count_of = (int)(sizeof(std::remove_reference_t<A>) / sizeof(float));

// ------------------------------------------------------------------ reductions over the workgroup
template <class T, class OP>
__device__ __forceinline__ T wave_reduce(T v, OP op) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d, 64));
  return v;
}
struct MaxOp {
  // a NaN on either side stays
  template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a > b || a != a ? a : b; }
};
struct SumOp {
  template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
// every thread gets the result, added up in a fixed order; `red` holds NT / 64 values and is free
// again after the caller's next barrier
template <int NT, class T, class OP>
__device__ __forceinline__ T block_reduce(T v, T* red, OP op) {
  v = wave_reduce(v, op);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  T r = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r = op(r, red[i]);
  return r;
}

// ------------------------------------------------------------------ the teacher's top logits
// Order: larger logit first, NaN before everything, -0 equal to 0, equal logits by lower index: a
// 64-bit key with the logit's order-preserving bits above the inverted index, unique per element.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t full_key(uint32_t key, int at) { return (uint64_t)key << 32 | ~(uint32_t)at; }
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 1. Each thread's largest key; the k-th largest of these NT keys bounds the k-th largest element from
//    below (k threads hold at least one element that large each), and hardly more than k elements
//    reach it (74 for k = 64 of 256 threads, evenly spread). Its upper 16 bits are enough.
// 2. The elements at or above the bound go to LDS; each counts the candidates above it: its rank is its
//    place in the output. Ranks depend on keys alone, so the order of arrival does not matter.
// 3. The others' maximum and sum give rest.
// If more than TOPK_CAND elements reach the bound (long runs of equal logits), the k-th key itself is
// found bit by bit, by counting over the whole row.
template <int DT, int NT, int HOLD>
__global__ __launch_bounds__(NT) void bc_topk_logits_kernel(const void* __restrict__ logits, int64_t vocab,
                                                            int64_t row_stride, int k, ExpScale es, double inv_t,
                                                            void* __restrict__ values, int32_t* __restrict__ indices,
                                                            float* __restrict__ rest) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  __shared__ uint64_t cand[TOPK_CAND];
  __shared__ float left[TOPK_CAND];
  __shared__ uint32_t tmax[NT];
  __shared__ uint32_t redu[NT / 64];
  __shared__ float redf[NT / 64];
  __shared__ double redd[NT / 64];
  __shared__ int count, bound_s;
  const int tid = threadIdx.x;
  const int64_t n = blockIdx.x;
  const char* row = (const char*)logits + n * row_stride * E;
  Row<DT, NT, HOLD> r;
  r.open(row, vocab);

  uint32_t best = 0;                     // below every key of a number
  r.each([&](int, auto& v) {
    for (float x : v) {
      const uint32_t key = order_key(x);
      best = key > best ? key : best;
    }
  });
  tmax[tid] = best;
  if (tid == 0) count = 0;
  __syncthreads();
  if (tid < 64) {                        // largest b with k thread maxima whose upper halves reach it
    uint32_t mine[NT / 64];
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) mine[i] = tmax[i * 64 + tid] >> 16;
    uint32_t b = 0;
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t trial = b | 1u << bit;
      int c = 0;
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) c += __popcll(__ballot(mine[i] >= trial));
      if (c >= k) b = trial;
    }
    if (tid == 0) bound_s = (int)b;
  }
  __syncthreads();
  const uint32_t bound = (uint32_t)bound_s << 16;

  // candidates: key > cut_key, or key == cut_key at an index up to cut_index
  uint32_t cut_key = bound;
  int cut_index = 0x7fffffff;
  float below = -INFINITY;               // largest logit that is no candidate
  auto gather = [&]() {
    r.each([&](int at, auto& v) {
#pragma unroll
      for (int j = 0; j < count_of<decltype(v)>; ++j) {
        const uint32_t key = order_key(v[j]);
        if (key > cut_key || (key == cut_key && at <= cut_index - j)) {
          const int p = atomicAdd(&count, 1);
          if (p < TOPK_CAND) cand[p] = full_key(key, at + j);
        } else {
          below = fmaxf(below, v[j]);
        }
      }
    });
    __syncthreads();
  };
  gather();
  int m = count;
  if (m > TOPK_CAND) {                   // uniform over the workgroup
    // the k-th largest logit's key, and how many of its equals belong to the k
    auto count_over = [&](auto&& test) {
      uint32_t c = 0;
      r.each([&](int at, auto& v) {
#pragma unroll
        for (int j = 0; j < count_of<decltype(v)>; ++j) c += test(order_key(v[j]), at, j);
      });
      return (int64_t)block_reduce<NT>(c, redu, SumOp());
    };
    uint32_t kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = kth | 1u << bit;
      if (count_over([&](uint32_t key, int, int) { return key >= trial; }) >= k) kth = trial;
    }
    const int64_t equals = k - count_over([&](uint32_t key, int, int) { return key > kth; });
    int before = -1;                     // largest index that fewer than `equals` of them come up to
    for (int bit = 30; bit >= 0; --bit) {
      const int trial = before + (1 << bit);
      if (trial < 0) continue;
      if (count_over([&](uint32_t key, int at, int j) { return key == kth && at <= trial - j; }) < equals) before = trial;
    }
    cut_key = kth;
    cut_index = before + 1;
    below = -INFINITY;
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    gather();                            // exactly k of them
    m = k;
  }

  float top_left = -INFINITY;            // largest logit among the candidates that are not taken
  for (int i = tid; i < m; i += NT) {
    const uint64_t mine = cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < m; ++j) rank += cand[j] > mine;
    const uint32_t at = ~(uint32_t)mine;
    if (rank < k) {
      if constexpr (DT == BCFFT_F32) ((uint32_t*)values)[n * k + rank] = ((const uint32_t*)row)[at];
      else ((uint16_t*)values)[n * k + rank] = ((const uint16_t*)row)[at];
      indices[n * k + rank] = (int32_t)at;
    } else {
      const float v = key_value((uint32_t)(mine >> 32));
      left[rank] = v;
      top_left = fmaxf(top_left, v);
    }
  }
  const float mr = block_reduce<NT>(fmaxf(below, top_left), redf, MaxOp());
  const float ref = mr == -INFINITY ? 0.f : mr;
  float s = 0.f;
  r.each([&](int at, auto& v) {
#pragma unroll
    for (int j = 0; j < count_of<decltype(v)>; ++j) {
      const uint32_t key = order_key(v[j]);
      const bool taken = key > cut_key || (key == cut_key && at <= cut_index - j);
      s += taken ? 0.f : exp_scaled(v[j] - ref, es);
    }
  });
  for (int i = k + tid; i < m; i += NT) s += exp_scaled(left[i] - ref, es);
  const double sum = block_reduce<NT>((double)s, redd, SumOp());
  if (tid == 0) rest[n] = (float)((double)ref * inv_t + log(sum));      // log 0 = -inf: nothing left
}

// ------------------------------------------------------------------ the student's loss and gradient
struct DistillArgs {
  const void* logits;
  int64_t vocab, row_stride;
  const void* values;                    // teacher's entries (N, k), dtype vdt
  const void* indices;                   // (N, k), 32 or 64 bits; out of [0, vocab): no entry
  const float* rest;                     // (N) or null
  const float* weight;                   // (N) or null
  const float* upstream;                 // (N), backward
  float* loss;                           // (N)
  float* stats;                          // (N, 4): what the backward needs of the row's sums, or null
  void* grad;                            // (N, vocab) contiguous
  int k, vdt, idx64;
  ExpScale es;
  double inv_t;
};

// LDS of a row's entries, behind them the bitmap of the vocabulary
struct Entries {
  double p[TOPK_MAX];                    // teacher's logit over T, then its probability
  float s[TOPK_MAX];                     // student's logit
  int32_t at[TOPK_MAX];                  // index, or -1
  double redd[16];
  float redf[16];
  int dup;
};

// Loads the entries, sets the bitmap, computes the teacher's softmax: p[j] = exp(a_j - am) and their
// sum; false where the row has no mass to learn from. `am` and `total` come back in every thread.
template <int DT, int NT>
__device__ __forceinline__ bool teacher_softmax(const DistillArgs& a, int64_t n, const char* row, Entries& en,
                                                uint32_t* bits, double& am, double& total, double& rest_p) {
  const int tid = threadIdx.x;
  for (int64_t w = tid; w < (a.vocab + 31) / 32; w += NT) bits[w] = 0;
  if (tid == 0) en.dup = 0;
  __syncthreads();
  double mx = -INFINITY;
  for (int j = tid; j < a.k; j += NT) {
    const int64_t e = n * a.k + j;
    const int64_t at = a.idx64 ? ((const int64_t*)a.indices)[e] : (int64_t)((const int32_t*)a.indices)[e];
    const bool ok = at >= 0 && at < a.vocab;
    const double t = ok ? (double)load_scalar(a.values, e, a.vdt) * a.inv_t : -INFINITY;
    en.at[j] = ok ? (int32_t)at : -1;
    en.p[j] = t;
    en.s[j] = ok ? load_scalar(row, at, DT) : -INFINITY;
    if (ok && (atomicOr(&bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1)) en.dup = 1;
    mx = t > mx || t != t ? t : mx;      // NaN stays: it makes the row NaN, as in a softmax
  }
  const double rest = a.rest ? (double)a.rest[n] : -INFINITY;
  mx = rest > mx || rest != rest ? rest : mx;
  mx = block_reduce<NT>(mx, en.redd, MaxOp());
  am = mx;
  if (mx == -INFINITY) return false;     // (a NaN among the terms below makes the sum NaN)
  double sum = 0.0;
  for (int j = tid; j < a.k; j += NT) {
    const double p = en.at[j] >= 0 ? exp(en.p[j] - mx) : 0.0;
    sum += p;
  }
  rest_p = a.rest ? exp(rest - mx) : 0.0;
  total = block_reduce<NT>(sum, en.redd, SumOp()) + rest_p;
  rest_p /= total;
  return true;
}

// 1 where entry j is the first with its index; mass: the probability of all entries with that index
template <int NT>
__device__ __forceinline__ bool first_of(const Entries& en, int k, int j, double& mass) {
  if (!en.dup) return true;
  const int at = en.at[j];
  double m = 0.0;
  int first = j;
  for (int i = 0; i < k; ++i) {
    if (en.at[i] == at) {
      m += en.p[i];
      if (i < first) first = i;
    }
  }
  mass = m;
  return first == j;
}

// v as the output's type: 16 bytes at an element-aligned address, or one element
template <int DT>
__device__ __forceinline__ void store_one(void* row, int64_t at, float v) {
  if constexpr (DT == BCFFT_F32) ((float*)row)[at] = v;
  else ((uint16_t*)row)[at] = (uint16_t)pack16<DT>(v, 0.f);
}
template <int DT, int N>
__device__ __forceinline__ void store_piece(void* row, int64_t at, const float (&v)[N]) {
  if constexpr (N == 1) {
    store_one<DT>(row, at, v[0]);
  } else {
    Raw16<DT> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == BCFFT_F32) o.w[i] = __float_as_uint(v[i]);
      else o.w[i] = pack16<DT>(v[2 * i], v[2 * i + 1]);
    }
    *reinterpret_cast<Raw16<DT>*>((char*)row + at * (DT == BCFFT_F32 ? 4 : 2)) = o;
  }
}

// the bits of elements `at` .. `at + N` of one piece
template <int N>
__device__ __forceinline__ uint32_t piece_bits(const uint32_t* bits, int at) {
  return bits[at >> 5] >> (at & 31) & ((1u << N) - 1);
}

// The whole gradient row: elements outside the entries are exp(x / T) times `coef` (0 where the entry
// sits, written after), then the entries. The wait makes the pieces' stores complete (acknowledged by
// L2) before other waves of the workgroup store the entries into the same lines.
template <int DT, int NT, class ROW>
__device__ __forceinline__ void write_gradient(const DistillArgs& a, int64_t n, ROW& r, Entries& en,
                                               const uint32_t* bits, float ref, float coef, float m_all,
                                               float inv_s, double total, float scale) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  char* out = (char*)a.grad + n * a.vocab * E;
  const float c = coef * scale;
  r.each([&](int at, auto& v) {
    constexpr int N = count_of<decltype(v)>;
    const uint32_t b = piece_bits<N>(bits, at);
    float g[N];
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = b >> j & 1 ? 0.f : exp_scaled(v[j] - ref, a.es) * c;
    store_piece<DT>(out, at, g);
  });
  wait_vmcnt<0>();
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += NT) {
    if (en.at[j] < 0) continue;
    double mass = en.p[j];
    if (!first_of<NT>(en, a.k, j, mass)) continue;
    const float q = exp_scaled(en.s[j] - m_all, a.es) * inv_s;
    store_one<DT>(out, en.at[j], (q - (float)(mass / total)) * scale);
  }
}

template <int DT, int NT>
__device__ __forceinline__ void write_zero(const DistillArgs& a, int64_t n) {
  constexpr int VEC = RowType<DT>::VEC;
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  char* out = (char*)a.grad + n * a.vocab * E;
  const float z[VEC] = {};
  const int64_t pieces = a.vocab / VEC, end = pieces * VEC + threadIdx.x;
  for (int64_t p = threadIdx.x; p < pieces; p += NT) store_piece<DT>(out, p * VEC, z);
  if (end < a.vocab) store_one<DT>(out, end, 0.f);
}

// Loss of a row and, with GRAD, its gradient, in one read of the row. The sums are kept apart: the
// entries' relative to their largest logit, the others' relative to theirs, so that neither underflows
// whatever lies between them.
template <int DT, int NT, int HOLD, bool GRAD>
__global__ __launch_bounds__(NT) void bc_distill_kernel(DistillArgs a) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  __shared__ Entries en;
  extern __shared__ uint32_t bits[];
  using ROW = Row<DT, NT, HOLD>;
  const int tid = threadIdx.x;
  const int64_t n = blockIdx.x;
  const float w = a.weight ? a.weight[n] : 1.f;
  const char* row = (const char*)a.logits + n * a.row_stride * E;
  double am = 0.0, total = 1.0, rest_p = 0.0;
  ROW r;
  bool live = w != 0.f;                  // uniform: a row of weight 0 is not read
  if (live) {
    r.open(row, a.vocab);
    live = teacher_softmax<DT, NT>(a, n, row, en, bits, am, total, rest_p);
  }
  if (!live) {
    if (tid == 0) {
      a.loss[n] = 0.f;
      if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * n) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if constexpr (GRAD) write_zero<DT, NT>(a, n);
    return;
  }
  // maxima of the two parts
  float mo = -INFINITY, me = -INFINITY;
  r.each([&](int at, auto& v) {
    constexpr int N = count_of<decltype(v)>;
    const uint32_t b = piece_bits<N>(bits, at);
#pragma unroll
    for (int j = 0; j < N; ++j) mo = fmaxf(mo, b >> j & 1 ? -INFINITY : v[j]);
  });
  for (int j = tid; j < a.k; j += NT) me = fmaxf(me, en.s[j]);
  mo = block_reduce<NT>(mo, en.redf, MaxOp());
  me = block_reduce<NT>(me, en.redf, MaxOp());
  const float ro = mo == -INFINITY ? 0.f : mo, re = me == -INFINITY ? 0.f : me;
  // their sums, and the loss's part that is linear in the logits
  float so = 0.f;
  r.each([&](int at, auto& v) {
    constexpr int N = count_of<decltype(v)>;
    const uint32_t b = piece_bits<N>(bits, at);
#pragma unroll
    for (int j = 0; j < N; ++j) so += b >> j & 1 ? 0.f : exp_scaled(v[j] - ro, a.es);
  });
  double se = 0.0, lin = 0.0;
  for (int j = tid; j < a.k; j += NT) {
    if (en.at[j] < 0) continue;
    const double t = en.p[j] - am, p = exp(t), x = ((double)en.s[j] - (double)re) * a.inv_t;
    en.p[j] = p;                         // (read again by first_of, after a barrier)
    if (p > 0.0) lin += p * (t - x);
    else if (p != p) lin = p;
  }
  const double sum_o = block_reduce<NT>((double)so, en.redd, SumOp());
  for (int j = tid; j < a.k; j += NT) {
    double mass;
    if (en.at[j] >= 0 && first_of<NT>(en, a.k, j, mass)) se += exp(((double)en.s[j] - (double)re) * a.inv_t);
  }
  const double sum_e = block_reduce<NT>(se, en.redd, SumOp());
  lin = block_reduce<NT>(lin, en.redd, SumOp()) / total;
  const float m_top = fmaxf(mo, me), m_all = m_top == -INFINITY ? 0.f : m_top;
  const double fo = mo == -INFINITY ? 0.0 : (double)exp_scaled(mo - m_all, a.es);
  const double fe = me == -INFINITY ? 0.0 : (double)exp_scaled(me - m_all, a.es);
  const double sum = sum_o * fo + sum_e * fe;
  const float inv_s = (float)(1.0 / sum);
  const float coef = (float)(fo / sum - (rest_p != 0.0 && sum_o != 0.0 ? rest_p / sum_o : 0.0));
  if (tid == 0) {
    // lin holds sum_j P_j ((a_j - am) - (s_j - re) / T); the logarithms of both sums and the shift of
    // the student's reference from re to m_all complete it
    const double ls = log((mo == -INFINITY ? 0.0 : sum_o * exp(((double)mo - (double)m_all) * a.inv_t)) +
                          (me == -INFINITY ? 0.0 : sum_e * exp(((double)me - (double)m_all) * a.inv_t)));
    const double shift = ((double)re - (double)m_all) * a.inv_t;
    double loss = lin - (1.0 - rest_p) * shift + ls - log(total);
    if (rest_p != 0.0)
      loss += rest_p * (((double)a.rest[n] - am) - (((double)ro - (double)m_all) * a.inv_t + log(sum_o)));
    a.loss[n] = (float)loss * w;
    if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * n) = make_float4(ro, coef, m_all, inv_s);
  }
  if constexpr (GRAD) write_gradient<DT, NT>(a, n, r, en, bits, ro, coef, m_all, inv_s, total, (float)(w * a.inv_t));
}

// Gradient from the forward's sums: one read of the row, one write
template <int DT, int NT>
__global__ __launch_bounds__(NT) void bc_distill_backward_kernel(DistillArgs a) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  __shared__ Entries en;
  extern __shared__ uint32_t bits[];
  using ROW = Row<DT, NT, 0>;
  const int64_t n = blockIdx.x;
  const float w = a.weight ? a.weight[n] : 1.f;
  const char* row = (const char*)a.logits + n * a.row_stride * E;
  double am = 0.0, total = 1.0, rest_p = 0.0;
  if (w == 0.f || !teacher_softmax<DT, NT>(a, n, row, en, bits, am, total, rest_p)) {
    write_zero<DT, NT>(a, n);
    return;
  }
  for (int j = threadIdx.x; j < a.k; j += NT)
    if (en.at[j] >= 0) en.p[j] = exp(en.p[j] - am);
  const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * n);
  ROW r;
  r.open(row, a.vocab);
  write_gradient<DT, NT>(a, n, r, en, bits, st.x, st.y, st.z, st.w, total, (float)(w * a.inv_t) * a.upstream[n]);
}

// ------------------------------------------------------------------ launches
// log2(e) / T as c + lo with c rounded down and lo > 0
static ExpScale exp_scale(double temperature) {
  const double c = 1.4426950408889634 / temperature;
  float hi = (float)c;
  if ((double)hi >= c) hi = nextafterf(hi, 0.f);
  return {hi, (float)(c - (double)hi)};
}

// Threads and pieces per thread by the row's number of 16-byte pieces: the fewest threads that hold it
// with 8 pieces each (more rows per CU), then 16 pieces, then a row that is read again.
template <int DT, class F>
static void by_row(int64_t vocab, int64_t min_threads, F&& go) {
  const int64_t pieces = (vocab + RowType<DT>::VEC - 1) / RowType<DT>::VEC;
  using std::integral_constant;
  if (pieces <= 512 && min_threads <= 256) go(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (pieces <= 2048 && min_threads <= 256) go(integral_constant<int, 256>(), integral_constant<int, 8>());
  else if (pieces <= 4096 && min_threads <= 512) go(integral_constant<int, 512>(), integral_constant<int, 8>());
  else if (pieces <= 8192) go(integral_constant<int, 1024>(), integral_constant<int, 8>());
  else if (pieces <= 16384) go(integral_constant<int, 1024>(), integral_constant<int, 16>());
  else go(integral_constant<int, 1024>(), integral_constant<int, 0>());
}

template <int DT>
static void launch_topk_dt(const void* logits, int64_t n, int64_t vocab, int64_t row_stride, int k, double temperature,
                           void* values, int32_t* indices, float* rest, hipStream_t s) {
  by_row<DT>(vocab, k, [&](auto nt, auto hold) {
    hipLaunchKernelGGL((bc_topk_logits_kernel<DT, nt.value, hold.value>), dim3((unsigned)n), dim3(nt.value), 0, s,
                       logits, vocab, row_stride, k, exp_scale(temperature), 1.0 / temperature, values, indices, rest);
  });
}

template <int DT>
static void launch_distill_dt(const DistillArgs& a, int64_t n, hipStream_t s) {
  const unsigned lds = (unsigned)((a.vocab + 31) / 32 * 4);
  if (a.upstream) {
    hipLaunchKernelGGL((bc_distill_backward_kernel<DT, 512>), dim3((unsigned)n), dim3(512), lds, s, a);
    return;
  }
  by_row<DT>(a.vocab, 1, [&](auto nt, auto hold) {
    if (a.grad) hipLaunchKernelGGL((bc_distill_kernel<DT, nt.value, hold.value, true>), dim3((unsigned)n), dim3(nt.value), lds, s, a);
    else hipLaunchKernelGGL((bc_distill_kernel<DT, nt.value, hold.value, false>), dim3((unsigned)n), dim3(nt.value), lds, s, a);
  });
}
static int launch_distill(int dt, const DistillArgs& a, int64_t n, hipStream_t s) {
  if (dt == BCFFT_F32) launch_distill_dt<BCFFT_F32>(a, n, s);
  else if (dt == BCFFT_F16) launch_distill_dt<BCFFT_F16>(a, n, s);
  else launch_distill_dt<BCFFT_BF16>(a, n, s);
  return record_launch_status();
}

static bool valid_dt(int d) { return d == BCFFT_F32 || d == BCFFT_F16 || d == BCFFT_BF16; }
static bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
static int elem(int d) { return d == BCFFT_F32 ? 4 : 2; }
// sizes shared by the three entry points; n == 0 is served before
static int check_rows(int64_t n, int64_t vocab, int64_t row_stride, int k, double temperature, int64_t most) {
  if (n < 0 || n > 0x7fffffff || vocab < 1 || vocab > most || row_stride < vocab) return BCFFT_ERR_SHAPE;
  if (k < 1 || k > TOPK_MAX) return BCFFT_ERR_SHAPE;
  if (!(temperature >= 1e-6 && temperature <= 1e6)) return BCFFT_ERR_ARG;
  return BCFFT_OK;
}

}  // namespace bcfft

using namespace bcfft;

extern "C" {

int bcfft_topk_logits(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride, int k,
                      double temperature, void* values, int32_t* indices, float* rest, void* stream) {
  if (!valid_dt(dtype)) return BCFFT_ERR_DTYPE;
  if (int st = check_rows(n_rows, vocab, row_stride, k, temperature, 0x7fffffff)) return st;
  if (k > vocab) return BCFFT_ERR_SHAPE;
  if (n_rows == 0) return BCFFT_OK;
  if (!logits || !values || !indices || !rest) return BCFFT_ERR_ARG;
  if (!aligned_to(logits, elem(dtype)) || !aligned_to(values, elem(dtype)) || !aligned_to(indices, 4) || !aligned_to(rest, 4))
    return BCFFT_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == BCFFT_F32) launch_topk_dt<BCFFT_F32>(logits, n_rows, vocab, row_stride, k, temperature, values, indices, rest, s);
  else if (dtype == BCFFT_F16) launch_topk_dt<BCFFT_F16>(logits, n_rows, vocab, row_stride, k, temperature, values, indices, rest, s);
  else launch_topk_dt<BCFFT_BF16>(logits, n_rows, vocab, row_stride, k, temperature, values, indices, rest, s);
  return record_launch_status();
}

int bcfft_distill_topk(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                       const void* values, int values_dtype, const void* indices, int index_bytes, int k,
                       const float* rest, const float* weight, double temperature, float* loss, float* stats,
                       void* grad, void* stream) {
  if (!valid_dt(dtype) || !valid_dt(values_dtype)) return BCFFT_ERR_DTYPE;
  if (int st = check_rows(n_rows, vocab, row_stride, k, temperature, DISTILL_VOCAB_MAX)) return st;
  if (index_bytes != 4 && index_bytes != 8) return BCFFT_ERR_ARG;
  if (n_rows == 0) return BCFFT_OK;
  if (!logits || !values || !indices || !loss) return BCFFT_ERR_ARG;
  if (!aligned_to(logits, elem(dtype)) || !aligned_to(values, elem(values_dtype)) || !aligned_to(indices, index_bytes) ||
      !aligned_to(rest, 4) || !aligned_to(weight, 4) || !aligned_to(loss, 4) || !aligned_to(stats, 16) ||
      !aligned_to(grad, elem(dtype)))
    return BCFFT_ERR_ALIGN;
  const DistillArgs a{logits, vocab, row_stride, values, indices, rest, weight, nullptr, loss, stats, grad,
                      k, values_dtype, index_bytes == 8, exp_scale(temperature), 1.0 / temperature};
  return launch_distill(dtype, a, n_rows, (hipStream_t)stream);
}

int bcfft_distill_topk_backward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                                const void* values, int values_dtype, const void* indices, int index_bytes, int k,
                                const float* rest, const float* weight, double temperature, const float* stats,
                                const float* upstream, void* grad, void* stream) {
  if (!valid_dt(dtype) || !valid_dt(values_dtype)) return BCFFT_ERR_DTYPE;
  if (int st = check_rows(n_rows, vocab, row_stride, k, temperature, DISTILL_VOCAB_MAX)) return st;
  if (index_bytes != 4 && index_bytes != 8) return BCFFT_ERR_ARG;
  if (n_rows == 0) return BCFFT_OK;
  if (!logits || !values || !indices || !stats || !upstream || !grad) return BCFFT_ERR_ARG;
  if (!aligned_to(logits, elem(dtype)) || !aligned_to(values, elem(values_dtype)) || !aligned_to(indices, index_bytes) ||
      !aligned_to(rest, 4) || !aligned_to(weight, 4) || !aligned_to(upstream, 4) || !aligned_to(stats, 16) ||
      !aligned_to(grad, elem(dtype)))
    return BCFFT_ERR_ALIGN;
  const DistillArgs a{logits, vocab, row_stride, values, indices, rest, weight, upstream, nullptr, (float*)stats, grad,
                      k, values_dtype, index_bytes == 8, exp_scale(temperature), 1.0 / temperature};
  return launch_distill(dtype, a, n_rows, (hipStream_t)stream);
}

}  // extern "C"
