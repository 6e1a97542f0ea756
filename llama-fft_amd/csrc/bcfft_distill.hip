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
// One workgroup per row. A row is read once, into registers (HOLD 16-byte pieces per thread, up to 131072
// 16-bit logits); longer rows are read again, out of L2 / the memory-side cache. The floor is HBM: 3.2 us a
// CU for a row of 32000 16-bit logits read, 6.4 us read and written back. A CU serves 64 lane operations a
// clock (an exponential counts four), so a row's floor allows 14 (28) of them per logit: what the passes
// cost is counted beside them, and exponentials that the gradient needs again stay in registers.
//
// The loss is a small difference of logarithms: a thread's part of a sum is kept in fp32 for at most 128 terms
// of one sign and the element behind the last whole piece (longer rows add it to an fp64 sum as often), the sums
// over threads, the teacher's softmax and the logarithms in fp64.
#include "bcfft_device.h"

#include <type_traits>

namespace bcfft {

constexpr int TOPK_MAX = 1024;          // entries per row
constexpr int DISTILL_VOCAB_MAX = 1 << 18;   // the entries' bitmap: 32 KB of LDS

// exp((v - ref) / T) as exp2(x c + x lo), x = v - ref: c + lo = log2(e) / T to 48 bits, so the constant's own
// rounding (up to 3e-8 relative, times x: the same sign in every term) does not shift the sum. c is rounded
// down and lo > 0: for x = -inf both products are -inf, never inf - inf. The difference is taken first: with
// ref = the type's lowest value (a row masked by it alone) ref c would overflow.
struct ExpScale {
  float c, lo;
};
__device__ __forceinline__ float exp_at(float v, ExpScale e, float ref) {
  const float x = v - ref;
  return __builtin_amdgcn_exp2f(fmaf(x, e.c, x * e.lo));
}
// the same without lo, for sums whose terms lie near ref: what is left of the constant's rounding is at most
// as much as the argument's own
__device__ __forceinline__ float exp_near(float v, ExpScale e, float ref) { return __builtin_amdgcn_exp2f((v - ref) * e.c); }

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
// One thread's sum over the row, in fp32 with its registers where a row is held. A row that is read again has
// vocab / 1024 elements per thread (4096 of 2^22 logits: equal terms, whose roundings have one sign, were up to
// 5e-5 off): every 128 of them go to an fp64 sum.
template <int HOLD>
struct ThreadSum {
  float part = 0.f;
  double whole = 0.0;
  int terms = 0;
  __device__ __forceinline__ void operator+=(float e) { part += e; }
  template <int N>
  __device__ __forceinline__ void piece_done() {
    if constexpr (HOLD == 0) {
      terms += N;
      if (terms >= 128) {
        whole += (double)part;
        part = 0.f;
        terms = 0;
      }
    }
  }
  __device__ __forceinline__ double value() const { return HOLD == 0 ? whole + (double)part : (double)part; }
};
template <class A> constexpr int count_of = (int)(sizeof(std::remove_reference_t<A>) / sizeof(float));

// ------------------------------------------------------------------ reductions over the workgroup
// Lanes trade values inside the vector unit: by shuffles through LDS a sum of doubles over the workgroup takes
// 1600 clocks, so 500. Steps 1, 2: neighbours in groups of 4; 4, 8: a mirror image of 8, 16 lanes, whose halves
// each hold one value by then.
template <int STEP>
__device__ __forceinline__ uint32_t other_lane(uint32_t v) {
  constexpr int CTRL = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : STEP == 4 ? 0x141 : 0x140;
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int STEP, class T>
__device__ __forceinline__ T other(T v) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(T, (uint64_t)other_lane<STEP>((uint32_t)(b >> 32)) << 32 | other_lane<STEP>((uint32_t)b));
  } else {
    return __builtin_bit_cast(T, other_lane<STEP>(__builtin_bit_cast(uint32_t, v)));
  }
}
// over LANES <= 16 neighbouring lanes
template <int LANES, class T, class OP>
__device__ __forceinline__ T lanes_reduce(T v, OP op) {
  if constexpr (LANES > 1) v = op(v, other<1>(v));
  if constexpr (LANES > 2) v = op(v, other<2>(v));
  if constexpr (LANES > 4) v = op(v, other<4>(v));
  if constexpr (LANES > 8) v = op(v, other<8>(v));
  return v;
}
template <class T, class OP>
__device__ __forceinline__ T wave_reduce(T v, OP op) {
  v = lanes_reduce<16>(v, op);
  T w[4];                                // the four groups' results, the same in every lane
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if constexpr (sizeof(T) == 8) {
      const uint64_t b = __builtin_bit_cast(uint64_t, v);
      w[g] = __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 16 * g) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 16 * g));
    } else {
      w[g] = __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16 * g));
    }
  }
  return op(op(w[0], w[1]), op(w[2], w[3]));
}
struct MaxOp {
  // a NaN on either side stays
  template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a > b || a != a ? a : b; }
};
struct SumOp {
  template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
// the waves' results, joined by every wave for itself (lane i takes wave i's: one value per thread, where a
// loop over them would hold all)
template <int NT, class T, class OP>
__device__ __forceinline__ T across_waves(const T* red, OP op) {
  return lanes_reduce<NT / 64>(red[threadIdx.x & (NT / 64 - 1)], op);
}
// every thread gets the result, added up in a fixed order; `red` holds NT / 64 values and is free
// again after the caller's next barrier
template <int NT, class T, class OP>
__device__ __forceinline__ T block_reduce(T v, T* red, OP op) {
  v = wave_reduce(v, op);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return across_waves<NT>(red, op);
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

// 1. The largest logit of each thread (of 1024 threads: of each half of its pieces) or, for k <= 128, of each of
//    256 groups of threads: at least 2 k maxima. The k-th largest of them bounds the k-th largest element from
//    below (k groups hold at least one that large each), and hardly more than k elements reach it (74 for k = 64
//    of 256, evenly spread; but 900 for k = 249 of 256: 1609 x 2960 fp32 195 us, 51 with 512). Its upper 16 bits
//    are enough: one wave finds it bit by bit, by ballots over G / 64 maxima per lane (16 of them took 8000 of
//    the kernel's 29000 clocks at 20 x 32000, so there are no more than 4 where k allows it).
//                                                                                  1.5 operations a logit
// 2. The elements at or above the bound go to LDS, the others' exponentials relative to it are summed.    9
// 3. Each candidate counts the candidates above it: its rank is its place in the output. Ranks depend on
//    keys alone, so the order of arrival does not matter.
// If more than TOPK_CAND elements reach the bound (long runs of equal logits), the k-th key itself is
// found bit by bit, by counting over the whole row; if the sum under the bound vanishes in fp32 (a gap of
// 45 T below the bound), the others' own maximum takes the bound's place as its reference.
template <int DT, int NT, int HOLD>
__global__ __launch_bounds__(NT, NT == 512 ? 6 : 1) void bc_topk_logits_kernel(const void* __restrict__ logits, int64_t vocab,
                                                            int64_t row_stride, int k, ExpScale es, double inv_t,
                                                            void* __restrict__ values, int32_t* __restrict__ indices,
                                                            float* __restrict__ rest) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  constexpr int TOPK_CAND = NT == 256 ? 1024 : 2048;     // candidates ranked in LDS
  constexpr bool TWO = NT == 1024;
  constexpr int VEC = RowType<DT>::VEC, CHUNK = HOLD > 0 ? 64 / VEC : 1;    // pieces per 64-bit mask
  __shared__ int at_s[TOPK_CAND];        // the candidates: indices, as they come
  __shared__ uint64_t cand[TOPK_CAND];   // their keys
  __shared__ uint32_t raw[TOPK_CAND];    // their logits as they stand in the row
  __shared__ float left[TOPK_CAND];
  __shared__ uint32_t gmax[TWO ? 2 * NT : NT];
  __shared__ uint32_t redu[NT / 64];
  __shared__ float redf[NT / 64];
  __shared__ double redd[NT / 64];
  __shared__ int count, bound_s;
  const int tid = threadIdx.x;
  if (tid == 0) count = 0;
  const int64_t n = blockIdx.x;
  const char* row = (const char*)logits + n * row_stride * E;
  Row<DT, NT, HOLD> r;
  r.open(row, vocab);

  float best = -INFINITY, second = -INFINITY;        // NaN passes them by: it still is a candidate below
  int seen = 0;                          // pieces; with TWO the odd ones' maximum is kept apart
  r.each([&](int, auto& v) {
    float mx = v[0];
    if constexpr (count_of<decltype(v)> > 1) mx = fmaxf(mx, v[1]);
#pragma unroll
    for (int j = 2; j + 1 < count_of<decltype(v)>; j += 2) mx = fmaxf(fmaxf(mx, v[j]), v[j + 1]);
    if (TWO && (seen & 1)) second = fmaxf(second, mx);
    else best = fmaxf(best, mx);
    ++seen;
  });
  // 0 is below every key of a number
  const bool grouped = NT > 256 && k <= 128;
  uint32_t key = seen ? order_key(grouped ? fmaxf(best, second) : best) : 0;
  if (TWO && !grouped) gmax[NT + tid] = seen > 1 ? order_key(second) : 0;
  if (grouped) {
    key = lanes_reduce<NT / 256>(key, MaxOp());
    if (tid % (NT / 256) == 0) gmax[tid / (NT / 256)] = key;
  } else {
    gmax[tid] = key;
  }
  __syncthreads();
  if (tid < 64) {                        // largest b with k maxima whose upper halves reach it
    auto search = [&](auto per_lane) {
      uint32_t mine[per_lane.value];
#pragma unroll
      for (int i = 0; i < per_lane.value; ++i) mine[i] = gmax[i * 64 + tid] >> 16;
      uint32_t b = 0;
      for (int bit = 15; bit >= 0; --bit) {
        const uint32_t trial = b | 1u << bit;
        int c = 0;
#pragma unroll
        for (int i = 0; i < per_lane.value; ++i) c += __popcll(__ballot(mine[i] >= trial));
        if (c >= k) b = trial;
        if (c == k) break;               // exactly k: lower bits only raise the bound between two maxima
      }
      if (tid == 0) bound_s = (int)b;
    };
    if (grouped) search(std::integral_constant<int, 4>());
    else search(std::integral_constant<int, (TWO ? 2 : 1) * NT / 64>());
  }
  __syncthreads();
  // an element reaches the bound unless it is less: NaN does, and without a bound all do
  const uint32_t bound_key = (uint32_t)bound_s << 16;
  const float bound = bound_key ? key_value(bound_key) : -INFINITY;
  ThreadSum<HOLD> s;
  // one bit per logit of a thread that reaches the bound, listed after the pass: no branch in it
  uint64_t reach = 0;
  int bit = 0, first = tid;              // the next piece's bit, and the piece of bit 0
  auto list = [&]() {
    if (reach) {
      int p = atomicAdd(&count, __popcll(reach));
      for (; reach; reach &= reach - 1, ++p) {
        const int b = __builtin_ctzll(reach);
        if (p < TOPK_CAND) at_s[p] = (first + b / VEC * NT) * VEC + b % VEC;
      }
    }
  };
  r.each([&](int at, auto& v) {
    constexpr int N = count_of<decltype(v)>;
    if constexpr (N > 1) {
      uint32_t m = 0;
#pragma unroll
      for (int j = N - 1; j >= 0; --j) {
        const bool under = v[j] < bound;
        s += under ? exp_near(v[j], es, bound) : 0.f;
        m = m << 1 | (under ? 0 : 1);
      }
      s.template piece_done<N>();
      if (bit == 0) first = at / VEC;
      reach |= (uint64_t)m << bit;
      bit += N;
      if (bit == CHUNK * VEC) {
        list();
        bit = 0;
        reach = 0;
      }
    } else {
      list();                            // what the pieces left, then the element behind them
      reach = 0;
      if (v[0] < bound) {
        s += exp_near(v[0], es, bound);
      } else {
        const int p = atomicAdd(&count, 1);
        if (p < TOPK_CAND) at_s[p] = at;
      }
    }
  });
  list();
  // log of the sum of exp(x / T) over the elements under the bound
  const double sum = block_reduce<NT>(s.value(), redd, SumOp());
  int m = count;
  const bool flood = m > TOPK_CAND;      // uniform over the workgroup, as all that follows from it
  // the mass that is left, as log(under) + ref / T
  double under = sum;
  float ref = bound;
  if (flood || !(sum > 1e-20 && sum < 1e30)) {
    // the exact cut: an element is taken up if key > cut_key, or key == cut_key at an index up to cut_index
    uint32_t cut_key = bound_key;
    int cut_index = 0x7fffffff;
    if (flood) {
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
      int before = -1;                   // largest index that fewer than `equals` of them come up to
      for (int bit = 30; bit >= 0; --bit) {
        const int trial = before + (1 << bit);
        if (count_over([&](uint32_t key, int at, int j) { return key == kth && at <= trial - j; }) < equals) before = trial;
      }
      cut_key = kth;
      cut_index = before + 1;
      __syncthreads();
      if (tid == 0) count = 0;
      __syncthreads();
    }
    float below = -INFINITY;             // largest logit that is not taken up
    r.each([&](int at, auto& v) {
#pragma unroll
      for (int j = 0; j < count_of<decltype(v)>; ++j) {
        const uint32_t key = order_key(v[j]);
        if (!(key > cut_key || (key == cut_key && at <= cut_index - j))) below = fmaxf(below, v[j]);
        else if (flood) at_s[atomicAdd(&count, 1)] = at + j;                      // exactly k of them
      }
    });
    below = block_reduce<NT>(below, redf, MaxOp());
    ref = below == -INFINITY ? 0.f : below;
    ThreadSum<HOLD> s2;
    r.each([&](int at, auto& v) {
#pragma unroll
      for (int j = 0; j < count_of<decltype(v)>; ++j) {
        const uint32_t key = order_key(v[j]);
        const bool taken = key > cut_key || (key == cut_key && at <= cut_index - j);
        s2 += taken ? 0.f : exp_at(v[j], es, ref);
      }
      s2.template piece_done<count_of<decltype(v)>>();
    });
    under = block_reduce<NT>(s2.value(), redd, SumOp());
    if (flood) m = k;
  }

  for (int i = tid; i < m; i += NT) {
    const int at = at_s[i];
    uint32_t u;
    if constexpr (DT == BCFFT_F32) u = ((const uint32_t*)row)[at];
    else u = ((const uint16_t*)row)[at];
    raw[i] = u;
    cand[i] = full_key(order_key(DT == BCFFT_F32 ? __uint_as_float(u) : unpack16<DT == BCFFT_F32 ? BCFFT_BF16 : DT>(u).x), at);
  }
  __syncthreads();
  // 16 lanes per candidate: each compares it with every 16th
  for (int i = tid / 16; i < (m + 3) / 4 * 4; i += NT / 16) {      // whole waves: they shuffle
    const uint64_t key = cand[i < m ? i : 0];
    int rank = 0;
#pragma unroll 4
    for (int j = tid % 16; j < m; j += 16) rank += cand[j] > key;
    rank = lanes_reduce<16>(rank, SumOp());
    if (i < m && tid % 16 == 0) {
      if (rank < k) {
        if constexpr (DT == BCFFT_F32) ((uint32_t*)values)[n * k + rank] = raw[i];
        else ((uint16_t*)values)[n * k + rank] = (uint16_t)raw[i];
        indices[n * k + rank] = (int32_t)~(uint32_t)key;
      } else {
        left[rank] = key_value((uint32_t)(key >> 32));
      }
    }
  }
  if (m > k) __syncthreads();            // candidates that were not taken join the rest, in rank order
  if (tid < 64) {
    double hi = (double)ref * inv_t, sum_left = under;
    if (m > k) {
      const double top = (double)left[k] * inv_t;
      if (!(fabs(top - hi) <= 600.0)) {  // a reference of their own (or infinite, or NaN)
        const double log_under = under > 0.0 ? hi + log(under) : -INFINITY;
        sum_left = top == INFINITY || top == -INFINITY ? 0.0 : exp(log_under - top);
        hi = top;
      }
      double e = 0.0;
      if (hi - hi == 0.0) {
        for (int i = k + tid; i < m; i += 64) e += exp((double)left[i] * inv_t - hi);
      }
      sum_left += wave_reduce(e, SumOp());
    }
    // an infinite or NaN `top` is the answer itself; the log of nothing is -inf
    if (tid == 0) rest[n] = (float)(m > k && hi - hi != 0.0 ? hi : sum_left > 0.0 ? hi + log(sum_left) : sum_left != sum_left ? sum_left : -INFINITY);
  }
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
  double p[TOPK_MAX];                    // teacher's logit over T, then exp(that - the largest)
  double e[TOPK_MAX];                    // student's logit, then exp((that - the row's largest) / T)
  int32_t at[TOPK_MAX];                  // index, or -1
  double redd[4][16];
  double topd[16];
  float redf[16];
  int dup;
};

// the bits of elements `at` .. `at + N` of one piece; bytes, as a piece of 8 is one
template <int N>
__device__ __forceinline__ uint32_t piece_bits(const uint32_t* bits, int at) {
  const uint32_t b = ((const uint8_t*)bits)[at >> 3];
  return N == 8 ? b : b >> (at & 7) & ((1u << N) - 1);
}
// e, or 0 where bit j of a piece is set: two operations
__device__ __forceinline__ float unless(uint32_t not_bits, int j, float e) {
  return __uint_as_float(__float_as_uint(e) & (uint32_t)__builtin_amdgcn_sbfe((int)not_bits, (uint32_t)j, 1u));
}

// Loads the entries and sets the bitmap; the largest teacher logit over T of this thread's entries
template <int DT, int NT>
__device__ __forceinline__ double load_entries(const DistillArgs& a, int64_t n, const char* row, Entries& en, uint32_t* bits) {
  const int tid = threadIdx.x;
  for (int w = tid; w < (int)((a.vocab + 31) / 32); w += NT) bits[w] = 0;
  if (tid == 0) en.dup = 0;
  __syncthreads();
  double mx = a.rest && tid == 0 ? (double)a.rest[n] : -INFINITY;
  for (int j = tid; j < a.k; j += NT) {
    const int64_t e = n * a.k + j;
    const int64_t at = a.idx64 ? ((const int64_t*)a.indices)[e] : (int64_t)((const int32_t*)a.indices)[e];
    const bool ok = at >= 0 && at < a.vocab;
    const double t = ok ? (double)load_scalar(a.values, e, a.vdt) * a.inv_t : -INFINITY;
    en.at[j] = ok ? (int32_t)at : -1;
    en.p[j] = t;
    en.e[j] = ok ? load_scalar(row, at, DT) : -INFINITY;
    if (ok && (atomicOr(&bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1)) en.dup = 1;
    mx = t > mx || t != t ? t : mx;      // NaN stays: it makes the row NaN, as in a softmax
  }
  return mx;
}

// whether entry j is the first with its index; mass: the sum of p over all entries with that index
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

// The entries' gradients, over the zeros that the pass before them left there. The wait makes that pass's
// stores complete (acknowledged by L2) before other waves of the workgroup store into the same lines.
template <int DT, int NT>
__device__ __forceinline__ void write_entries(const DistillArgs& a, int64_t n, Entries& en, double inv_s, double inv_total,
                                              float scale) {
  char* out = (char*)a.grad + n * a.vocab * (DT == BCFFT_F32 ? 4 : 2);
  wait_vmcnt<0>();
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += NT) {
    if (en.at[j] < 0) continue;
    double mass = en.p[j];
    if (!first_of(en, a.k, j, mass)) continue;
    store_one<DT>(out, en.at[j], (float)(en.e[j] * inv_s - mass * inv_total) * scale);
  }
}
// The other elements': exp((v - ref) / T) times coef
template <int DT, class ROW>
__device__ __forceinline__ void write_others(const DistillArgs& a, int64_t n, ROW& r, const uint32_t* bits, float ref,
                                             float coef) {
  char* out = (char*)a.grad + n * a.vocab * (DT == BCFFT_F32 ? 4 : 2);
  r.each([&](int at, auto& v) {
    constexpr int N = count_of<decltype(v)>;
    const uint32_t keep = ~piece_bits<N>(bits, at);
    float g[N];
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = unless(keep, j, exp_at(v[j], a.es, ref) * coef);
    store_piece<DT>(out, at, g);
  });
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

// Loss of a row and, with GRAD, its gradient, in one read of the row.
// 1. the row's maximum                                                             1.5 operations a logit
// 2. the sum of the exponentials outside the entries, the entries' own in fp64 beside it               10
// 3. gradient: the exponentials from 2, where up to 64 per thread stay in registers                   1.5
// Where the sum of 2 vanishes in fp32 (all of the row 45 T below its maximum but the entries) and the
// teacher's rest needs its logarithm, 2 runs again relative to the others' own maximum.
template <int DT, int NT, int HOLD, bool GRAD>
__global__ __launch_bounds__(NT, NT == 512 ? (GRAD ? 4 : 6) : 1) void bc_distill_kernel(DistillArgs a) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2, VEC = RowType<DT>::VEC;
  constexpr bool KEEP = GRAD && HOLD > 0 && HOLD * VEC <= 64;
  __shared__ Entries en;
  extern __shared__ uint32_t bits[];
  const int tid = threadIdx.x;
  const int64_t n = blockIdx.x;
  const float w = a.weight ? a.weight[n] : 1.f;
  const char* row = (const char*)a.logits + n * a.row_stride * E;
  Row<DT, NT, HOLD> r;
  double am = -INFINITY;
  if (w != 0.f) {                        // uniform: a row of weight 0 is not read
    r.open(row, a.vocab);
    am = load_entries<DT, NT>(a, n, row, en, bits);
  }
  float mx = -INFINITY;
  if (w != 0.f) {
    r.each([&](int, auto& v) {
#pragma unroll
      for (int j = 0; j + 1 < count_of<decltype(v)>; j += 2) mx = fmaxf(fmaxf(mx, v[j]), v[j + 1]);
      if constexpr (count_of<decltype(v)> == 1) mx = fmaxf(mx, v[0]);
    });
  }
  am = wave_reduce(am, MaxOp());
  mx = wave_reduce(mx, MaxOp());
  if ((tid & 63) == 0) {
    en.topd[tid >> 6] = am;
    en.redf[tid >> 6] = mx;
  }
  __syncthreads();
  am = across_waves<NT>(en.topd, MaxOp());
  mx = across_waves<NT>(en.redf, MaxOp());
  if (am == -INFINITY) {                 // no teacher mass (or weight 0): uniform over the workgroup
    if (tid == 0) {
      a.loss[n] = 0.f;
      if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * n) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if constexpr (GRAD) write_zero<DT, NT>(a, n);
    return;
  }
  const float m_all = mx == -INFINITY ? 0.f : mx;

  // sums over the entries: the teacher's total, the student's, the loss's part linear in the logits. Before
  // the pass over the row: fp64 functions take 40 registers
  double total = 0.0, se = 0.0, lin = 0.0;
  for (int j = tid; j < a.k; j += NT) {
    if (en.at[j] < 0) continue;
    const double t = en.p[j] - am, p = exp(t), x = (en.e[j] - (double)m_all) * a.inv_t, e = exp(x);
    en.p[j] = p;
    en.e[j] = e;
    total += p;
    if (p > 0.0) lin += p * (t - x);
    else if (p != p) lin = p;
    if (!en.dup) se += e;
  }
  if (en.dup) {                          // uniform: each index once
    __syncthreads();
    for (int j = tid; j < a.k; j += NT) {
      double mass;
      if (en.at[j] >= 0 && first_of(en, a.k, j, mass)) se += en.e[j];
    }
  }
  // the other elements' sum
  ThreadSum<HOLD> so;
  float kept[KEEP ? HOLD : 1][VEC], kept_tail = 0.f;
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int p = i * NT + tid;
      if (p < (int)r.pieces) {
        float v[VEC];
        unpack<DT>(r.held[i], v);
        const uint32_t keep = ~piece_bits<VEC>(bits, p * VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          kept[i][j] = unless(keep, j, exp_at(v[j], a.es, m_all));
          so += kept[i][j];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (tid < r.tail) {
      kept_tail = unless(~piece_bits<1>(bits, (int)(r.pieces * VEC) + tid), 0, exp_at(r.last, a.es, m_all));
      so += kept_tail;
    }
  } else {
    r.each([&](int at, auto& v) {
      constexpr int N = count_of<decltype(v)>;
      const uint32_t keep = ~piece_bits<N>(bits, at);
#pragma unroll
      for (int j = 0; j < N; ++j) so += unless(keep, j, exp_at(v[j], a.es, m_all));
      so.template piece_done<N>();
    });
  }
  double sums[4] = {so.value(), total, se, lin};
#pragma unroll
  for (int q = 0; q < 4; ++q) sums[q] = wave_reduce(sums[q], SumOp());
  if ((tid & 63) == 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) en.redd[q][tid >> 6] = sums[q];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) sums[q] = across_waves<NT>(en.redd[q], SumOp());
  const double rest_a = a.rest ? (double)a.rest[n] - am : -INFINITY, rest_e = exp(rest_a);
  const double inv_total = 1.0 / (sums[1] + rest_e), rest_p = rest_e * inv_total;
  double sum_o = sums[0];                // relative to m_all
  const double sum_e = sums[2];
  float ref = m_all;
  double sum_ref = sum_o;                // the others' sum relative to ref
  const bool again = rest_p != 0.0 && sum_o < 1e-20;             // uniform
  if (again) {
    float mo = -INFINITY;
    Row<DT, NT, 0> r2;
    r2.open(row, a.vocab);
    r2.each([&](int at, auto& v) {
      constexpr int N = count_of<decltype(v)>;
      const uint32_t b = piece_bits<N>(bits, at);
#pragma unroll
      for (int j = 0; j < N; ++j) mo = fmaxf(mo, b >> j & 1 ? -INFINITY : v[j]);
    });
    mo = block_reduce<NT>(mo, en.redf, MaxOp());
    ref = mo == -INFINITY ? 0.f : mo;
    ThreadSum<HOLD> s2;                  // as many terms per thread as where the row is held
    r2.each([&](int at, auto& v) {
      constexpr int N = count_of<decltype(v)>;
      const uint32_t keep = ~piece_bits<N>(bits, at);
#pragma unroll
      for (int j = 0; j < N; ++j) s2 += unless(keep, j, exp_at(v[j], a.es, ref));
      s2.template piece_done<N>();
    });
    sum_ref = block_reduce<NT>(s2.value(), en.topd, SumOp());
    sum_o = mo == -INFINITY ? 0.0 : sum_ref * exp(((double)ref - (double)m_all) * a.inv_t);
  }
  const double sum = sum_o + sum_e, inv_s = 1.0 / sum;
  // d loss / d s of an element outside the entries, over exp((v - ref) / T)
  const double shift = ref == m_all ? 1.0 : exp(((double)ref - (double)m_all) * a.inv_t);
  const double coef = shift * inv_s - (rest_p != 0.0 && sum_ref != 0.0 ? rest_p / sum_ref : 0.0);
  if constexpr (GRAD) {
    const float scale = (float)(w * a.inv_t);
    if (KEEP && !again) {
      char* out = (char*)a.grad + n * a.vocab * E;
      const float c = (float)coef * scale;
#pragma unroll
      for (int i = 0; i < (KEEP ? HOLD : 0); ++i) {
        const int p = i * NT + tid;
        if (p < (int)r.pieces) {
          float g[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[j] = kept[i][j] * c;
          store_piece<DT>(out, p * VEC, g);
        }
      }
      if (tid < r.tail) store_one<DT>(out, r.pieces * VEC + tid, kept_tail * c);
    } else {
      const float c = (float)coef * scale;
      if (HOLD > 0 && !KEEP) {
        write_others<DT>(a, n, r, bits, ref, c);
      } else {
        Row<DT, NT, 0> r2;
        r2.open(row, a.vocab);
        write_others<DT>(a, n, r2, bits, ref, c);
      }
    }
    write_entries<DT, NT>(a, n, en, inv_s, inv_total, scale);
  }
  if (tid == NT - 1) {                   // the last wave: the first ones write the entries meanwhile
    // sum_j P_j ((a_j - am) - (s_j - m_all) / T) + log sum - log total, and the rest's part
    double loss = sums[3] * inv_total + log(sum) + log(inv_total);
    if (rest_p != 0.0) loss += rest_p * (rest_a - (((double)ref - (double)m_all) * a.inv_t + log(sum_ref)));
    a.loss[n] = (float)loss * w;
    if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * n) = make_float4(ref, (float)coef, m_all, (float)inv_s);
  }
}

// Gradient from the forward's sums: one read of the row, one write
template <int DT, int NT>
__global__ __launch_bounds__(NT) void bc_distill_backward_kernel(DistillArgs a) {
  constexpr int E = DT == BCFFT_F32 ? 4 : 2;
  __shared__ Entries en;
  extern __shared__ uint32_t bits[];
  const int64_t n = blockIdx.x;
  const float w = a.weight ? a.weight[n] : 1.f;
  const char* row = (const char*)a.logits + n * a.row_stride * E;
  double am = -INFINITY;
  if (w != 0.f) am = block_reduce<NT>(load_entries<DT, NT>(a, n, row, en, bits), en.topd, MaxOp());   // uniform
  if (am == -INFINITY) {
    write_zero<DT, NT>(a, n);
    return;
  }
  const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * n);
  double total = 0.0;
  for (int j = threadIdx.x; j < a.k; j += NT) {
    if (en.at[j] < 0) continue;
    en.p[j] = exp(en.p[j] - am);
    en.e[j] = exp((en.e[j] - (double)st.z) * a.inv_t);
    total += en.p[j];
  }
  total = block_reduce<NT>(total, en.topd, SumOp()) + (a.rest ? exp((double)a.rest[n] - am) : 0.0);
  const float scale = (float)(w * a.inv_t) * a.upstream[n];
  Row<DT, NT, 0> r;
  r.open(row, a.vocab);
  write_others<DT>(a, n, r, bits, st.x, st.y * scale);
  write_entries<DT, NT>(a, n, en, st.w, 1.0 / total, scale);
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
static void by_row(int64_t vocab, F&& go) {
  const int64_t pieces = (vocab + RowType<DT>::VEC - 1) / RowType<DT>::VEC;
  using std::integral_constant;
  if (pieces <= 512) go(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (pieces <= 2048) go(integral_constant<int, 256>(), integral_constant<int, 8>());
  else if (pieces <= 4096) go(integral_constant<int, 512>(), integral_constant<int, 8>());
  else if (pieces <= 8192) go(integral_constant<int, 1024>(), integral_constant<int, 8>());
  else if (pieces <= 16384) go(integral_constant<int, 1024>(), integral_constant<int, 16>());
  else go(integral_constant<int, 1024>(), integral_constant<int, 0>());
}

// A launch holds fewer than 2^32 threads: rows by the 2^21 (of up to 1024 threads each)
constexpr int64_t LAUNCH_ROWS = 1 << 21;
template <class F>
static void by_rows(int64_t n, F&& go) {
  for (int64_t first = 0; first < n; first += LAUNCH_ROWS) go(first, n - first < LAUNCH_ROWS ? n - first : LAUNCH_ROWS);
}

// The same for the top k, with at least 2 k threads (k <= 512)
template <int DT, class F>
static void by_row_topk(int64_t vocab, int64_t k, F&& go) {
  const int64_t pieces = (vocab + RowType<DT>::VEC - 1) / RowType<DT>::VEC;
  using std::integral_constant;
  if (2 * k <= 256 && pieces <= 2048) {
    if (pieces <= 512) go(integral_constant<int, 256>(), integral_constant<int, 2>());
    else go(integral_constant<int, 256>(), integral_constant<int, 8>());
  } else if (2 * k <= 512 && pieces <= 4096) {
    if (pieces <= 1024) go(integral_constant<int, 512>(), integral_constant<int, 2>());
    else go(integral_constant<int, 512>(), integral_constant<int, 8>());
  } else if (pieces <= 2048) {
    go(integral_constant<int, 1024>(), integral_constant<int, 2>());
  } else if (pieces <= 8192) {
    go(integral_constant<int, 1024>(), integral_constant<int, 8>());
  } else if (pieces <= 16384) {
    go(integral_constant<int, 1024>(), integral_constant<int, 16>());
  } else {
    go(integral_constant<int, 1024>(), integral_constant<int, 0>());
  }
}

template <int DT>
static void launch_topk_dt(const void* logits, int64_t n, int64_t vocab, int64_t row_stride, int k, double temperature,
                           void* values, int32_t* indices, float* rest, hipStream_t s) {
  constexpr int64_t E = DT == BCFFT_F32 ? 4 : 2;
  by_row_topk<DT>(vocab, k, [&](auto nt, auto hold) {
    by_rows(n, [&](int64_t at, int64_t rows) {
      hipLaunchKernelGGL((bc_topk_logits_kernel<DT, nt.value, hold.value>), dim3((unsigned)rows), dim3(nt.value), 0, s,
                         (const char*)logits + at * row_stride * E, vocab, row_stride, k, exp_scale(temperature),
                         1.0 / temperature, (char*)values + at * k * E, indices + at * k, rest + at);
    });
  });
}

// the operands from row `at` on
template <int DT>
static DistillArgs from_row(const DistillArgs& a, int64_t at) {
  constexpr int64_t E = DT == BCFFT_F32 ? 4 : 2;
  auto plus = [&](auto* p, int64_t by) { return p ? p + by : nullptr; };
  DistillArgs b = a;
  b.logits = (const char*)a.logits + at * a.row_stride * E;
  b.values = (const char*)a.values + at * a.k * (a.vdt == BCFFT_F32 ? 4 : 2);
  b.indices = (const char*)a.indices + at * a.k * (a.idx64 ? 8 : 4);
  b.rest = plus(a.rest, at);
  b.weight = plus(a.weight, at);
  b.upstream = plus(a.upstream, at);
  b.loss = plus(a.loss, at);
  b.stats = plus(a.stats, 4 * at);
  b.grad = plus((char*)a.grad, at * a.vocab * E);
  return b;
}
template <int DT>
static void launch_distill_rows(const DistillArgs& a, int64_t n, hipStream_t s) {
  const unsigned lds = (unsigned)((a.vocab + 31) / 32 * 4);
  if (a.upstream) {
    hipLaunchKernelGGL((bc_distill_backward_kernel<DT, 512>), dim3((unsigned)n), dim3(512), lds, s, a);
    return;
  }
  by_row<DT>(a.vocab, [&](auto nt, auto hold) {
    if (a.grad) hipLaunchKernelGGL((bc_distill_kernel<DT, nt.value, hold.value, true>), dim3((unsigned)n), dim3(nt.value), lds, s, a);
    else hipLaunchKernelGGL((bc_distill_kernel<DT, nt.value, hold.value, false>), dim3((unsigned)n), dim3(nt.value), lds, s, a);
  });
}
template <int DT>
static void launch_distill_dt(const DistillArgs& a, int64_t n, hipStream_t s) {
  by_rows(n, [&](int64_t at, int64_t rows) { launch_distill_rows<DT>(from_row<DT>(a, at), rows, s); });
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
