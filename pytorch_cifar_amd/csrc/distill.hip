// Distillation from a teacher's top logits: the K largest logits a row with the row's
// log-sum-exp (top_logits), and the loss of a student's logits against them with its gradient
// (distill_*). Rows are [R][V] in fp32 / bf16 / fp16 with any row stride; one workgroup a row.
//
// Both read each logit once: a row of up to 16 chunks of 16 bytes a thread stays in registers
// between its passes (maximum, then sum of exponentials, then gradient or selection); longer rows
// are read again for each pass.
#include "distill.h"

#include <algorithm>

namespace pca {
namespace {

typedef _Float16 f16;

template <typename T>
constexpr int kVE = 16 / (int)sizeof(T);   // elements of a 16-byte chunk

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float to_f(f16 v) { return static_cast<float>(v); }

__device__ __forceinline__ void unpack(const uint4& u, float* f, float) {
  f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float* f, bf16) { unpack8(u, f); }
__device__ __forceinline__ void unpack(const uint4& u, float* f, f16) {
  f16 h[8];
  __builtin_memcpy(h, &u, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(h[i]);
}
__device__ __forceinline__ uint4 pack(const float* f, float) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float* f, bf16) { return pack8(f); }
__device__ __forceinline__ uint4 pack(const float* f, f16) {
  f16 h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = static_cast<f16>(f[i]);
  uint4 u;
  __builtin_memcpy(&u, h, 16);
  return u;
}

// Chunk c of a row, whose elements are aligned to themselves only (an odd V or row stride): the
// 16-byte access is legal at any address here. Elements past the row read as -inf (exp 0).
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const T* __restrict__ row, int c, int V) {
  uint4 u;
  const T* p = row + (size_t)c * kVE<T>;
  if ((c + 1) * kVE<T> <= V) {
    __builtin_memcpy(&u, p, 16);
    return u;
  }
  float f[kVE<T>];
#pragma unroll
  for (int i = 0; i < kVE<T>; ++i) f[i] = c * kVE<T> + i < V ? to_f(p[i]) : -INFINITY;
  return pack(f, T());
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ row, int c, int V, const float* f) {
  const uint4 u = pack(f, T());
  T* p = row + (size_t)c * kVE<T>;
  if ((c + 1) * kVE<T> <= V) {
    __builtin_memcpy(p, &u, 16);
    return;
  }
  T h[kVE<T>];
  __builtin_memcpy(h, &u, 16);
#pragma unroll
  for (int i = 0; i < kVE<T>; ++i)
    if (c * kVE<T> + i < V) p[i] = h[i];
}

// A row's chunks as one thread owns them: c = thread, thread + BLOCK, ... NC > 0: held in
// registers after load(); NC == 0: read again at each use.
template <typename T, int BLOCK, int NC>
struct Row {
  const T* p;
  int V, n;   // n: chunks of the row
  uint4 u[NC > 0 ? NC : 1];

  __device__ __forceinline__ void load(const T* row, int V_) {
    p = row, V = V_, n = (V_ + kVE<T> - 1) / kVE<T>;
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = threadIdx.x + i * BLOCK;
        if (c < n) u[i] = load_chunk(p, c, V);
      }
    }
  }
  // fn(chunk number, its elements as float)
  template <typename F>
  __device__ __forceinline__ void each(F&& fn) const {
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = threadIdx.x + i * BLOCK;
        if (c < n) {
          // (opaque, so that the passes unpack anew: kept across them, the floats spill)
          uint4 v = u[i];
          asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
          float f[kVE<T>];
          unpack(v, f, T());
          fn(c, f);
        }
      }
    } else {
#pragma unroll 4
      for (int c = threadIdx.x; c < n; c += BLOCK) {
        const uint4 v = load_chunk(p, c, V);
        float f[kVE<T>];
        unpack(v, f, T());
        fn(c, f);
      }
    }
  }
};

struct MaxOp {
  template <typename A>
  __device__ __forceinline__ A operator()(A a, A b) const { return a > b ? a : b; }
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};
struct SumOp {
  template <typename A>
  __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};

// v of all threads, folded in a fixed order; every thread gets the result. red: BLOCK/64 values.
template <int BLOCK, typename A, typename Op>
__device__ __forceinline__ A block_fold(A v, A* red, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  if constexpr (BLOCK == 64) return v;
  constexpr int NW = BLOCK / 64;
  __syncthreads();   // (red may still be read by the fold before)
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  A r = red[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) r = op(r, red[w]);
  return r;
}

// ------------------------------------------------------------------------------- top_logits
// Order of the selection as one whole number: the larger logit first (NaN above all, -0 equal to
// +0), among equal ones the lower class. 32 bits of the logit above kIdxBits of the class.
constexpr int kIdxBits = 18;
static_assert((1 << kIdxBits) == kDistillMaxClasses, "classes fit the index bits");

__device__ __forceinline__ uint32_t order_bits(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.f);   // (-0 + 0 is +0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float f, int idx) {
  return ((uint64_t)order_bits(f) << kIdxBits) | (uint32_t)(kDistillMaxClasses - 1 - idx);
}
__device__ __forceinline__ int key_index(uint64_t k) {
  return kDistillMaxClasses - 1 - (int)(k & (kDistillMaxClasses - 1));
}

constexpr int kList = 2048;   // candidates that are ranked
// a selection may end with this many candidates: ranking them costs less than a further pass
__device__ __forceinline__ int enough(int k) { return k + k / 2 + 64; }
static_assert(kDistillMaxK + kDistillMaxK / 2 + 64 <= kList, "candidates fit");

// The largest bound of the form lo + (hi - lo) / 2 ... for which at least k keys are as large,
// halving until at most enough(k) are. Keys differ, so it ends for any row (NaN, all equal, all
// -inf), after at most 50 passes.
template <typename T, int BLOCK, int NC>
__device__ uint64_t bound_of_keys(const Row<T, BLOCK, NC>& row, int k, int* red) {
  uint64_t lo = 0, hi = 1ull << (32 + kIdxBits);
  int n = row.V;
  while (n > enough(k)) {
    const uint64_t mid = lo + (hi - lo) / 2;
    int c = 0;
    row.each([&](int ch, const float* f) {
#pragma unroll
      for (int j = 0; j < kVE<T>; ++j) {
        const int idx = ch * kVE<T> + j;
        c += idx < row.V && order_key(f[j], idx) >= mid;
      }
    });
    c = block_fold<BLOCK>(c, red, SumOp());
    if (c >= k) lo = mid, n = c;
    else hi = mid;
  }
  return lo;
}

// The same over the maxima of the row's threads (one wave, BLOCK / 64 of them a lane): at least k
// logits are as large as the k-th largest of them, and in a row in no particular order few more.
template <int BLOCK>
__device__ uint32_t bound_of_maxima(const uint32_t* maxima, int k) {
  constexpr int N = BLOCK / 64;
  uint32_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = maxima[threadIdx.x + i * 64];
  uint64_t lo = 0, hi = 1ull << 32;
  int n = BLOCK;
  while (n > k + k / 4 + 8 && hi - lo > 1) {
    const uint32_t mid = (uint32_t)(lo + (hi - lo) / 2);
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += __popcll(__ballot(v[i] >= mid));
    if (c >= k) lo = mid, n = c;
    else hi = mid;
  }
  return (uint32_t)lo;
}

// One pass over the row gives each thread its maximum and its sum of exponentials (relative to its
// running maximum). The k largest are then sought among the logits of the threads whose maximum
// reaches a bound; a row that defeats the bound (NaN, many equal logits, k near the number of
// threads) is halved by counting.
template <typename T, int BLOCK, int NC>
__global__ __launch_bounds__(BLOCK) void top_logits_kernel(const T* __restrict__ z, int64_t ld,
                                                           int V, int k, float c, double inv_t,
                                                           T* __restrict__ values,
                                                           int32_t* __restrict__ indices,
                                                           float* __restrict__ lse) {
  __shared__ double red[16];
  __shared__ uint32_t maxima[BLOCK];
  __shared__ uint64_t list[kList];
  __shared__ uint32_t found, bound;
  const int64_t r = blockIdx.x;
  Row<T, BLOCK, NC> row;
  row.load(z + r * ld, V);

  float m = -INFINITY, base = 0.f, s = 0.f;   // base: m where it is finite
  row.each([&](int, const float* f) {
    float cm = f[0];
#pragma unroll
    for (int j = 1; j < kVE<T>; ++j) cm = fmaxf(cm, f[j]);
    m = fmaxf(m, cm);
    const float b = isinf(m) ? 0.f : m;
    s *= __builtin_amdgcn_exp2f((base - b) * c);
    base = b;
#pragma unroll
    for (int j = 0; j < kVE<T>; ++j) s += __builtin_amdgcn_exp2f((f[j] - b) * c);
  });
  // (a row of -inf: log 0; one with +inf: log inf; NaN stays)
  float all = block_fold<BLOCK>(m, reinterpret_cast<float*>(red), MaxOp());
  if (isinf(all)) all = 0.f;
  s *= __builtin_amdgcn_exp2f((base - all) * c);
  const double sum = block_fold<BLOCK>((double)s, red, SumOp());
  if (threadIdx.x == 0) {
    lse[r] = (float)((double)all * inv_t + log(sum));
    found = 0;
    bound = 0;
  }
  const uint32_t mine = order_bits(m);
  maxima[threadIdx.x] = mine;
  __syncthreads();

  bool few = k <= BLOCK / 4 * 3 && sum == sum;   // (a thread's maximum passes over NaN)
  if (few) {
    if (threadIdx.x < 64) {
      const uint32_t b = bound_of_maxima<BLOCK>(maxima, k);
      if (threadIdx.x == 0) bound = b;
    }
    __syncthreads();
    const uint32_t b = bound;
    if (mine >= b) {
      row.each([&](int ch, const float* f) {
#pragma unroll
        for (int j = 0; j < kVE<T>; ++j) {
          const int idx = ch * kVE<T> + j;
          if (idx < V && order_bits(f[j]) >= b) {
            const uint32_t at = atomicAdd(&found, 1u);
            if (at < kList) list[at] = order_key(f[j], idx);
          }
        }
      });
    }
    __syncthreads();
    few = found <= kList;
  }
  if (!few) {
    __syncthreads();
    if (threadIdx.x == 0) found = 0;
    const uint64_t b = bound_of_keys(row, k, reinterpret_cast<int*>(red));
    __syncthreads();
    row.each([&](int ch, const float* f) {
#pragma unroll
      for (int j = 0; j < kVE<T>; ++j) {
        const int idx = ch * kVE<T> + j;
        const uint64_t key = order_key(f[j], idx);
        if (idx < V && key >= b) {
          const uint32_t at = atomicAdd(&found, 1u);
          if (at < kList) list[at] = key;
        }
      }
    });
    __syncthreads();
  }
  // a candidate's place is the number of candidates before it
  const int n = (int)found;
  for (int i = threadIdx.x; i < n; i += BLOCK) {
    const uint64_t key = list[i];
    int at = 0;
    for (int j = 0; j < n; ++j) at += list[j] > key;
    if (at < k) {
      const int idx = key_index(key);
      values[r * k + at] = row.p[idx];
      indices[r * k + at] = idx;
    }
  }
}

// Rows of up to 64 classes: a wave each, a class a lane. The place of a logit is the number of
// logits before it, counted over the lanes.
template <typename T>
__global__ __launch_bounds__(256) void top_small_kernel(const T* __restrict__ z, int64_t ld,
                                                        int64_t R, int V, int k, float c,
                                                        double inv_t, T* __restrict__ values,
                                                        int32_t* __restrict__ indices,
                                                        float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (r >= R) return;
  const T v = z[r * ld + min(lane, V - 1)];
  const float f = lane < V ? to_f(v) : -INFINITY;
  float m = wave_max(f);
  if (isinf(m)) m = 0.f;
  const float s = wave_sum(__builtin_amdgcn_exp2f((f - m) * c));
  const uint32_t key = order_bits(f);
  int at = 0;
  for (int j = 0; j < V; ++j) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)key, j);
    at += other > key || (other == key && j < lane);
  }
  if (lane < V && at < k) {
    values[r * k + at] = v;
    indices[r * k + at] = lane;
  }
  if (lane == 0) lse[r] = (float)((double)m * inv_t + log((double)s));
}

// ------------------------------------------------------------------------------ distill_loss
// Row of the loss, with q = softmax(z/T), e_j = exp((z_j - max z)/T), s = sum e:
//   KD   = sum_k p_k (log p_k - log q_k) + rest (log rest - log q_rest)
//   loss = alpha T^2 KD + (1 - alpha) (lse(z) - z_y)
//   d/dz_j = e_j A - [not kept] e_j B - [kept] alpha T p_j + (1 - alpha)(softmax(z)_j - [j = y])
// with A = alpha T (sum p + rest) / s and B = alpha T rest / s_rest, s_rest the sum of e over the
// classes that are not kept: summed by itself (a difference s - s_kept would lose it where the
// kept classes hold nearly all). The K values of the teacher's side are computed in 64 bits: what
// is left of its mass, 1 - sum p, is a difference.
//
// A bit a class marks the kept ones (LDS, V / 8 bytes). It gives s_rest, and finds an index that
// a row names twice: its entries are then gathered for each of them.
template <typename T, int BLOCK, int NC, bool GRAD>
__global__ __launch_bounds__(BLOCK) void distill_kernel(DistillArgs a, float c_t, float c_1) {
  extern __shared__ char smem[];
  __shared__ double red[16];
  __shared__ int flags[4];   // kept entries, an index twice, an index past the classes
  const int64_t r = blockIdx.x;
  const int V = a.V, K = a.K, t = threadIdx.x;
  double* p = reinterpret_cast<double*>(smem);          // [K] the teacher's probabilities
  int* cls = reinterpret_cast<int*>(p + K);             // [K] their classes, -1: not kept
  uint32_t* mark = reinterpret_cast<uint32_t*>(cls + K);
  const uint8_t* mark8 = reinterpret_cast<const uint8_t*>(mark);
  const int words = (V + 31) / 32;

  for (int i = t; i < words; i += BLOCK) mark[i] = 0;
  if (t < 4) flags[t] = 0;
  __syncthreads();

  // ---- the teacher's side
  double tmax = -INFINITY;
  int kept = 0, twice = 0, bad = 0;
  for (int k = t; k < K; k += BLOCK) {
    const int64_t at = r * K + k;
    const int64_t idx = a.index64 ? reinterpret_cast<const int64_t*>(a.indices)[at]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.indices)[at];
    double v = a.value_type == LOGIT_F32 ? (double)reinterpret_cast<const float*>(a.values)[at]
               : a.value_type == LOGIT_BF16
                   ? (double)to_f(reinterpret_cast<const bf16*>(a.values)[at])
                   : (double)to_f(reinterpret_cast<const f16*>(a.values)[at]);
    int j = -1;
    if (idx >= V) bad = 1;
    if (idx >= 0 && idx < V) {
      j = (int)idx;
      const uint32_t bit = 1u << (j & 31);
      if (atomicOr(&mark[j >> 5], bit) & bit) twice = 1;
      v /= a.temp;
      kept = 1;
      tmax = v != v ? v : fmax(tmax, v);
    }
    cls[k] = j;
    p[k] = j < 0 ? -INFINITY : v;
  }
  if (kept) atomicOr(&flags[0], 1);
  if (twice) atomicOr(&flags[1], 1);
  if (bad) atomicOr(&flags[2], 1);
  int64_t y = a.target ? a.target[r] : a.ignore_index;
  const bool label = a.target && y != a.ignore_index && a.alpha != 1.0;
  bool poison = label && (y < 0 || y >= V);
  if (poison) y = 0;
  tmax = block_fold<BLOCK>(tmax, red, MaxOp());
  __syncthreads();
  poison |= flags[2] != 0;
  // a teacher's row without mass (nothing kept, or -inf alone) has no part in the loss
  const double part = a.tail ? (double)a.lse[r] : tmax;
  const bool kd = flags[0] != 0 && a.alpha != 0.0 && part != -INFINITY;

  const T* zr = reinterpret_cast<const T*>(a.z) + r * a.ld;
  T* dr = GRAD ? reinterpret_cast<T*>(a.dz) + r * V : nullptr;
  constexpr int VE = kVE<T>;
  const int nchunk = (V + VE - 1) / VE;
  if (!kd && !label && !poison) {   // no term: the row's logits are not looked at
    if (t == 0) a.row_loss[r] = 0.f;
    if constexpr (GRAD) {
      float f[VE] = {};
      for (int c = t; c < nchunk; c += BLOCK) store_chunk(dr, c, V, f);
    }
    return;
  }
  if (poison) {
    if (t == 0) a.row_loss[r] = __builtin_nanf("");
    if constexpr (GRAD) {
      float f[VE];
      for (int j = 0; j < VE; ++j) f[j] = __builtin_nanf("");
      for (int c = t; c < nchunk; c += BLOCK) store_chunk(dr, c, V, f);
    }
    return;
  }

  double mass = 0, rest = 0, kd_loss = 0;
  if (kd) {
    double lt = part;
    if (!a.tail) {
      double s = 0;
      for (int k = t; k < K; k += BLOCK) s += cls[k] < 0 ? 0.0 : exp(p[k] - tmax);
      lt = tmax + log(block_fold<BLOCK>(s, red, SumOp()));
    }
    double s = 0;
    for (int k = t; k < K; k += BLOCK) {
      if (cls[k] < 0) {
        p[k] = 0;
        continue;
      }
      const double lp = p[k] - lt, pk = exp(lp);
      p[k] = pk;
      s += pk;
      if (pk > 0) kd_loss += pk * lp;
    }
    mass = block_fold<BLOCK>(s, red, SumOp());
    if (a.tail) {
      int n = 0;
      for (int i = t; i < words; i += BLOCK) n += __popc(mark[i]);
      n = block_fold<BLOCK>(n, reinterpret_cast<int*>(red), SumOp());
      rest = n < V ? 1.0 - mass : 0.0;
      if (rest < kDistillRest) rest = 0.0;
    }
  }

  // ---- the student's side
  Row<T, BLOCK, NC> row;
  row.load(zr, V);
  float m = -INFINITY;
  row.each([&](int, const float* f) {
#pragma unroll
    for (int j = 0; j < VE; ++j) m = fmaxf(m, f[j]);
  });
  m = block_fold<BLOCK>(m, reinterpret_cast<float*>(red), MaxOp());
  const bool one = label && (!kd || c_t != c_1);   // softmax at temperature 1 of its own
  const bool tail = kd && rest > 0;
  const float ct = kd ? c_t : c_1;
  float s_t = 0.f, s_k = 0.f, s_1 = 0.f;
  row.each([&](int c, const float* f) {
    float e[VE], sum = 0.f;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      e[j] = __builtin_amdgcn_exp2f((f[j] - m) * ct);
      sum += e[j];
    }
    const uint32_t bits = tail ? (mark8[c * VE >> 3] >> (c * VE & 7)) & ((1u << VE) - 1) : 0;
    if (bits) {
      float in = 0.f, out = 0.f;
#pragma unroll
      for (int j = 0; j < VE; ++j) (bits >> j & 1 ? in : out) += e[j];
      s_k += in;
      sum = out;
    }
    s_t += sum;
    if (one && kd) {
#pragma unroll
      for (int j = 0; j < VE; ++j) s_1 += __builtin_amdgcn_exp2f((f[j] - m) * c_1);
    }
  });
  const double left = block_fold<BLOCK>((double)s_t, red, SumOp());
  double total = left;
  if (tail) total += block_fold<BLOCK>((double)s_k, red, SumOp());
  double total1 = total;
  if (one && kd) total1 = block_fold<BLOCK>((double)s_1, red, SumOp());
  if (kd) {
    // (differences to the maximum: a row of the type's lowest value has no digits left beside it)
    for (int k = t; k < K; k += BLOCK)
      if (p[k] > 0) kd_loss -= p[k] * (((double)to_f(zr[cls[k]]) - (double)m) / a.temp);
    kd_loss = block_fold<BLOCK>(kd_loss, red, SumOp());
  }
  const double at2 = a.alpha * a.temp;
  if (t == 0) {
    double loss = 0;
    if (kd) {
      // kd_loss holds sum p (log p - (z - max)/T); log q = (z - max)/T - log s
      loss = kd_loss + mass * log(total);
      if (tail) loss += rest * (log(rest) - log(left / total));
      loss *= at2 * a.temp;
    }
    if (label) loss += (1 - a.alpha) * ((double)m - (double)to_f(zr[y]) + log(total1));
    a.row_loss[r] = (float)loss;
  }
  if constexpr (!GRAD) return;

  const double gs = a.grad_scale;
  const double A = kd ? gs * at2 * (mass + rest) / total : 0.0;
  const double B = tail && left > 0 ? gs * at2 * rest / left : 0.0;
  const double D = label ? gs * (1 - a.alpha) / total1 : 0.0;
  const bool both = kd && one;
  const float ca = (float)(both ? A - B : A - B + D), cd = (float)D;
  row.each([&](int c, const float* f) {
    float d[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      d[j] = ca * __builtin_amdgcn_exp2f((f[j] - m) * ct);
      if (both) d[j] += cd * __builtin_amdgcn_exp2f((f[j] - m) * c_1);
    }
    store_chunk(dr, c, V, d);
  });
  // the kept classes and the label's, after the plain values above are written
  __syncthreads();
  const bool dup = flags[1] != 0;
  auto fix = [&](int j, double pk) {
    const double z = (double)to_f(zr[j]) - (double)m;
    double g = -gs * at2 * pk;
    if (kd) g += A * exp(z / a.temp);
    if (label) g += D * exp(z) - (j == (int)y ? gs * (1 - a.alpha) : 0.0);
    dr[j] = static_cast<T>((float)g);
  };
  if (kd) {
    for (int k = t; k < K; k += BLOCK) {
      if (cls[k] < 0) continue;
      double pk = p[k];
      if (dup) {   // every entry of the class writes the same sum
        pk = 0;
        for (int i = 0; i < K; ++i)
          if (cls[i] == cls[k]) pk += p[i];
      }
      fix(cls[k], pk);
    }
  }
  if (label && t == 0 && !(kd && (mark[y >> 5] >> (y & 31) & 1))) {
    const double z = (double)to_f(zr[y]) - (double)m;
    double g = D * exp(z) - gs * (1 - a.alpha);
    if (kd) g += (A - B) * exp(z / a.temp);
    dr[y] = static_cast<T>((float)g);
  }
}

__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ v, int64_t n,
                                                           double scale, float* __restrict__ out) {
  __shared__ double red[16];
  double s = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += v[i];
  s = block_fold<1024>(s, red, SumOp());
  if (threadIdx.x == 0) out[0] = (float)(s * scale);
}

template <typename T>
__global__ __launch_bounds__(256) void scale_rows_kernel(T* __restrict__ dz, int64_t R, int V,
                                                         const float* __restrict__ s, int per_row) {
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const float g = s[r * per_row];
    if (g == 1.f) continue;
    T* p = dz + r * V;
    for (int c = threadIdx.x; c * kVE<T> < V; c += 256) {
      const uint4 u = load_chunk(p, c, V);
      float f[kVE<T>];
      unpack(u, f, T());
#pragma unroll
      for (int j = 0; j < kVE<T>; ++j) f[j] *= g;
      store_chunk(p, c, V, f);
    }
  }
}

// Threads and register chunks of a row: calls fn<BLOCK, NC>. again: long rows are read again
template <typename T, typename F>
void pick_row(int V, bool again, F&& fn) {
  using std::integral_constant;
  const int n = (V + kVE<T> - 1) / kVE<T>;
  if (n <= 64) fn(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (n <= 256) fn(integral_constant<int, 64>(), integral_constant<int, 4>());
  else if (n <= 1024) fn(integral_constant<int, 256>(), integral_constant<int, 4>());
  else if (n <= 2048) fn(integral_constant<int, 256>(), integral_constant<int, 8>());
  else if (again) fn(integral_constant<int, 1024>(), integral_constant<int, 0>());
  else if (n <= 8192) fn(integral_constant<int, 1024>(), integral_constant<int, 8>());
  else if (n <= 16384) fn(integral_constant<int, 1024>(), integral_constant<int, 16>());
  else fn(integral_constant<int, 1024>(), integral_constant<int, 0>());
}

template <typename F>
void pick_type(int type, F&& fn) {
  if (type == LOGIT_F32) fn(float());
  else if (type == LOGIT_BF16) fn(bf16());
  else fn(f16());
}

}  // namespace

void top_logits_launch(const void* z, int type, int64_t ld, int64_t R, int V, int k, double temp,
                       void* values, int32_t* indices, float* lse, hipStream_t st) {
  const float c = (float)(1.4426950408889634 / temp);
  pick_type(type, [&](auto tv) {
    using T = decltype(tv);
    if (V <= 64) {
      hipLaunchKernelGGL((top_small_kernel<T>), dim3((uint32_t)((R + 3) / 4)), dim3(256), 0, st,
                         reinterpret_cast<const T*>(z), ld, R, V, k, c, 1.0 / temp,
                         reinterpret_cast<T*>(values), indices, lse);
      return;
    }
    pick_row<T>(V, true, [&](auto block, auto nc) {
      constexpr int BLOCK = decltype(block)::value, NC = decltype(nc)::value;
      hipLaunchKernelGGL((top_logits_kernel<T, BLOCK, NC>), dim3((uint32_t)R), dim3(BLOCK), 0, st,
                         reinterpret_cast<const T*>(z), ld, V, k, c, 1.0 / temp,
                         reinterpret_cast<T*>(values), indices, lse);
    });
  });
}

void distill_launch(const DistillArgs& a, hipStream_t st) {
  const float c_t = (float)(1.4426950408889634 / a.temp), c_1 = 1.4426950408889634f;
  const size_t lds = (size_t)a.K * 12 + (size_t)((a.V + 31) / 32) * 4;
  pick_type(a.type, [&](auto tv) {
    using T = decltype(tv);
    pick_row<T>(a.V, false, [&](auto block, auto nc) {
      constexpr int BLOCK = decltype(block)::value, NC = decltype(nc)::value;
      if (a.dz)
        hipLaunchKernelGGL((distill_kernel<T, BLOCK, NC, true>), dim3((uint32_t)a.R), dim3(BLOCK),
                           lds, st, a, c_t, c_1);
      else
        hipLaunchKernelGGL((distill_kernel<T, BLOCK, NC, false>), dim3((uint32_t)a.R), dim3(BLOCK),
                           lds, st, a, c_t, c_1);
    });
  });
}

void distill_sum_launch(const float* row_loss, int64_t R, double scale, float* loss,
                        hipStream_t st) {
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, row_loss, R, scale, loss);
}

void scale_rows_launch(void* dz, int type, int64_t R, int V, const float* s, int per_row,
                       hipStream_t st) {
  const uint32_t grid = (uint32_t)std::min<int64_t>(R, 4096);
  pick_type(type, [&](auto tv) {
    using T = decltype(tv);
    hipLaunchKernelGGL((scale_rows_kernel<T>), dim3(grid), dim3(256), 0, st,
                       reinterpret_cast<T*>(dz), R, V, s, per_row);
  });
}

}  // namespace pca
