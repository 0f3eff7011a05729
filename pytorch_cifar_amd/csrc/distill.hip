// Distillation from a teacher's top logits: the K largest logits a row with the row's
// log-sum-exp (top_logits), and the loss of a student's logits against them with its gradient
// (distill_*). Rows are [R][V] in fp32 / bf16 / fp16 with any row stride; one workgroup a row.
//
// Rows of up to 1024 chunks of 16 bytes stay in registers between their passes; longer ones are
// streamed in one pass (sums, selection), which the gradient follows with a second one.
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
  const T* p = row + (uint32_t)c * kVE<T>;
  if ((c + 1) * kVE<T> <= V) {
    __builtin_memcpy(&u, p, 16);
    return u;
  }
  float f[kVE<T>];
#pragma unroll
  for (int i = 0; i < kVE<T>; ++i) f[i] = c * kVE<T> + i < V ? to_f(p[i]) : -INFINITY;
  return pack(f, T());
}

// (STREAM: past the caches, which then keep the rows that are read again: distill_loss with gradient,
// 4096 x 128000 bf16, 514 -> 478 us)
template <bool STREAM = false, typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ row, int c, int V, const float* f,
                                            bool whole = false) {
  const uint4 u = pack(f, T());
  T* p = row + (uint32_t)c * kVE<T>;
  if (whole || (c + 1) * kVE<T> <= V) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
    if constexpr (STREAM)
      __builtin_nontemporal_store((u32x4){u.x, u.y, u.z, u.w}, reinterpret_cast<u32x4*>(p));
    else
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
  // fn(chunk number, its elements as float, whether it is known to be whole)
  template <typename F>
  __device__ __forceinline__ void each(F&& fn) const {
    constexpr std::integral_constant<bool, true> whole;
    constexpr std::integral_constant<bool, false> any;
    float f[kVE<T>];
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = threadIdx.x + i * BLOCK;
        if (c < n) {
          // (opaque, so that the passes unpack anew: kept across them, the floats spill)
          uint4 v = u[i];
          asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
          unpack(v, f, T());
          fn(c, f, any);
        }
      }
    } else {
      // (the next two chunks are on their way while two are worked on; without the barrier the
      // compiler waits for each load where it is issued)
      constexpr int U = 2;
      const int rounds = V / kVE<T> / BLOCK / U;
      int c = threadIdx.x;
      uint4 v[U], next[U];
      auto fetch = [&](uint4* to, int at) {
#pragma unroll
        for (int j = 0; j < U; ++j)
          __builtin_memcpy(&to[j], p + (uint32_t)(at + j * BLOCK) * kVE<T>, 16);
      };
      if (rounds > 0) fetch(v, c);
      for (int i = 0; i < rounds; ++i, c += U * BLOCK) {
        if (i + 1 < rounds) fetch(next, c + U * BLOCK);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < U; ++j) {
          unpack(v[j], f, T());
          fn(c + j * BLOCK, f, whole);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = next[j];
      }
      for (; c < n; c += BLOCK) {
        unpack(load_chunk(p, c, V), f, T());
        fn(c, f, any);
      }
    }
  }
};

// the largest of a chunk (a NaN is passed over) and m
template <int N>
__device__ __forceinline__ float chunk_max(const float* f, float m) {
#pragma unroll
  for (int j = 0; j < N; j += 2)
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(f[j]), "v"(f[j + 1]));
  return m;
}

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

// v of N neighbouring lanes, in a fixed order
template <int N = 64, typename A, typename Op>
__device__ __forceinline__ A wave_fold(A v, Op op) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  return v;
}

// v of all threads, folded in a fixed order; every thread gets the result. red: BLOCK/64 values.
template <int BLOCK, typename A, typename Op>
__device__ __forceinline__ A block_fold(A v, A* red, Op op) {
  v = wave_fold(v, op);
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

// Sum of 2^(x - base) over a thread's x = z c, in one pass without the maximum: a term costs one
// multiply-add, the exponential and the add. The base is the first chunk's largest x, as a whole number:
// sums of different bases are joined by exact powers of two, which meet the sum before it is rounded (a
// thread's may be 2^127 above its base, and the base more than that below the row's: 2^-130 as a factor
// would be zero). 2^60 above and all below it is room for what follows. A row that leaves it (a first
// chunk of masked classes, |x| past 2^22, infinities, NaN) is summed again against its maximum (`plain`
// below).
//
// x - base is rounded to 24 bits, and c = log2(e) / T is one fp32 number: together a term is off by some
// |x - base| 2^-24 relative, the row's largest too, whose distance from its maximum would be exact.
constexpr float kNoBase = -4194304.f, kFar = 4194304.f;
constexpr double kMost = 1152921504606846976.0;   // 2^60

// (What was summed before a base was found is relative to kNoBase: masks of some -2^22, or nothing.
// scale(d): shift those sums by 2^d)
template <int N, typename F>
__device__ __forceinline__ void first_base(float& base, const float* f, float c, F&& scale) {
  if (base != kNoBase) return;
  const float x = chunk_max<N>(f, f[0]) * c;
  if (x > kNoBase && x < kFar) {
    base = rintf(x);
    scale((int)(kNoBase - base));
  }
}

__device__ __forceinline__ float term(float z, float c, float base) {
  return __builtin_amdgcn_exp2f(fmaf(z, c, -base));
}
// the same against a maximum m that may be anything
__device__ __forceinline__ float term_at(float z, float m, float c) {
  return __builtin_amdgcn_exp2f((z - m) * c);
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
__device__ __forceinline__ float float_of(uint32_t bits) {   // of order_bits
  return __uint_as_float(bits & 0x80000000u ? bits ^ 0x80000000u : ~bits);
}
__device__ __forceinline__ uint64_t order_key(float f, int idx) {
  return ((uint64_t)order_bits(f) << kIdxBits) | (uint32_t)(kDistillMaxClasses - 1 - idx);
}
__device__ __forceinline__ int key_index(uint64_t k) {
  return kDistillMaxClasses - 1 - (int)(k & (kDistillMaxClasses - 1));
}

constexpr int kList = 2048;   // candidates that are ranked at most
constexpr int kCount = 16;    // comparisons a thread up to which their places are counted
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
    row.each([&](int ch, const float* f, auto) {
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

// The same over the maxima of parts of the row (one wave, M / 64 of them a lane; 0: no such part): at
// least k logits are as large as the k-th largest of them, and in a row in no particular order few more.
template <int M>
__device__ uint32_t bound_of_maxima(const uint32_t* maxima, int k, int spare) {   // at most k + spare maxima reach it, if they differ
  constexpr int N = M / 64;
  uint32_t v[N], least = ~0u, most = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = maxima[threadIdx.x + i * 64];
    least = min(least, v[i] ? v[i] : ~0u), most = max(most, v[i]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    least = min(least, (uint32_t)__shfl_xor((int)least, o, 64));
    most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
  }
  uint64_t lo = least, hi = most + 1ull;
  int n = M;
  while (n > k + spare && hi - lo > 1) {
    const uint32_t mid = (uint32_t)(lo + (hi - lo) / 2);
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += __popcll(__ballot(v[i] >= mid));
    if (c >= k) lo = mid, n = c;
    else hi = mid;
  }
  return (uint32_t)lo;
}

// the wave's keys in descending order, one a lane (bitonic)
__device__ __forceinline__ uint64_t wave_sort(uint64_t key) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int size = 2; size <= 64; size *= 2) {
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2) {
      const uint64_t other = __shfl_xor(key, d, 64);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0);
      key = (key > other) == larger ? key : other;
    }
  }
  return key;
}

// One pass over the row gives each thread its maximum, its sum of exponentials, and, where the row is
// long, the candidates: a bound on the first four chunks of the threads, low enough that with some
// three standard deviations to spare k logits of a row in random order reach it, is known after them,
// and what reaches it is put on a list as it comes by. A row whose list is short or overflows (one
// in some other order) takes the chunks of the threads whose maximum reaches a bound on all maxima; a
// row that defeats this too (NaN, many equal logits, k near the number of threads) is halved by
// counting.
//
// Long rows are bound by the read: 2048 x 128000 bf16, k 64, in 98 us (5.4 TB/s; a large copy reaches
// 4.85), few rows by the steps of one: 509 x 32003 fp32, k 256, 26 us. Places counted over all candidates
// took 34 there, and 281 us of 2048 x 128000 with k 512, now 168.
template <typename T, int BLOCK, int NC>
__global__ __launch_bounds__(BLOCK)
__attribute__((amdgpu_waves_per_eu(NC == 0 ? 8 : 1))) void top_logits_kernel(
    const T* __restrict__ z, int64_t ld, int V, int k, float c, double inv_t,
    int cap, T* __restrict__ values, int32_t* __restrict__ indices, float* __restrict__ lse) {
  __shared__ double red[16];
  constexpr int NW = BLOCK / 64, VE = kVE<T>;
  __shared__ struct { float m, base, s; } part[NW];
  constexpr int M = NC > 0 ? BLOCK * NC : BLOCK;   // parts: a chunk each, or a thread's chunks
  __shared__ uint32_t maxima[M];
  __shared__ uint16_t who[BLOCK];
  extern __shared__ uint64_t list[];   // [cap]
  __shared__ uint32_t found, who_n, bound;
  const int64_t r = blockIdx.x;
  // (a wave finds a bound of few maxima sooner, but not one near their number: 8388 x 8000 bf16 by 256
  // threads' / 1000 chunks' maxima, k 5 44 / 63 us, k 192 235 / 106)
  const bool chunks = NC > 0 && k > BLOCK / 2;
  Row<T, BLOCK, NC> row;
  row.load(z + r * ld, V);

  float m = -INFINITY, base = kNoBase, s = 0.f;
  auto found_base = [&](int d) { s = ldexpf(s, d); };
  auto take = [&](const float* f) {
    const float cm = chunk_max<VE>(f, -INFINITY);
    m = fmaxf(m, cm);
#pragma unroll
    for (int j = 0; j < VE; ++j) s += term(f[j], c, base);
    return cm;
  };
  // the logits of a chunk that reach a bound (no NaN among them); false once the list is full.
  // (compared as they are: most of a wave's chunks hold one such logit or none)
  auto collect = [&](int ch, const float* f, float low) {
    bool room = true;
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (f[j] >= low) {
        const uint32_t at = atomicAdd(&found, 1u);
        if (at < cap) list[at] = order_key(f[j], ch * VE + j);
        else room = false;
      }
    return room;
  };
  if constexpr (NC > 0) {
    if (chunks) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int ch = threadIdx.x + i * BLOCK;
        if (ch >= row.n) maxima[ch] = 0;
      }
    }
    row.each([&](int ch, const float* f, auto) {
      first_base<VE>(base, f, c, found_base);
      const float cm = take(f);
      if (chunks) maxima[ch] = order_bits(cm);
    });
    if (threadIdx.x == 0) found = who_n = 0;
  } else {
    constexpr int A = 4, U = 2;   // chunks of the first part; loads in flight after it
    uint4 v[A], next[U];
    float f[VE];
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < A; ++j) v[j] = load_chunk(row.p, min(t + j * BLOCK, row.n - 1), V);
    auto fetch = [&](int at) {
#pragma unroll
      for (int j = 0; j < U; ++j) next[j] = load_chunk(row.p, min(at + j * BLOCK, row.n - 1), V);
    };
    fetch(t + A * BLOCK);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < A; ++j)
      if (t + j * BLOCK < row.n) {
        unpack(v[j], f, T());
        first_base<VE>(base, f, c, found_base);
        take(f);
      }
    maxima[t] = order_bits(m);
    if (t == 0) found = who_n = 0;
    __syncthreads();
    if (t < 64) {
      const float share = k * fminf(1.f, A * BLOCK / (float)row.n);
      const int j = row.n > A * BLOCK ? (int)(share + 3.f * sqrtf(share)) + 3 : k;
      const uint32_t least = bound_of_maxima<BLOCK>(maxima, min(j, BLOCK - 1), j / 8 + 2);
      if (t == 0) bound = least;
    }
    __syncthreads();
    const float low = float_of(bound);
    // (nothing is put down for a bound of -inf: a masked part)
    bool room = low > -INFINITY;
#pragma unroll
    for (int j = 0; j < A; ++j)
      if (t + j * BLOCK < row.n) {
        unpack(v[j], f, T());
        if (room && chunk_max<VE>(f, -INFINITY) >= low) room = collect(t + j * BLOCK, f, low);
      }
    for (int ch = t + A * BLOCK; ch < row.n; ch += U * BLOCK) {
#pragma unroll
      for (int j = 0; j < U; ++j) v[j] = next[j];
      fetch(ch + U * BLOCK);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (ch + j * BLOCK < row.n) {
          unpack(v[j], f, T());
          if (take(f) >= low && room) room = collect(ch + j * BLOCK, f, low);
        }
    }
    __syncthreads();   // (the first part's bound was read; maxima are written again)
  }
  const uint32_t mine = order_bits(m);
  if (!chunks) maxima[threadIdx.x] = mine;
  const float wb = wave_fold(base, MaxOp());
  const float ws = wave_fold(ldexpf(s, (int)(base - wb)), SumOp());
  m = wave_fold(m, MaxOp());
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = {m, wb, ws};
  __syncthreads();
  // (a wave's part a lane: every wave joins them for itself)
  const auto mp = part[threadIdx.x & (NW - 1)];
  float all = wave_fold<NW>(mp.m, MaxOp());
  const float b = wave_fold<NW>(mp.base, MaxOp());
  double sum = wave_fold<NW>(ldexp((double)mp.s, (int)(mp.base - b)), SumOp());
  bool finite = true;   // no NaN in the row
  if (sum > 0 && sum < kMost) {
    if (threadIdx.x == 0) lse[r] = (float)(((double)b + log2(sum)) * 0.6931471805599453);
  } else {
    // (a row of -inf: log 0; one with +inf: log inf; NaN stays)
    if (isinf(all)) all = 0.f;
    s = 0.f;
    row.each([&](int, const float* f, auto) {
#pragma unroll
      for (int j = 0; j < kVE<T>; ++j) s += term_at(f[j], all, c);
    });
    sum = block_fold<BLOCK>((double)s, red, SumOp());
    finite = sum == sum;
    if (threadIdx.x == 0) lse[r] = (float)((double)all * inv_t + log(sum));
  }

  bool few = finite && (int)found >= k && found <= cap;
  if (!few && finite && k <= (chunks ? row.n / 8 * 5 : BLOCK / 4 * 3)) {   // (a maximum passes over NaN)
    __syncthreads();
    if (threadIdx.x < 64) {
      const uint32_t v = chunks ? bound_of_maxima<M>(maxima, k, k / 4 + 8)
                                : bound_of_maxima<BLOCK>(maxima, k, k / 4 + 8);
      if (threadIdx.x == 0) bound = v, found = 0;
    }
    __syncthreads();
    const uint32_t least = bound;
    const float low = float_of(least);
    // (a bound of -inf would take in what pads the row's last chunk)
    if (chunks) {
      if (low > -INFINITY)
        row.each([&](int ch, const float* f, auto) {
          if (chunk_max<VE>(f, -INFINITY) >= low) collect(ch, f, low);
        });
    } else {
      if (mine >= least && low > -INFINITY) who[atomicAdd(&who_n, 1u)] = threadIdx.x;
      __syncthreads();
      // the chunks of those threads, read again by all threads at once
      const int per = (row.n + BLOCK - 1) / BLOCK, items = (int)who_n * per;
      for (int w = threadIdx.x; w < items; w += BLOCK) {
        const int ch = who[w / per] + w % per * BLOCK;
        if (ch >= row.n) continue;
        float f[VE];
        unpack(load_chunk(row.p, ch, V), f, T());
        collect(ch, f, low);
      }
    }
    __syncthreads();
    few = (int)found >= k && found <= cap;
  }
  if (!few) {
    __syncthreads();
    if (threadIdx.x == 0) found = 0;
    const uint64_t b = bound_of_keys(row, k, reinterpret_cast<int*>(red));
    __syncthreads();
    row.each([&](int ch, const float* f, auto) {
#pragma unroll
      for (int j = 0; j < kVE<T>; ++j) {
        const int idx = ch * kVE<T> + j;
        const uint64_t key = order_key(f[j], idx);
        if (idx < V && key >= b) {
          const uint32_t at = atomicAdd(&found, 1u);
          if (at < cap) list[at] = key;
        }
      }
    });
    __syncthreads();
  }
  const int n = (int)found;
  auto put = [&](uint64_t key, int at) {
    if (at >= k) return;
    const int idx = key_index(key);
    values[r * k + at] = row.p[idx];
    indices[r * k + at] = idx;
  };
  // A candidate's place is the number of candidates before it.
  if (n * n <= kCount * BLOCK) {   // counted by `parts` lanes each
    int parts = 1;
    while (parts < 64 && 2 * parts * n <= BLOCK) parts *= 2;
    const int part_of = threadIdx.x & (parts - 1);
    for (int i0 = 0; i0 < n; i0 += BLOCK / parts) {
      const int i = i0 + threadIdx.x / parts;
      const uint64_t key = i < n ? list[i] : 0;
      int at = 0;
#pragma unroll 8
      for (int j = part_of; j < n; j += parts) at += list[j] > key;
      for (int o = 1; o < parts; o *= 2) at += __shfl_xor(at, o, 64);
      if (i < n && part_of == 0) put(key, at);
    }
  } else {   // in its wave's 64, which are sorted, and by search in every other 64
    const int lane = threadIdx.x & 63, blocks = (n + 63) / 64;
    for (int b = threadIdx.x >> 6; b < blocks; b += NW)
      list[64 * b + lane] = wave_sort(64 * b + lane < n ? list[64 * b + lane] : 0);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += BLOCK) {
      const uint64_t key = list[i];
      int at = i & 63;
#pragma unroll 4
      for (int o = 1; o < blocks; ++o) {
        const int b = i / 64 + o;
        const uint64_t* other = list + 64 * (b < blocks ? b : b - blocks);
        int before = 0;
#pragma unroll
        for (int half = 32; half > 0; half /= 2) before += other[before + half - 1] > key ? half : 0;
        at += before + (other[before] > key);
      }
      put(key, at);
    }
  }
}

// Rows of up to 64 classes: a wave each, a class a lane. The place of a logit is the number of
// logits before it, counted over the lanes. Bound by the launch: 1024 x 10 fp32 6 us.
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
// Row of the loss, with q = softmax(z/T), e_j = exp(z_j/T) and s = sum e, both relative to a base:
//   KD   = sum_k p_k (log p_k - log q_k) + rest (log rest - log q_rest)
//   loss = alpha T^2 KD + (1 - alpha) (lse(z) - z_y)
//   d/dz_j = e_j A - [not kept] e_j B - [kept] alpha T p_j + (1 - alpha)(softmax(z)_j - [j = y])
// with A = alpha T (sum p + rest) / s and B = alpha T rest / s_rest, s_rest the sum of e over the
// classes that are not kept: summed by itself (a difference s - s_kept would lose it where the
// kept classes hold nearly all). The K values of the teacher's side are computed in 64 bits: what
// is left of its mass, 1 - sum p, is a difference.
//
// Where the kept classes stand so far above all others (41 in z/T) that s_rest is less than 2^-60 of the
// base, the rest is summed again against its own maximum, which costs two more passes: terms below 2^-126
// of a base are zero in 32 bits, and so shares e_j / s_rest below 2^-66 are all that is lost.
//
// A bit a class marks the kept ones (LDS, V / 8 bytes). It gives s_rest, and finds an index that
// a row names twice: its entries are then gathered for each of them.
//
// Bound by the read and the write of a row; the read for the gradient finds it in registers or in the
// cache behind the L2s. 4096 x 128000 bf16, k 64, with rest and labels, 480 us (4.4 TB/s of 2.1 GB);
// the loss alone of 2000 x 50257 fp16 50 us (4.0 TB/s).
//
// The loss's own gradient multiplies a row's in fp32 and 64 bits, before its one rounding: under a loss
// scale (fp16) most shares of a long row have no 16-bit number without it.
//
// The label's softmax is at temperature 1. Where T is 2 or 4 its exponentials are powers of those at
// T, which saves the second quarter-rate instruction of a class and pass.
constexpr double kFaint = 1 / kMost;   // 2^-60
struct Sums {
  float base, base1;         // at T, at temperature 1
  float rest, kept, one;     // of e over the classes not kept, the kept ones; of all at 1
};

template <typename T, int BLOCK, int NC, bool GRAD>
__global__ __launch_bounds__(BLOCK)
__attribute__((amdgpu_waves_per_eu(NC == 0 ? 8 : 1))) void distill_kernel(DistillArgs a, float c_t) {
  extern __shared__ char smem[];
  constexpr int NW = BLOCK / 64, VE = kVE<T>;
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr double kLn2 = 0.6931471805599453;
  __shared__ double red[16];
  __shared__ Sums part[NW];
  __shared__ double side[3];   // the teacher's side: sum p, rest, sum p log p
  __shared__ int flags[4];     // kept entries with mass, an index twice, an index past the classes
  const int64_t r = blockIdx.x;
  const int V = a.V, K = a.K, t = threadIdx.x, wave = t >> 6;
  const float seed = GRAD && a.seed ? a.seed[r * a.seed_rows] : 1.f;
  if (GRAD && a.keep && seed == 1.f) return;
  double* p = reinterpret_cast<double*>(smem);          // [K] the teacher's probabilities
  float* zk = reinterpret_cast<float*>(p + K);          // [K] the student's logits there
  int* cls = reinterpret_cast<int*>(zk + K);            // [K] their classes, -1: not kept
  uint32_t* mark = reinterpret_cast<uint32_t*>(cls + K);
  const uint8_t* mark8 = reinterpret_cast<const uint8_t*>(mark);
  const T* zr = reinterpret_cast<const T*>(a.z) + r * a.ld;

  Row<T, BLOCK, NC> row;
  row.load(zr, V);
  int64_t y = a.target ? a.target[r] : a.ignore_index;
  const bool label = a.target && y != a.ignore_index && a.alpha != 1.0;
  bool poison = label && (y < 0 || y >= V);
  if (poison || !label) y = 0;
  const float zy = to_f(zr[y]);
  const float lse = a.tail ? a.lse[r] : 0.f;

  for (int i = t; i < (V + 31) / 32; i += BLOCK) mark[i] = 0;
  if (t < 4) flags[t] = 0;
  __syncthreads();
  int mass_here = 0, twice = 0, bad = 0;
  for (int k = t; k < K; k += BLOCK) {
    const int64_t at = r * K + k;
    const int64_t idx = a.index64 ? reinterpret_cast<const int64_t*>(a.indices)[at]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.indices)[at];
    const float v = a.value_type == LOGIT_F32 ? reinterpret_cast<const float*>(a.values)[at]
                    : a.value_type == LOGIT_BF16
                        ? to_f(reinterpret_cast<const bf16*>(a.values)[at])
                        : to_f(reinterpret_cast<const f16*>(a.values)[at]);
    const bool in = idx >= 0 && idx < V;
    if (idx >= V) bad = 1;
    if (in) {
      const uint32_t bit = 1u << (idx & 31);
      if (atomicOr(&mark[idx >> 5], bit) & bit) twice = 1;
      mass_here |= a.tail || v != -INFINITY;
      zk[k] = to_f(zr[idx]);
    }
    cls[k] = in ? (int)idx : -1;
    p[k] = in ? (double)v / a.temp : -INFINITY;
  }
  if (mass_here) flags[0] = 1;
  if (twice) flags[1] = 1;
  if (bad) flags[2] = 1;
  __syncthreads();
  poison |= flags[2] != 0;
  // a teacher's row without mass (nothing kept, or -inf alone) has no part in the loss
  const bool kd = flags[0] != 0 && a.alpha != 0.0 && lse != -INFINITY;
  T* dr = GRAD ? reinterpret_cast<T*>(a.dz) + r * V : nullptr;
  if (poison || (!kd && !label)) {   // without a term the row's logits do not count
    const float v = poison ? __builtin_nanf("") : 0.f;
    if (t == 0 && a.row_loss) a.row_loss[r] = v;
    if constexpr (GRAD) {
      float f[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) f[j] = v;
      for (int c = t; c * VE < V; c += BLOCK) store_chunk(dr, c, V, f);
    }
    return;
  }

  // ---- the teacher's side, by the first wave (the others go on)
  if (wave == 0 && kd) {
    double lt = lse;
    if (!a.tail) {
      double m = -INFINITY, s = 0;
      for (int k = t; k < K; k += 64) m = p[k] != p[k] ? p[k] : fmax(m, p[k]);
      m = wave_fold(m, MaxOp());
      for (int k = t; k < K; k += 64) s += cls[k] < 0 ? 0.0 : exp(p[k] - m);
      lt = m + log(wave_fold(s, SumOp()));
    }
    double s = 0, plogp = 0;
    for (int k = t; k < K; k += 64) {
      const double lp = p[k] - lt, pk = cls[k] < 0 ? 0.0 : exp(lp);
      p[k] = pk;
      s += pk;
      if (pk > 0) plogp += pk * lp;
    }
    s = wave_fold(s, SumOp());
    plogp = wave_fold(plogp, SumOp());
    double rest = 0;
    if (a.tail) {
      bool other = true;   // is any class not kept?
      if (K >= V) {
        int n = 0;
        for (int i = t; i < (V + 31) / 32; i += 64) n += __popc(mark[i]);
        other = wave_fold(n, SumOp()) < V;
      }
      rest = other ? 1.0 - s : 0.0;
      if (rest < kDistillRest) rest = 0.0;
    }
    if (t == 0) side[0] = s, side[1] = rest, side[2] = plogp;
  }

  // ---- the student's sums. power: exponentials at temperature 1 as that power of those at T
  const bool one = label && (!kd || a.temp != 1.0);   // a softmax at temperature 1 of its own
  const bool two = one && kd;
  const float ct = kd ? c_t : kLog2e;
  const int power = two ? (a.temp == 2.0 ? 2 : a.temp == 4.0 ? 4 : 0) : 0;
  const bool tail = kd && a.tail;
  Sums s = {kNoBase, kNoBase, 0.f, 0.f, 0.f};
  float base1 = kNoBase;
  // e: the chunk's exponentials at T
  auto add = [&](int c, const float* e) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < VE; ++j) sum += e[j];
    const uint32_t bits = tail ? (mark8[c * VE >> 3] >> (c * VE & 7)) & ((1u << VE) - 1) : 0;
    if (bits) {
      float in = 0.f, out = 0.f;
#pragma unroll
      for (int j = 0; j < VE; ++j) (bits >> j & 1 ? in : out) += e[j];
      s.kept += in;
      sum = out;
    }
    s.rest += sum;
    if (power == 2) {
#pragma unroll
      for (int j = 0; j < VE; ++j) s.one = fmaf(e[j], e[j], s.one);
    } else if (power == 4) {
#pragma unroll
      for (int j = 0; j < VE; ++j) s.one = fmaf(e[j] * e[j], e[j] * e[j], s.one);
    }
  };
  row.each([&](int c, const float* f, auto) {
    first_base<VE>(s.base, f, ct, [&](int d) {
      s.rest = ldexpf(s.rest, d);
      s.kept = ldexpf(s.kept, d);
      if (power) s.one = ldexpf(s.one, power * d);
    });
    float e[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) e[j] = term(f[j], ct, s.base);
    add(c, e);
    if (two && !power) {
      first_base<VE>(base1, f, kLog2e, [&](int d) { s.one = ldexpf(s.one, d); });
#pragma unroll
      for (int j = 0; j < VE; ++j) s.one += term(f[j], kLog2e, base1);
    }
  });
  if (power) base1 = s.base * power;
  // sums of the threads, in a fixed order: each wave's at its own base, then all of them
  const float wb = wave_fold(s.base, MaxOp()), wb1 = wave_fold(base1, MaxOp());
  auto join = [&](int d, int d1) {
    const Sums w = {wb, wb1, wave_fold(ldexpf(s.rest, d), SumOp()), wave_fold(ldexpf(s.kept, d), SumOp()),
                    wave_fold(ldexpf(s.one, d1), SumOp())};
    __syncthreads();
    if ((t & 63) == 0) part[wave] = w;
    __syncthreads();
  };
  join((int)(s.base - wb), (int)(base1 - wb1));
  // (a wave's part a lane: every wave joins them for itself)
  Sums v = part[t & (NW - 1)];
  const float b = wave_fold<NW>(v.base, MaxOp()), b1 = wave_fold<NW>(v.base1, MaxOp());
  double left = 0, inner = 0, total1 = 0;
  auto total = [&](int d, int d1) {
    left = wave_fold<NW>(ldexp((double)v.rest, d), SumOp());
    if (tail) inner = wave_fold<NW>(ldexp((double)v.kept, d), SumOp());
    if (two) total1 = wave_fold<NW>(ldexp((double)v.one, d1), SumOp());
  };
  total((int)(v.base - b), (int)(v.base1 - b1));
  // plain: exponentials against the row's maximum, for both temperatures
  const double sum = left + inner;
  const bool plain = !(sum > 0 && sum < kMost && (!two || (total1 > 0 && total1 < kMost)));
  float m = 0.f;
  if (plain) {
    m = -INFINITY;
    row.each([&](int, const float* f, auto) { m = chunk_max<VE>(f, m); });
    m = block_fold<BLOCK>(m, reinterpret_cast<float*>(red), MaxOp());
    s = {};
    row.each([&](int c, const float* f, auto) {
      float e[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) e[j] = term_at(f[j], m, ct);
      add(c, e);
      if (two && !power) {
#pragma unroll
        for (int j = 0; j < VE; ++j) s.one += term_at(f[j], m, kLog2e);
      }
    });
    join(0, 0);
    v = part[t & (NW - 1)];
    total(0, 0);
  }
  const double all = left + inner;
  if (!two) total1 = all;
  const double mass = kd ? side[0] : 0, rest = kd ? side[1] : 0;
  // log of the rest's share; far: its exponentials are against mr, the largest of its classes
  double lrest = 0;
  float mr = -INFINITY;
  bool far = rest > 0 && left < kFaint;
  if (far) {
    auto others = [&](auto&& fn) {
      row.each([&](int c, const float* f, auto) {
        const uint32_t bits = mark8[c * VE >> 3] >> (c * VE & 7);
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (!(bits >> j & 1)) fn(f[j]);
      });
    };
    others([&](float z) { mr = fmaxf(mr, z); });
    mr = block_fold<BLOCK>(mr, reinterpret_cast<float*>(red), MaxOp());
    far = mr != -INFINITY;   // (no mass at all: log 0)
    if (far) {
      float sr = 0.f;
      others([&](float z) { sr += term_at(z, mr, ct); });
      left = block_fold<BLOCK>((double)sr, red, SumOp());
      const double x = plain ? ((double)mr - (double)m) * (double)ct : (double)mr * (double)ct - (double)b;
      lrest = x * kLn2 + log(left) - log(all);
    }
  }
  if (rest > 0 && !far) lrest = log(left / all);
  const double at2 = a.alpha * a.temp;

  if (wave == 0) {
    // log2 of a class's share, from the same constants as its exponential
    double kl = 0;
    if (kd) {
      for (int k = t; k < K; k += 64) {
        if (!(p[k] > 0)) continue;
        const double x = plain ? ((double)zk[k] - (double)m) * (double)ct
                               : (double)zk[k] * (double)ct - (double)b;
        kl -= p[k] * x;
      }
      kl = wave_fold(kl, SumOp()) * kLn2 + side[2] + mass * log(all);
      if (rest > 0) kl += rest * (log(rest) - lrest);
    }
    if (t == 0 && a.row_loss) {
      double loss = kd ? kl * at2 * a.temp : 0;
      if (label) {
        const float c1 = two ? kLog2e : ct;
        const double x = plain ? ((double)zy - (double)m) * (double)c1
                               : (double)zy * (double)c1 - (double)(two ? b1 : b);
        loss += (1 - a.alpha) * (log(total1) - x * kLn2);
      }
      a.row_loss[r] = (float)loss;
    }
  }
  if constexpr (!GRAD) return;

  const double gs = (double)a.grad_scale * seed;
  const double A = kd ? gs * at2 * (mass + rest) / all : 0.0;
  const double Br = rest > 0 && left > 0 ? gs * at2 * rest / left : 0.0;
  const double B = far ? 0.0 : Br;   // (far: a term of its own, at its own base)
  const double D = label ? gs * (1 - a.alpha) / total1 : 0.0;
  const float ca = (float)(two ? A - B : A - B + D), cd = (float)D;
  if (far) {
    row.each([&](int c, const float* f, auto whole) {
      float g[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        g[j] = ca * (plain ? term_at(f[j], m, ct) : term(f[j], ct, b)) - (float)Br * term_at(f[j], mr, ct);
        if (two) g[j] += cd * (plain ? term_at(f[j], m, kLog2e) : term(f[j], kLog2e, b1));
      }
      store_chunk<NC == 0>(dr, c, V, g, whole);
    });
  } else if (plain) {
    row.each([&](int c, const float* f, auto whole) {
      float g[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        g[j] = ca * term_at(f[j], m, ct);
        if (two) g[j] += cd * term_at(f[j], m, kLog2e);
      }
      store_chunk<NC == 0>(dr, c, V, g, whole);
    });
  } else {
    row.each([&](int c, const float* f, auto whole) {
      float g[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) g[j] = term(f[j], ct, b);
      if (!two) {
#pragma unroll
        for (int j = 0; j < VE; ++j) g[j] *= ca;
      } else if (power == 2) {
        // (A - B) e + D e^2
#pragma unroll
        for (int j = 0; j < VE; ++j) g[j] *= fmaf(cd, g[j], ca);
      } else if (power == 4) {
#pragma unroll
        for (int j = 0; j < VE; ++j) g[j] *= fmaf(cd * g[j], g[j] * g[j], ca);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) g[j] = fmaf(cd, term(f[j], kLog2e, b1), ca * g[j]);
      }
      store_chunk<NC == 0>(dr, c, V, g, whole);
    });
  }
  // the kept classes and the label's, after the plain values above are written
  __syncthreads();
  const bool dup = flags[1] != 0;
  auto fix = [&](int j, float z, double share, double pk, bool kept) {
    double g = -gs * at2 * pk;
    if (far && !kept) g -= Br * term_at(z, mr, ct);
    if (kd) g += share * (plain ? term_at(z, m, ct) : term(z, ct, b));
    if (label) {
      const float c1 = two ? kLog2e : ct;
      g += D * (plain ? term_at(z, m, c1) : term(z, c1, two ? b1 : b));
      if (j == (int)y) g -= gs * (1 - a.alpha);
    }
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
      fix(cls[k], zk[k], A, pk, true);
    }
  }
  if (label && t == 0 && !(kd && (mark[y >> 5] >> (y & 31) & 1))) fix((int)y, zy, A - B, 0.0, false);
}

__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ v, int64_t n,
                                                           double scale, float* __restrict__ out) {
  __shared__ double red[16];
  double s = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += v[i];
  s = block_fold<1024>(s, red, SumOp());
  if (threadIdx.x == 0) out[0] = (float)(s * scale);
}

// Threads and register chunks of a row of n chunks: calls fn<BLOCK, NC>. Up to 1024 chunks are held in
// registers; longer rows are streamed by `threads` threads.
template <typename F>
void pick_row(int n, int threads, F&& fn) {
  using std::integral_constant;
  if (threads >= 1024) fn(integral_constant<int, 1024>(), integral_constant<int, 0>());
  else if (n > 1024 && threads == 512) fn(integral_constant<int, 512>(), integral_constant<int, 0>());
  else if (n > 1024) fn(integral_constant<int, 256>(), integral_constant<int, 0>());
  else if (threads > 64 || n > 256) fn(integral_constant<int, 256>(), integral_constant<int, 4>());
  else if (n > 64) fn(integral_constant<int, 64>(), integral_constant<int, 4>());
  else fn(integral_constant<int, 64>(), integral_constant<int, 1>());
}

// Rows that do not give each of the 256 CUs `fill` threads take more threads each. top_logits, fill 1024:
// 509 rows of 32003 fp32, k 16, by 256 / 512 / 1024 threads 21 / 17 / 19 us, k 256 37 / 26 / 26.
int few_rows(int64_t R, int threads, int fill) {
  while (threads < 1024 && R * threads * 2 <= 256 * fill) threads *= 2;
  return threads;
}

// A launch holds less than 2^32 threads: fn(first, rows) for each part of the R rows that one can take.
template <typename F>
void row_parts(int64_t R, F&& fn) {
  constexpr int64_t kRows = 1 << 21;   // (of up to 1024 threads)
  for (int64_t r = 0; r < R; r += kRows) fn(r, std::min(kRows, R - r));
}

template <typename F>
void pick_type(int type, F&& fn) {
  if (type == LOGIT_F32) fn(float());
  else if (type == LOGIT_BF16) fn(bf16());
  else fn(f16());
}

}  // namespace

void top_logits_launch(const void* logits, int type, int64_t ld, int64_t R, int V, int k, double temp,
                       void* top, int32_t* indices, float* lse, hipStream_t st) {
  const float c = (float)(1.4426950408889634 / temp);
  pick_type(type, [&](auto tv) {
    using T = decltype(tv);
    const T* z = reinterpret_cast<const T*>(logits);
    T* values = reinterpret_cast<T*>(top);
    if (V <= 64) {
      row_parts(R, [&](int64_t r, int64_t rows) {
        hipLaunchKernelGGL((top_small_kernel<T>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st,
                           z + r * ld, ld, rows, V, k, c, 1.0 / temp, values + r * k, indices + r * k,
                           lse + r);
      });
      return;
    }
    // Short rows, 134 MB by 64 / 256 threads: 33554 x 2000 bf16, k 5, 52 / 146 us, k 100 128 / 189; 67108
    // x 1000 bf16, k 192, 271 / 663. Long rows: few threads a row leave more rows to hide a row's steps
    // behind, until the first part (four chunks a thread) is too small a sample, or its candidates too
    // many for the threads: by 256 / 512 / 1024 threads 8388 x 32000 bf16, k 64, 124 / 139 / 212, k 512
    // 404 / 380 / 389; 2048 x 131072 bf16, k 64, 107 / 101 / 113, k 1000 1118 / 450 / 265.
    const int n = (V + kVE<T> - 1) / kVE<T>;
    const int threads = n <= 1024 ? 64
                        : few_rows(R, k <= 256 && 8 * k <= n && n <= 8192 ? 256
                                      : n <= 16384 && (k <= 384 || (k <= 640 && 8 * k <= n)) ? 512 : 1024,
                                   1024);
    pick_row(n, threads, [&](auto block, auto nc) {
      constexpr int BLOCK = decltype(block)::value, NC = decltype(nc)::value;
      // (a short row's list is short: its workgroups are small, and LDS would be what limits them)
      const int cap = NC ? std::min(kList, (3 * k + 255) / 64 * 64) : kList;
      row_parts(R, [&](int64_t r, int64_t rows) {
        hipLaunchKernelGGL((top_logits_kernel<T, BLOCK, NC>), dim3((uint32_t)rows), dim3(BLOCK), cap * 8, st,
                           z + r * ld, ld, V, k, c, 1.0 / temp, cap, values + r * k, indices + r * k, lse + r);
      });
    });
  });
}

void distill_launch(const DistillArgs& a, hipStream_t st) {
  const float c_t = (float)(1.4426950408889634 / a.temp);
  const size_t lds = (size_t)a.K * 16 + (size_t)((a.V + 31) / 32) * 4;
  pick_type(a.type, [&](auto tv) {
    using T = decltype(tv);
    // The rows at work at once are read again for the gradient: with few threads a row there are more of
    // them than the cache behind the L2s keeps (2048 x 131072 bf16 by 256 / 512 / 1024 threads 335 /
    // 309 / 279 us; 16384 x 16384 275 / 263 / 402). The loss alone reads them once (8388 x 32000 bf16
    // 110 / 124 / 192 us).
    const int n = (a.V + kVE<T> - 1) / kVE<T>;
    const int threads = n <= 1024 ? 64
                                  : few_rows(a.R, a.dz ? (n <= 8192 ? 512 : 1024)
                                                       : n <= 8192 ? 256 : 512, 2048);
    pick_row(n, threads, [&](auto block, auto nc) {
      constexpr int BLOCK = decltype(block)::value, NC = decltype(nc)::value;
      row_parts(a.R, [&](int64_t r, int64_t rows) {
        DistillArgs b = a;
        b.R = rows;
        b.z = reinterpret_cast<const T*>(a.z) + r * a.ld;
        b.values = reinterpret_cast<const char*>(a.values) + r * a.K * (a.value_type == LOGIT_F32 ? 4 : 2);
        b.indices = reinterpret_cast<const char*>(a.indices) + r * a.K * (a.index64 ? 8 : 4);
        if (a.lse) b.lse = a.lse + r;
        if (a.target) b.target = a.target + r;
        if (a.dz) b.dz = reinterpret_cast<T*>(a.dz) + r * a.V;
        if (a.row_loss) b.row_loss = a.row_loss + r;
        if (a.seed) b.seed = a.seed + r * a.seed_rows;
        if (a.dz)
          hipLaunchKernelGGL((distill_kernel<T, BLOCK, NC, true>), dim3((uint32_t)rows), dim3(BLOCK),
                             lds, st, b, c_t);
        else
          hipLaunchKernelGGL((distill_kernel<T, BLOCK, NC, false>), dim3((uint32_t)rows), dim3(BLOCK),
                             lds, st, b, c_t);
      });
    });
  });
}

void distill_sum_launch(const float* row_loss, int64_t R, double scale, float* loss,
                        hipStream_t st) {
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, row_loss, R, scale, loss);
}

}  // namespace pca
