// Gated linear layer: h = act(x Wg^T) * (x Wu^T) and its gradients.
//
// Three products run on one tiled kernel, each with fp32 sums on the matrix cores:
//   forward  both projections of a tile of hidden units in one pass over x, the activation and the
//            product in the epilogue (the projections never leave the registers, but for the fp32
//            copies that a backward pass wants);
//   dX       [dg | du] times [Wg; Wu], one sum over both halves;
//   dW       [dg | du]^T x.
// dg = dh u act'(g) and du = dh act(g) are formed from the fp32 projections and rounded once to the
// operands' type; in small products, which do not average the roundings out, in two parts.
#include "gated.h"
#include "mfma_util.h"

#include <algorithm>

namespace pca {
namespace {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// -------------------------------------------------------------------------- matrix fragments
// A K step takes 64 bytes of each row: 32 16-bit or 16 fp32 terms. A lane holds 16 bytes of it:
// row (lane & 15), piece (lane >> 4). mma() sums over the step into a 16 x 16 tile: lane l gets
// column (l & 15) of the second operand and rows 4 (l >> 4) .. + 3 of the first.
template <typename E>
struct Mat;

template <>
struct Mat<bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ void mma(const frag& a, const frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mat<f16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ void mma(const frag& a, const frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mat<float> {
  typedef f32x4 frag;
  // instruction e sums over element e of the four lane groups' pieces: terms e, 4 + e, 8 + e, 12 + e
  static __device__ __forceinline__ void mma(const frag& a, const frag& b, f32x4& c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  }
};

// fp32 products on the bf16 matrix instruction. A float is the exact sum of three bf16: itself rounded to
// nearest, what is left (at most 2^-8 of its power of two) rounded likewise, and the rest (2^-17). Of the
// nine products of two such sums the six largest are taken: what is left out is 2^-24 of a product at
// most, of either sign (parts that are cut off instead leave out 2^-21, always toward zero, for the same
// eleven instructions a pair; the large product below runs 3 % faster on them). Six instructions of 32
// terms take 96 cycles, the eight fp32 ones 256: gated_linear of 1021 x 512 -> 1365 forward and backward
// 127 -> 103 us; 2048 x 2048 -> 5504 forward at 188 TFLOP/s, the library's fp32 product at 140. (Below
// 2^-110 the last parts leave the type's range.) An infinity, and what rounds to one, has no such parts: a
// tile that meets one is computed again by the fp32 instruction.
constexpr float kSplitMost = 0x1.ffp127f;   // from here on
typedef float f32x8 __attribute__((ext_vector_type(8)));
struct Split {
  bf16x8 h, m, l;
};
__device__ __forceinline__ Split split3(const f32x8& v) {
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = v[2 * i], y = v[2 * i + 1];
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      const uint32_t p = pack2(x, y);
      w[part][i] = p;
      x -= __uint_as_float(p << 16);
      y -= __uint_as_float(p & 0xffff0000u);
    }
  }
  Split s;
  __builtin_memcpy(&s, w, sizeof(s));
  return s;
}
constexpr int kRow = 128;   // bytes of a row that a K tile takes: 64 16-bit or 32 fp32 terms
template <typename E>
constexpr int kBK = kRow / (int)sizeof(E);
template <typename E>
constexpr int kPiece = 16 / (int)sizeof(E);   // elements of 16 bytes

// LDS images of a K tile; both are written by 1-KiB DMA pieces, whose lanes choose the address they
// read so that the bytes land swizzled.
//   rows:  [tile row][128 bytes of its terms], 16-byte piece c of row r at c ^ (r & 7): the 16 rows
//          of a fragment read spread over all banks.
//   terms: operands whose terms are their rows. Blocks of [term][256 bytes of columns], read
//          transposed (16-bit: ds_read_b64_tr; fp32: four reads of 4 bytes).
template <typename E>
__device__ __forceinline__ typename Mat<E>::frag frag_rows(const char* lds, int r0, int s, int lane) {
  const int r = r0 + (lane & 15), c = 4 * s + (lane >> 4);
  return *reinterpret_cast<const typename Mat<E>::frag*>(lds + r * kRow + ((c ^ (r & 7)) << 4));
}

template <typename E>
__device__ __forceinline__ int swz_terms(int term) {
  if constexpr (sizeof(E) == 2) return tr_swz<256>(term);
  else return ((term >> 2) & 3) << 2;
}

template <typename E>
__device__ __forceinline__ typename Mat<E>::frag frag_terms(const char* lds, int c0, int s, int lane) {
  constexpr int kCols = 256 / (int)sizeof(E);        // columns of a block
  const char* blk = lds + (c0 / kCols) * (kBK<E> * 256);
  if constexpr (sizeof(E) == 2) {
    return __builtin_bit_cast(typename Mat<E>::frag, tr_frag<128>(blk, 32 * s, c0 % kCols, lane));
  } else {
    f32x4 v;
    const int col = c0 % kCols + (lane & 15);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 16 * s + 4 * (lane >> 4) + e;
      v[e] = *reinterpret_cast<const float*>(
          blk + k * 256 + (((col >> 2) ^ swz_terms<float>(k)) << 4) + ((col & 3) << 2));
    }
    return v;
  }
}

// The reciprocal instruction (1 step) in the place of the quotient, ten instructions: the epilogue
// takes a sigmoid of every hidden unit while the matrix cores stand still. The exponent is one rounded
// product with a rounded constant: for negative x the result is off by some (1.25 |x| + 2) 2^-24 relative.
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}
__device__ __forceinline__ float act_val(float g, int act) {
  if (act == ACT_SWISH) return g * sigmoid(g);
  if (act == ACT_SIGMOID) return sigmoid(g);
  return act == ACT_RELU && g < 0.f ? 0.f : g;   // (a NaN stays one)
}
// act(g) and its slope
__device__ __forceinline__ void act_both(float g, int act, float& v, float& slope) {
  if (act == ACT_SWISH || act == ACT_SIGMOID) {
    const float s = sigmoid(g);
    v = act == ACT_SWISH ? g * s : s;
    slope = act == ACT_SWISH ? fmaf(v, 1.f - s, s) : s * (1.f - s);
  } else {
    v = act == ACT_RELU && g < 0.f ? 0.f : g;
    slope = act == ACT_RELU && g <= 0.f ? 0.f : 1.f;
  }
}

// 4 consecutive outputs of a row at column n (N columns in all), at any alignment
template <typename O>
__device__ __forceinline__ void store4(O* row, int n, int N, const f32x4& v, bool whole) {
  O h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = static_cast<O>(v[i]);
  if (whole || n + 4 <= N) {
    __builtin_memcpy(row + n, h, sizeof(h));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) row[n + i] = h[i];
  }
}

// ---------------------------------------------------------------------------- tiled product
// Bound by the matrix instruction (fp32: and by the splitting before it). The wider the tile the fewer
// LDS reads a product takes: a wave of eight has 128 x 64 sums, half of its registers. Forward of
// 8192 x 4096 -> 10752 bf16 1044 us, 1.38 PFLOP/s (a square product of 8192 by the library 1.42); of
// 4096 x 2048 -> 5504 175 us, 1.06 PFLOP/s: 2.7 rounds of tiles, each with 12 us at its ends.
template <typename E, typename O, int FORM, int BM, int BN, int WM, int WN>
// (two waves a SIMD is what the LDS leaves room for: told so, the compiler keeps the sums out of AGPRs)
__global__ __launch_bounds__(WM* WN * 64)
__attribute__((amdgpu_waves_per_eu(2, 2))) void gated_kernel(GatedArgs a, int mt, int nt) {
  constexpr int NW = WM * WN, NT = NW * 64;
  constexpr int TM = BM / WM, TN = BN / WN;          // a wave's tile
  constexpr int MF = TM / 16, NF = TN / 16;
  constexpr bool kFwd = FORM == GATED_FWD;
  constexpr bool kTermsQ = FORM == GATED_DW, kTermsP = FORM != GATED_FWD;
  constexpr int BK = kBK<E>, ES = sizeof(E), PC = kPiece<E>;
  // bytes of a K tile (by terms: in whole blocks of columns)
  constexpr int QB = (kTermsQ ? (BM + 127) / 128 * 128 : BM) * kRow, PB = BN * kRow;
  constexpr int QP = QB / 1024 / NW, PP = PB / 1024 / NW;   // DMA pieces of a wave
  static_assert(QB % (1024 * NW) == 0 && PB % (1024 * NW) == 0, "whole pieces a wave");
  __shared__ __attribute__((aligned(1024))) char lds[2][QB + PB];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // consecutive workgroups of an XCD walk M first within a group of 8 N tiles
  const int wg = xcd_remap(blockIdx.x, gridDim.x);
  constexpr int G = 8;
  const int per = G * mt, grp = wg / per, first = grp * G, gn = min(G, nt - first);
  const int ni = first + (wg % per) % gn, mi0 = (wg % per) / gn;
  int half = 0, mi = mi0;
  if constexpr (FORM == GATED_DW) {
    half = mi0 >= mt / 2;
    mi = half ? mi0 - mt / 2 : mi0;
  }
  constexpr int NH = kFwd ? BN / 2 : BN;             // output columns of a tile
  const int m0 = mi * BM, n0 = ni * NH;

  const int per_seg = (a.K + BK - 1) / BK;
  const int nk = (FORM == GATED_DX ? 2 * a.parts : FORM == GATED_DW ? a.parts : 1) * per_seg;
  const int split = blockIdx.y;
  const int t0 = (int)((int64_t)nk * split / gridDim.y);
  const int t1 = (int)((int64_t)nk * (split + 1) / gridDim.y);

  // ---- where each lane's pieces come from, relative to a base that moves with the K tile
  uint32_t qoff[QP], poff[PP];
  int qk[QP], pk[PP];                                // first term of the piece in its K tile
#pragma unroll
  for (int i = 0; i < QP; ++i) {
    const int p = i * NW + wave;
    if constexpr (kTermsQ) {
      const int term = (p * 4 + (lane >> 4)) % BK, blk = p * 4 / BK;
      const int c = blk * (256 / ES) + (((lane & 15) ^ swz_terms<E>(term)) * PC);
      qk[i] = term;
      qoff[i] = c < BM && m0 + c < a.mcols ? (uint32_t)(term * a.ldq + c) * ES : kOOB;
    } else {
      const int r = p * 8 + (lane >> 3), c = ((lane & 7) ^ (r & 7)) * PC;
      qk[i] = c;
      qoff[i] = m0 + r < a.M ? (uint32_t)(r * a.ldq + c) * ES : kOOB;
    }
  }
  bool up[PP];                                       // (wave-uniform: a piece is 8 rows of one half)
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int p = i * NW + wave;
    up[i] = false;
    if constexpr (kTermsP) {
      const int term = (p * 4 + (lane >> 4)) % BK, blk = p * 4 / BK;
      const int c = blk * (256 / ES) + (((lane & 15) ^ swz_terms<E>(term)) * PC);
      pk[i] = term;
      poff[i] = n0 + c < a.ncols ? (uint32_t)(term * a.ldp + c) * ES : kOOB;
    } else {
      // a wave's TN rows: TN/2 of the gate, then the same TN/2 hidden units of the other
      const int r = p * 8 + (lane >> 3), c = ((lane & 7) ^ (r & 7)) * PC;
      const int rw = (p * 8) / TN, rq = r % TN;
      up[i] = (p * 8) % TN >= TN / 2;
      const int f = rw * (TN / 2) + rq % (TN / 2);
      pk[i] = c;
      poff[i] = n0 + f < a.N ? (uint32_t)(f * a.ldp + c) * ES : kOOB;
    }
  }
  const char* qb = reinterpret_cast<const char*>(a.q);
  if constexpr (kTermsQ) qb += ((int64_t)half * a.qseg + m0) * ES;
  else qb += (int64_t)m0 * a.ldq * ES;

  // (held in registers: picked from the arguments in the loop, the pointer would be loaded, and waited
  // for with all LDS reads, at every K tile)
  const char *p0 = reinterpret_cast<const char*>(a.p0), *p1 = reinterpret_cast<const char*>(a.p1);
  asm("" : "+s"(p0), "+s"(p1));
  const int qseg = (int)a.qseg;
  const bool two = a.parts == 2;
  // K tile t: its first term and where it lies
  struct Src {
    int k0;
    const char *q, *p, *u;
  };
  auto source = [&](int t) {
    int seg = 0;
    if constexpr (FORM == GATED_DX) {
      seg = t >= per_seg;
      if (two) seg += (t >= 2 * per_seg) + (t >= 3 * per_seg);
    }
    if constexpr (FORM == GATED_DW) seg = t >= per_seg;
    Src s;
    s.k0 = (t - seg * per_seg) * BK;
    s.q = qb + (kTermsQ ? (int64_t)s.k0 * a.ldq + 2 * seg * qseg : (int64_t)(s.k0 + seg * qseg)) * ES;
    const int64_t at = (kFwd ? (int64_t)n0 * a.ldp + s.k0 : (int64_t)s.k0 * a.ldp + n0) * ES;
    s.p = (FORM == GATED_DX && (seg & 1) ? p1 : p0) + at;
    s.u = p1 + at;   // (forward: the other weight)
    return s;
  };
  constexpr int kPieces = QP + PP;
  auto issue = [&](const Src& s, int buf, int i) {   // the wave's piece i of a tile
    if (i < QP) {
      dma16(make_rsrc(s.q, 0x7fffffffu), &lds[buf][(i * NW + wave) * 1024],
            s.k0 + qk[i] < a.K ? qoff[i] : kOOB);
    } else {
      const int j = i - QP;
      dma16(make_rsrc(kFwd && up[j] ? s.u : s.p, 0x7fffffffu), &lds[buf][QB + (j * NW + wave) * 1024],
            s.k0 + pk[j] < a.K ? poff[j] : kOOB);
    }
  };

  f32x4 acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  // A K tile is two steps of 64 bytes of terms (fp32: one of 128). While a step's products run, the
  // next step's fragments are read in the place of those that are done; between the last step of a
  // tile and the first of the next stands the tile's one barrier: all waves have read the old buffer,
  // which the tile after next then fills, and all pieces of the next have landed.
  constexpr bool kF32 = ES == 4;
  typedef std::conditional_t<kF32, f32x8, typename Mat<E>::frag> Frag;
  Frag q[MF], p[NF];
  auto fragment = [&](auto terms, const char* from, int at, int s) -> Frag {
    auto one = [&](int s) {
      return decltype(terms)::value ? frag_terms<E>(from, at, s, lane) : frag_rows<E>(from, at, s, lane);
    };
    if constexpr (kF32) return __builtin_shufflevector(one(0), one(1), 0, 1, 2, 3, 4, 5, 6, 7);
    else return one(s);
  };
  auto read_q = [&](int buf, int s, int j) {
    return fragment(std::integral_constant<bool, kTermsQ>(), lds[buf], wm * TM + 16 * j, s);
  };
  auto read_p = [&](int buf, int s, int i) {
    return fragment(std::integral_constant<bool, kTermsP>(), lds[buf] + QB, wn * TN + 16 * i, s);
  };
  // fp32: the largest magnitude that the wave has read (a NaN is passed over)
  float most = 0.f;
  auto look = [&](const Frag& v) {
    if constexpr (kF32) {
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(most) : "v"(most), "v"(v[e]), "v"(v[e + 1]));
    }
  };
  // products of q[j]; `between(j)` follows those of each
  auto products = [&](auto between) {
    if constexpr (!kF32) {
#pragma unroll
      for (int j = 0; j < MF; ++j) {
#pragma unroll
        for (int i = 0; i < NF; ++i) Mat<E>::mma(p[i], q[j], acc[i][j]);
        between(j);
      }
    } else {
      Split ps[NF];
#pragma unroll
      for (int i = 0; i < NF; ++i) look(p[i]), ps[i] = split3(p[i]);
      typedef Mat<bf16> B;
      look(q[0]);
      Split qs = split3(q[0]);
#pragma unroll
      for (int j = 0; j < MF; ++j) {
        Split then = qs;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NF; ++i) B::mma(ps[i].l, qs.h, acc[i][j]);
#pragma unroll
        for (int i = 0; i < NF; ++i) B::mma(ps[i].h, qs.l, acc[i][j]);
#pragma unroll
        for (int i = 0; i < NF; ++i) B::mma(ps[i].m, qs.m, acc[i][j]);
#pragma unroll
        for (int i = 0; i < NF; ++i) B::mma(ps[i].m, qs.h, acc[i][j]);
#pragma unroll
        for (int i = 0; i < NF; ++i) B::mma(ps[i].h, qs.m, acc[i][j]);
#pragma unroll
        for (int i = 0; i < NF; ++i) B::mma(ps[i].h, qs.h, acc[i][j]);
        if (j + 1 < MF) {   // the next fragment's parts between them
          look(q[j + 1]);
          then = split3(q[j + 1]);
        }
#pragma unroll
        for (int k = 0; k < 6 * NF; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
        }
        qs = then;
        between(j);
      }
    }
  };
  // The step's products on q, p, the reads of the next behind the first of them (by the step's end
  // they have long arrived), and, with `src`, the pieces of a later tile between them: issued all at
  // once they would hold the products up until the last wave's have been taken.
  auto step = [&](auto fill, int buf, int s, const Src& src, int to) {
    Frag nq[MF], np[NF];
    constexpr int kG = MF >= 4 ? MF / 2 : 1, kFrags = (NF + MF + kG - 1) / kG;
    constexpr int kEach = (kPieces + MF - 1) / MF;
    products([&](int j) {
      if constexpr (kF32) {   // (each in the registers of one that is done with)
        nq[j] = read_q(buf, s, j);
#pragma unroll
        for (int i = j; i < NF; i += MF) np[i] = read_p(buf, s, i);
      } else {
#pragma unroll
        for (int r = j * kFrags; r < (j + 1) * kFrags; ++r) {
          if (r < NF) np[r] = read_p(buf, s, r);
          else if (r < NF + MF) nq[r - NF] = read_q(buf, s, r - NF);
        }
      }
      if constexpr (decltype(fill)::value) {
#pragma unroll
        for (int i = j * kEach; i < (j + 1) * kEach && i < kPieces; ++i) issue(src, to, i);
      }
      if constexpr (!kF32) __builtin_amdgcn_sched_barrier(0);
    });
#pragma unroll
    for (int i = 0; i < NF; ++i) p[i] = np[i];
#pragma unroll
    for (int j = 0; j < MF; ++j) q[j] = nq[j];
  };
  constexpr std::integral_constant<bool, true> kFill;
  constexpr std::integral_constant<bool, false> kNoFill;
  if (t0 < t1) {
    const Src first = source(t0);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) issue(first, 0, i);
    if (t0 + 1 < t1) {
      const Src second = source(t0 + 1);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) issue(second, 1, i);
      wait_vmcnt<kPieces>();
    } else {
      wait_vmcnt<0>();
    }
    raw_barrier();
#pragma unroll
    for (int i = 0; i < NF; ++i) p[i] = read_p(0, 0, i);
#pragma unroll
    for (int j = 0; j < MF; ++j) q[j] = read_q(0, 0, j);
    // lgkmcnt(0): with a scalar load pending at the loop's entry every wait in it would be for all
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
  int t = t0;
  auto turn = [&]() {   // between two tiles
    __builtin_amdgcn_s_waitcnt(0x70);   // vmcnt(0) lgkmcnt(0): as the compiler knows it
    raw_barrier();
  };
  for (; t + 2 < t1; ++t) {
    const int buf = (t - t0) & 1;
    const Src src = source(t + 2);
    if constexpr (!kF32) step(kNoFill, buf, 1, src, 0);
    turn();
    step(kFill, buf ^ 1, 0, src, buf);
  }
  if (t + 1 < t1) {
    const int buf = (t - t0) & 1;
    if constexpr (!kF32) step(kNoFill, buf, 1, Src(), 0);
    turn();
    step(kNoFill, buf ^ 1, 0, Src(), 0);
    ++t;
  }
  if (t < t1) {
    if constexpr (!kF32) step(kNoFill, (t - t0) & 1, 1, Src(), 0);
    products([](int) {});
  }
  if constexpr (kF32) {
    int* met = reinterpret_cast<int*>(&lds[0][0]);
    __syncthreads();
    if (threadIdx.x == 0) *met = 0;
    __syncthreads();
    if (most >= kSplitMost) *met = 1;
    __syncthreads();
    const bool again = *met != 0;
    __syncthreads();
    if (again) {
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
      for (int t = t0; t < t1; ++t) {
        const Src src = source(t);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) issue(src, 0, i);
        turn();
#pragma unroll
        for (int j = 0; j < MF; ++j) {
          const Frag x = read_q(0, 0, j);
#pragma unroll
          for (int i = 0; i < NF; ++i) {
            const Frag y = read_p(0, 0, i);
            Mat<float>::mma(__builtin_shufflevector(y, y, 0, 1, 2, 3), __builtin_shufflevector(x, x, 0, 1, 2, 3), acc[i][j]);
            Mat<float>::mma(__builtin_shufflevector(y, y, 4, 5, 6, 7), __builtin_shufflevector(x, x, 4, 5, 6, 7), acc[i][j]);
          }
        }
        turn();
      }
    }
  }

  // ---- epilogue: lane holds columns 4 (lane >> 4) .. + 3 of row (lane & 15) of each 16 x 16 tile
  const int cl = 4 * (lane >> 4);
  const int act = a.act;
  auto put = [&](auto whole) {   // whole: all of the tile's rows and columns are there
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int j = 0; j < MF; ++j) {
      const int m = m0 + wm * TM + 16 * j + (lane & 15);
      if (!W && m >= a.M) continue;
      const int64_t at = (int64_t)m * a.N;
      if constexpr (kFwd) {
        O* out = reinterpret_cast<O*>(a.out0) + at;
        float* part = a.part ? a.part + ((int64_t)split * a.M + m) * 2 * a.N : nullptr;
#pragma unroll
        for (int i = 0; i < NF / 2; ++i) {
          const int n = n0 + wn * (TN / 2) + 16 * i + cl;
          const f32x4 g = acc[i][j], u = acc[i + NF / 2][j];
          if (part) {
            store4(part, n, a.N, g, W);
            store4(part + a.N, n, a.N, u, W);
            continue;
          }
          if (a.save_g) {
            store4(a.save_g + at, n, a.N, g, W);
            store4(a.save_u + at, n, a.N, u, W);
          }
          f32x4 h;
          if (act == ACT_SWISH) {
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = g[e] * sigmoid(g[e]) * u[e];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = act_val(g[e], act) * u[e];
          }
          store4(out, n, a.N, h, W);
        }
      } else {
        const int64_t rows = (FORM == GATED_DW ? 2 : 1) * (int64_t)a.M;
        float* part = a.part ? a.part + (split * rows + half * (int64_t)a.M + m) * a.N : nullptr;
        O* out = reinterpret_cast<O*>(half ? a.out1 : a.out0) + at;
#pragma unroll
        for (int i = 0; i < NF; ++i) {
          const int n = n0 + wn * TN + 16 * i + cl;
          if (part) store4(part, n, a.N, acc[i][j], W);
          else store4(out, n, a.N, acc[i][j], W);
        }
      }
    }
  };
  if (m0 + BM <= a.M && n0 + NH <= a.N) put(std::integral_constant<bool, true>());
  else put(std::integral_constant<bool, false>());
}

// ------------------------------------------------------------------------ few rows (forward)
// Up to 64 rows: the weights are read once, straight into the fragments' registers, and that read is
// all the time there is. A workgroup has 16 hidden units of both weights; its waves take every NW-th
// 64 bytes of the width, and their sums are joined in LDS, in order. The rows come from the caches
// (every workgroup reads all of them). One row, 4096 -> 10752 bf16 (176 MB): 37 us, 4.7 TB/s.
template <typename E, int MT, int NW>
__global__ __launch_bounds__(NW * 64) 
__attribute__((amdgpu_waves_per_eu(MT < 4 ? 4 : 2))) void gated_few_kernel(GatedArgs a) {
  constexpr int ES = sizeof(E), UB = 1, U = MT == 1 ? 4 : 2;   // 16-unit blocks; steps in flight
  __shared__ f32x4 sums[NW][2 * UB * MT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16 * UB;
  const int64_t at = (int64_t)n0 * a.ldp * ES;
  const auto rg = make_rsrc(reinterpret_cast<const char*>(a.p0) + at, 0x7fffffffu);
  const auto ru = make_rsrc(reinterpret_cast<const char*>(a.p1) + at, 0x7fffffffu);
  const auto rx = make_rsrc(a.q, 0x7fffffffu);
  const int r = lane & 15, c = (lane >> 4) * 16;
  uint32_t wo[UB], xo[MT];
#pragma unroll
  for (int i = 0; i < UB; ++i)
    wo[i] = n0 + 16 * i + r < a.N ? (uint32_t)((16 * i + r) * a.ldp) * ES + c : kOOB;
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xo[i] = 16 * i + r < a.M ? (uint32_t)((16 * i + r) * a.ldq) * ES + c : kOOB;
  const int bytes = a.K * ES, steps = (bytes + 63) / 64;

  typedef int i32x4 __attribute__((ext_vector_type(4)));
  typedef typename Mat<E>::frag frag;
  struct Step {
    i32x4 g[UB], u[UB], x[MT];
  };
  auto load = [&](Step& s, int i) {   // past the width: zeros
    const int k = i * 64;
    const bool in = k + c < bytes;
#pragma unroll
    for (int j = 0; j < UB; ++j) {
      s.g[j] = __builtin_amdgcn_raw_buffer_load_b128(rg, in ? wo[j] : kOOB, k, 0);
      s.u[j] = __builtin_amdgcn_raw_buffer_load_b128(ru, in ? wo[j] : kOOB, k, 0);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
      s.x[j] = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? xo[j] : kOOB, k, 0);
  };
  f32x4 acc[2 * UB][MT];
#pragma unroll
  for (int i = 0; i < 2 * UB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
  Step now[U], next[U];
#pragma unroll
  for (int j = 0; j < U; ++j) load(now[j], wave + j * NW);
  for (int i = wave; i < steps; i += U * NW) {
#pragma unroll
    for (int j = 0; j < U; ++j) load(next[j], i + (U + j) * NW);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int b = 0; b < UB; ++b) {
          const frag x = __builtin_bit_cast(frag, now[j].x[m]);
          Mat<E>::mma(__builtin_bit_cast(frag, now[j].g[b]), x, acc[b][m]);
          Mat<E>::mma(__builtin_bit_cast(frag, now[j].u[b]), x, acc[UB + b][m]);
        }
#pragma unroll
    for (int j = 0; j < U; ++j) now[j] = next[j];
  }
#pragma unroll
  for (int i = 0; i < 2 * UB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[wave][i * MT + j][lane] = acc[i][j];
  __syncthreads();
  for (int b = wave; b < UB * MT; b += NW) {
    const int i = b / MT, j = b % MT;
    f32x4 g = sums[0][i * MT + j][lane], u = sums[0][(UB + i) * MT + j][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      g += sums[w][i * MT + j][lane];
      u += sums[w][(UB + i) * MT + j][lane];
    }
    const int m = 16 * j + (lane & 15), n = n0 + 16 * i + 4 * (lane >> 4);
    if (m >= a.M) continue;
    const int64_t to = (int64_t)m * a.N;
    if (a.save_g) {
      store4(a.save_g + to, n, a.N, g, false);
      store4(a.save_u + to, n, a.N, u, false);
    }
    f32x4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = act_val(g[e], a.act) * u[e];
    store4(reinterpret_cast<E*>(a.out0) + to, n, a.N, h, false);
  }
}

// Sums of the K splits, in order, and the epilogue that follows them. Bound by the read of the sums:
// two splits of 4096 x 2048 16 us.
template <typename O, int FORM>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedArgs a, int64_t n) {
  const int64_t total = FORM == GATED_FWD || FORM == GATED_DW ? 2 * n : n;   // floats of a split
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    if constexpr (FORM == GATED_FWD) {
      const int64_t m = i / a.N, f = i % a.N;
      float g = 0.f, u = 0.f;
      for (int s = 0; s < a.splits; ++s) {
        const float* row = a.part + s * total + m * 2 * a.N;
        g += row[f];
        u += row[a.N + f];
      }
      reinterpret_cast<O*>(a.out0)[i] = static_cast<O>(act_val(g, a.act) * u);
      if (a.save_g) {
        a.save_g[i] = g;
        a.save_u[i] = u;
      }
    } else {
#pragma unroll
      for (int h = 0; h < (FORM == GATED_DW ? 2 : 1); ++h) {
        float v = 0.f;
        for (int s = 0; s < a.splits; ++s) v += a.part[s * total + h * n + i];
        reinterpret_cast<O*>(h ? a.out1 : a.out0)[i] = static_cast<O>(v);
      }
    }
  }
}

// ------------------------------------------------------------------------ elementwise passes
// dg and du. Bound by the bytes: 4096 x 5504 bf16 (316 MB) 66 us, the rate of a large copy.
//
// Two parts, a number and what it was rounded by, are as good as their sum in products with finite
// numbers; with an infinity the second gives one of the other sign, or NaN. An infinity in a row or a
// weight makes every projection that its product with dg or du belongs to infinite or NaN, so there, and
// where dg or du is one itself, both parts are half of the rounded number.
template <typename E>
__global__ __launch_bounds__(256) void gated_dact_kernel(const float* __restrict__ g,
                                                         const float* __restrict__ u,
                                                         const E* __restrict__ dh, int64_t lddh,
                                                         int64_t M, int F, int Fp, int act,
                                                         int parts, E* __restrict__ out) {
  constexpr int PC = kPiece<E>;
  const int pieces = Fp / PC;
  for (int64_t w = blockIdx.x * 256ll + threadIdx.x; w < M * pieces; w += (int64_t)gridDim.x * 256) {
    const int64_t m = w / pieces;
    const int f0 = (int)(w % pieces) * PC;
    E dg[PC], du[PC];
    bool wild[PC];
    float gv[PC], uv[PC];
    E d[PC];
    if (f0 + PC <= F) {
      __builtin_memcpy(gv, g + m * F + f0, sizeof(gv));
      __builtin_memcpy(uv, u + m * F + f0, sizeof(uv));
      __builtin_memcpy(d, dh + m * lddh + f0, sizeof(d));
    } else {
#pragma unroll
      for (int i = 0; i < PC; ++i) {
        const bool in = f0 + i < F;
        gv[i] = in ? g[m * F + f0 + i] : 0.f;
        uv[i] = in ? u[m * F + f0 + i] : 0.f;
        d[i] = in ? dh[m * lddh + f0 + i] : static_cast<E>(0.f);
      }
    }
#pragma unroll
    for (int i = 0; i < PC; ++i) {
      const float df = static_cast<float>(d[i]);
      float v, slope;
      act_both(gv[i], act, v, slope);
      wild[i] = !isfinite(gv[i]) || !isfinite(uv[i]);
      gv[i] = df * uv[i] * slope;
      uv[i] = df * v;
      dg[i] = static_cast<E>(gv[i]);
      du[i] = static_cast<E>(uv[i]);
    }
    E* row = out + m * 2 * parts * Fp + f0;
    if (parts == 2) {
      E dg2[PC], du2[PC];
      auto rest = [&](E& first, float v, bool far) {
        const float r = static_cast<float>(first);
        if (!far && !isinf(r)) return static_cast<E>(v - r);
        const E half = static_cast<E>(r * 0.5f);
        if (static_cast<float>(half) != 0.f) first = half;   // (the smallest number is counted twice)
        return first;
      };
#pragma unroll
      for (int i = 0; i < PC; ++i) {
        dg2[i] = rest(dg[i], gv[i], wild[i]);
        du2[i] = rest(du[i], uv[i], wild[i]);
      }
      __builtin_memcpy(row + 2 * Fp, dg2, 16);
      __builtin_memcpy(row + 3 * Fp, du2, 16);
    }
    __builtin_memcpy(row, dg, 16);
    __builtin_memcpy(row + Fp, du, 16);
  }
}

template <typename S, typename E>
__global__ __launch_bounds__(256) void gated_operand_kernel(const S* __restrict__ src, int64_t ld,
                                                            int64_t R, int n, E* __restrict__ dst,
                                                            int np) {
  constexpr int PC = kPiece<E>;
  const int pieces = np / PC;
  for (int64_t w = blockIdx.x * 256ll + threadIdx.x; w < R * pieces; w += (int64_t)gridDim.x * 256) {
    const int64_t r = w / pieces;
    const int c = (int)(w % pieces) * PC;
    E v[PC];
    if (c + PC <= n) {
      S s[PC];
      __builtin_memcpy(s, src + r * ld + c, sizeof(s));
#pragma unroll
      for (int i = 0; i < PC; ++i) v[i] = static_cast<E>(static_cast<float>(s[i]));
    } else {
#pragma unroll
      for (int i = 0; i < PC; ++i)
        v[i] = static_cast<E>(c + i < n ? static_cast<float>(src[r * ld + c + i]) : 0.f);
    }
    __builtin_memcpy(dst + r * np + c, v, 16);
  }
}

template <typename F>
void pick_type(int type, F&& fn) {
  if (type == GATED_F32) fn(float());
  else if (type == GATED_BF16) fn(bf16());
  else fn(f16());
}

uint32_t grid_for(int64_t n) { return (uint32_t)std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, 4096)); }

constexpr int kCUs = 256;

// Rows up to which gated_few_kernel is taken: it reads all rows once a 16 hidden units, which by some
// 30 rows is as much as the weights. In us, by it and by tiles: 4096 -> 10752 bf16 8 / 16 / 32 rows 40 /
// 44 / 54 and 38, 2048 -> 5504 17 / 32 / 48 rows 15 / 17 / 21 and 19, 1024 -> 4096 6 / 7 / 8 and 16.
bool few_rows(int type, int M, int N, int K) {
  const double weights = 2.0 * N * K * (type == GATED_F32 ? 4 : 2);
  return M <= 64 && weights * M <= 1.6e9;
}

// Tiles and splits of the sum by a model of the time in us, from measured times: a K tile of 64
// (fp32: 32) terms takes a 256 x 256 tile 1.25, a 192 x 256 tile 1.06 in the forward and 1.12 in the
// gradients, a 128 x 128 tile alone on its compute unit 0.65 (fp32 1.5) and two that share one 1.11
// (2.5); a tile's start and end take 12 and 8; the partial sums of splits are written and read at
// 4.5 TB/s by one more launch. (4096 x 2048, 5504 hidden units, bf16: dx in 128 large tiles 201 us as
// small ones, 162 + 16 in two splits; dW in 352 tiles of 256 rows, 1.4 rounds of the 256 compute
// units, 197, in 464 of 192 rows, 1.8 rounds, 178. Forward of 4096 x 1536 -> 4224 fp16 in 528 tiles of
// 256 rows 117, in 726 of 192 104.)
struct Plan {
  int bm, mt, nt, splits;
};
Plan plan(int form, int type, int M, int N, int K, int parts) {
  const int halves = form == GATED_DW ? 2 : 1, nh = form == GATED_FWD ? 2 : 1;
  const bool f32 = type == GATED_F32;
  const int nk = (form == GATED_DX ? 2 : 1) * parts * cdiv(K, kRow / (f32 ? 4 : 2));
  Plan best{};
  double least = 0;
  for (int bm = 128; bm <= (f32 ? 128 : 256); bm += 64) {
    const bool big = bm > 128;
    const int mt = halves * cdiv(M, bm), nt = cdiv(N * nh, big ? 256 : 128);
    for (int s = 1; s <= 16 && (s == 1 || nk / s >= 4); ++s) {
      const int64_t n = (int64_t)mt * nt * s;
      const double each = bm == 256 ? 1.25 : big ? (form == GATED_FWD ? 1.06 : 1.12) : n <= kCUs ? (f32 ? 1.5 : 0.65) : f32 ? 2.5 : 1.11;
      const double rounds = (double)cdiv64(n, big || n <= kCUs ? kCUs : 2 * kCUs);
      double us = rounds * (cdiv(nk, s) * each + (big ? 12 : 8));
      if (s > 1) us += 5 + (double)M * N * halves * nh * 4 * (2 * s) / 4.5e6;
      if (least == 0 || us < least) {
        least = us;
        best = {bm, mt, nt, s};
      }
    }
  }
  return best;
}

}  // namespace

int gated_parts(int type, int64_t M, int64_t C, int64_t F) {
  // One part's rounding is that of the result again, sqrt(2) of it together where many terms average
  // it out; up to 1.7 was seen in gradients of a few rows, and none above 1.5 in two parts. Twice the
  // terms are 8 M C F more operations: 256 x 512 -> 1536 backward 33 -> 34.5 us, at the bound 3 us of
  // some 40.
  return type != GATED_F32 && M * C * F <= 250000000 ? 2 : 1;
}

int gated_splits(int form, int type, int M, int N, int K, int parts) {
  if (form == GATED_FWD && few_rows(type, M, N, K)) return 1;
  return plan(form, type, M, N, K, parts).splits;
}

int64_t gated_part_floats(int form, int M, int N) {
  return (int64_t)M * N * (form == GATED_DX ? 1 : 2);
}

void gated_launch(int form, int type, bool out_f32, const GatedArgs& a, hipStream_t st) {
  if (form == GATED_FWD && few_rows(type, a.M, a.N, a.K)) {
    pick_type(type, [&](auto ev) {
      using E = decltype(ev);
      const dim3 grid((uint32_t)cdiv(a.N, 16));
      if (a.M <= 16) hipLaunchKernelGGL((gated_few_kernel<E, 1, 4>), grid, dim3(256), 0, st, a);
      else if (a.M <= 32) hipLaunchKernelGGL((gated_few_kernel<E, 2, 4>), grid, dim3(256), 0, st, a);
      else if (a.M <= 48) hipLaunchKernelGGL((gated_few_kernel<E, 3, 4>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((gated_few_kernel<E, 4, 4>), grid, dim3(256), 0, st, a);
    });
    return;
  }
  const Plan p = plan(form, type, a.M, a.N, a.K, std::max(a.parts, 1));
  const dim3 grid((uint32_t)(p.mt * p.nt), (uint32_t)a.splits);
  const int64_t n = (int64_t)a.M * a.N;
  auto go = [&](auto ev, auto ov, auto fv) {
    using E = decltype(ev);
    using O = decltype(ov);
    constexpr int FORM = decltype(fv)::value;
    if (p.bm > 128) {
      if constexpr (sizeof(E) == 2) {   // (fp32: its fragments take the registers of 128 x 128)
        if (p.bm == 256)
          hipLaunchKernelGGL((gated_kernel<E, O, FORM, 256, 256, 2, 4>), grid, dim3(512), 0, st, a, p.mt, p.nt);
        else
          hipLaunchKernelGGL((gated_kernel<E, O, FORM, 192, 256, 2, 4>), grid, dim3(512), 0, st, a, p.mt, p.nt);
      }
    } else
      hipLaunchKernelGGL((gated_kernel<E, O, FORM, 128, 128, 2, 2>), grid, dim3(256), 0, st, a, p.mt, p.nt);
    if (a.part)
      hipLaunchKernelGGL((gated_join_kernel<O, FORM>), dim3(grid_for(n)), dim3(256), 0, st, a, n);
  };
  pick_type(type, [&](auto ev) {
    using E = decltype(ev);
    using std::integral_constant;
    if (form == GATED_FWD) go(ev, ev, integral_constant<int, GATED_FWD>());
    else if (form == GATED_DX) go(ev, ev, integral_constant<int, GATED_DX>());
    else if (out_f32) go(ev, float(), integral_constant<int, GATED_DW>());
    else go(ev, ev, integral_constant<int, GATED_DW>());
  });
}

void gated_dact_launch(int type, const float* g, const float* u, const void* dh, int64_t lddh,
                       int64_t M, int F, int Fp, int act, int parts, void* dgdu, hipStream_t st) {
  pick_type(type, [&](auto ev) {
    using E = decltype(ev);
    hipLaunchKernelGGL((gated_dact_kernel<E>), dim3(grid_for(M * (Fp / kPiece<E>))), dim3(256), 0,
                       st, g, u, reinterpret_cast<const E*>(dh), lddh, M, F, Fp, act, parts,
                       reinterpret_cast<E*>(dgdu));
  });
}

void gated_operand_launch(const void* src, int src_type, int64_t ld, int64_t R, int n, void* dst,
                          int dst_type, int np, hipStream_t st) {
  pick_type(src_type, [&](auto sv) {
    pick_type(dst_type, [&](auto ev) {
      using S = decltype(sv);
      using E = decltype(ev);
      hipLaunchKernelGGL((gated_operand_kernel<S, E>), dim3(grid_for(R * (np / kPiece<E>))),
                         dim3(256), 0, st, reinterpret_cast<const S*>(src), ld, R, n,
                         reinterpret_cast<E*>(dst), np);
    });
  });
}

}  // namespace pca
