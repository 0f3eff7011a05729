// Host interface of gated.hip.
#pragma once
#include "common.h"

namespace pca {

enum GatedType : int { GATED_F32 = 0, GATED_BF16 = 1, GATED_F16 = 2 };

// One product of the layer. All operands have rows of whole 16-byte pieces at 16-byte addresses.
//   FWD  out[m][f]  = act(g) u with g, u = sum_c q[m][c] p0/p1[f][c]          (save: g, u in fp32)
//   DX   out[m][c]  = sum_f q[m][f] p0[f][c] + sum_f q[m][qseg + f] p1[f][c]
//   DW   out0/1[f][c] = sum_m q[m][f / qseg + f] p0[m][c]
// parts 2: q has further columns [2 qseg, 4 qseg), what the first were rounded by, summed likewise.
struct GatedArgs {
  const void* q;         // M side
  const void* p0;        // N side
  const void* p1;
  int64_t ldq, ldp, qseg;
  int M, N, K;           // output rows, output columns, terms of a sum
  int ncols;             // columns p may be read at (N rounded up to a whole piece)
  int mcols;             // DW: columns q may be read at
  void* out0;
  void* out1;
  float* save_g;         // FWD: [M][N] fp32 or null
  float* save_u;
  float* part;           // [splits][...] fp32 partial sums, or null
  int splits;
  int act;
  int parts;             // DX, DW: 1 or 2
};
enum GatedForm : int { GATED_FWD = 0, GATED_DX = 1, GATED_DW = 2 };

// splits the launch wants (1: no workspace); its workspace holds splits * gated_part_floats
int gated_splits(int form, int type, int M, int N, int K, int parts);
// parts that the gradients of the projections are kept in
int gated_parts(int type, int64_t M, int64_t C, int64_t F);
int64_t gated_part_floats(int form, int M, int N);
void gated_launch(int form, int type, bool out_f32, const GatedArgs& a, hipStream_t st);

// dgdu[m][0..F) = dh u act'(g), dgdu[m][Fp..Fp+F) = dh act(g), zero between F and Fp; parts 2: what
// they were rounded by at 2 Fp further on
void gated_dact_launch(int type, const float* g, const float* u, const void* dh, int64_t lddh,
                       int64_t M, int F, int Fp, int act, int parts, void* dgdu, hipStream_t st);
// dst[r][0..np) <- src[r][0..n) converted, zeros from n on
void gated_operand_launch(const void* src, int src_type, int64_t ld, int64_t R, int n, void* dst,
                          int dst_type, int np, hipStream_t st);

}  // namespace pca
