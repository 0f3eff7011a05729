// Host interface of distill.hip.
#pragma once
#include "common.h"

namespace pca {

constexpr int kDistillMaxClasses = 1 << 18;   // classes of a row (the kept-class map is 32 KiB)
constexpr int kDistillMaxK = 1024;            // kept logits of a row
constexpr double kDistillMinTemp = 5.421010862427522e-20;   // 2^-64
constexpr double kDistillRest = 1.0 / (1 << 20);

enum LogitType : int { LOGIT_F32 = 0, LOGIT_BF16 = 1, LOGIT_F16 = 2 };

// the K largest of each of R rows, descending, and log sum exp(z / T)
void top_logits_launch(const void* z, int type, int64_t ld, int64_t R, int V, int k, double temp,
                       void* values, int32_t* indices, float* lse, hipStream_t st);

struct DistillArgs {
  const void* z;            // [R][V], row stride ld
  int64_t ld;
  int64_t R;
  int V, K;
  const void* values;       // [R][K] of value_type, dense
  const void* indices;      // [R][K] int32 or int64, dense; negative: not kept
  const float* lse;         // [R], read if tail
  const int64_t* target;    // [R] or null
  void* dz;                 // [R][V] dense, or null: no gradient
  float* row_loss;          // [R], or null: not wanted
  const float* seed;        // the loss's gradient, [R] or one number for all, or null: ones
  double temp, alpha;       // alpha: weight of the teacher's part
  float grad_scale;         // of every gradient: 1/R for a mean
  int64_t ignore_index;
  int type, value_type;
  int index64, tail;
  int seed_rows;            // 1: a seed a row
  int keep;                 // rows of dz whose seed is one are there already
};
void distill_launch(const DistillArgs& a, hipStream_t st);
// loss <- scale * sum of R row losses (fixed order)
void distill_sum_launch(const float* row_loss, int64_t R, double scale, float* loss,
                        hipStream_t st);

}  // namespace pca
