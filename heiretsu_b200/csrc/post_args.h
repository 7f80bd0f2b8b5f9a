// Arguments of the post-training loss kernels (post_loss.cu), filled by the torch-facing
// checks (post_host.cpp).
#pragma once

#include <cstdint>

namespace hb {

// Element type of a logits matrix.
enum LogitType : int { kLogitBf16 = 0, kLogitF16 = 1, kLogitF32 = 2 };

struct LogitRows {
  const void* x;           // [M, >= V], row stride ld elements
  long ld;
  int M, V;
  int type;                // LogitType
  const int64_t* targets;  // [M]
  int64_t ignore_index;
  float* logp;             // [M] log-probability of the target (0 for ignored rows)
  float* lse;              // [M] log-sum-exp of the row (0 for ignored rows), or nullptr
  void* grad;              // [M, W], row stride gld, the logits' type; may be x itself; nullptr: none
  long gld;
  int W;                   // without a gradient: the logits' width
  int* status;
};

struct PolicyTerms {
  const float* old_logp;    // [M]
  const float* adv;         // [M / adv_rows]: one advantage per adv_rows consecutive rows
  int adv_rows;
  const float* ref_logp;    // [M], or nullptr
  const float* weights;     // [M], or nullptr: 1 / (rows whose target is not ignored)
  const float* grad_scale;  // [1] upstream gradient, or nullptr: 1
  float clip_lo, clip_hi;   // the ratio is clipped to [clip_lo, clip_hi]
  float kl_coef;
};

}  // namespace hb
