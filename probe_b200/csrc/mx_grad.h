// Host interface of the adapter-gradient kernel (mx_grad.cu).
#pragma once

#include "mx_linear.h"

namespace lora {

// out[c, j] = factor * sum_t V[t, c] P[t, j]; P is a sum of `parts` parts side by side
// (2 or 3), R16 columns each; V is 16-bit (ldv) of P's type or, with v_scales, an mxfp8
// tensor, P being bf16; transposed writes out[j, c].
struct MxGradOperands {
  const void *v, *v_scales, *p;
  void *out, *part;  // part: mx_grad_part_bytes
  int64_t ldv, ldp, ldo, M, C, R;
  float factor;
  int parts;
  bool transposed;
};

// Of both gradients, dA's P in `parts` parts.
size_t mx_grad_part_bytes(int64_t M, int64_t C, int64_t R, int parts);
// g[0]: a 16-bit V, g[1]: an mxfp8 V.  The partial sums of both in one launch, and
// their sums in another.
int mx_grad_launch(const MxGradOperands* g, int dtype, cudaStream_t stream);
int mx_grad_reduce_launch(const MxGradOperands* g, int dtype, cudaStream_t stream);

}  // namespace lora
