// Host interface of the input gradient of few rows (mx_dx.cu).
#pragma once

#include "mx_linear.h"

namespace lora {

// dx[t, k] = alpha (sum_n dy[t, n] Wv[n, k] + sum_j g[t, j] A[j, k]), Wv the values of the
// 4-bit W [N, K] times pow2.  bf16: g is the pair [hi | lo].  fp16: g [hi | mid | lo] and
// A = a + a_lo are sums of bf16 parts.
struct MxDxOperands {
  const void *dy, *w_codes, *w_scales, *g, *a, *a_lo;  // dy [M, lddy], rows of 16 bytes; a [R, lda], likewise
  void* dx;
  int64_t lddy, ldg, r16, lda, lddx, M, N, K, R;
  float alpha, pow2;
};

// Few rows: one tile of 256, or as many 256 x 128 tiles as there are SMs.
bool mx_dx_few(int64_t M, int64_t K, int num_sms);
int mx_dx_launch(const MxDxOperands& o, int fmt, int dtype, cudaStream_t stream);

}  // namespace lora
