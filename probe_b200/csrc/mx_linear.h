// Host interface between the 4-bit LoRA linear's entry point and its kernels.
#pragma once

#include "mx.cuh"

namespace lora {

// out = alpha (2^-dshift base + z B^T) + bias, base = the block-scaled product.
struct MxLinearOperands {
  const void *x_codes, *x_scales, *w_codes, *w_scales;
  const void* z;  // [M, ldz]: hi part at column 0, lo part at z_lo; R columns each are read
  const void* b;  // [N, ldb]
  const void* bias;
  void* out;
  int64_t ldz, z_lo, ldb, ldo, M, N, K, R;
  float alpha;
  int dshift;
};

// Few tokens (mx_small.cu) and many (mx_gemm.cu).
int mx_small_launch(const MxLinearOperands& o, int fmt, int dtype, cudaStream_t stream);
int mx_gemm_launch(const MxLinearOperands& o, int fmt, int dtype, cudaStream_t stream);

// 2-D TMA map over rows of `inner` elements of 1, 2 or 4 bytes.
bool mx_encode_map(CUtensorMap* map, const void* ptr, int elem, int64_t inner, int64_t outer, int64_t pitch_bytes,
                   int box_inner, int box_outer, bool swizzle);

inline size_t mx_align(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
inline bool mx_aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// alpha = product of the tensor scales = scale * 2^-shift, scale in [1, 2) where
// alpha is small enough (shift 0..30).
inline void mx_split_alpha(double alpha, float* scale, int* shift) {
  int e = 0;
  frexp(alpha, &e);  // alpha in [2^(e-1), 2^e)
  *shift = e - 1 < 0 ? (1 - e < 30 ? 1 - e : 30) : 0;
  *scale = static_cast<float>(ldexp(alpha, *shift));
}

}  // namespace lora
