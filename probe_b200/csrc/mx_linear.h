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

// Few tokens (mx_small.cu) and many (mx_gemm.cu).  Few: one tile of 128 tokens, or as
// many 128 x 128 tiles as there are SMs.
bool mx_few_tokens(int64_t M, int64_t N, int num_sms);
int mx_small_launch(const MxLinearOperands& o, int fmt, int dtype, cudaStream_t stream);
int mx_gemm_launch(const MxLinearOperands& o, int fmt, int dtype, cudaStream_t stream);

// Copies rows of `cols` elements of 2 bytes, of any alignment, to 16-byte aligned rows of
// `width` (a multiple of 8; zeros beyond cols).  Rows <= 2^31 - 1, width <= 2^28.
int mx_widen_launch(const void* in, int64_t ldi, void* out, int64_t rows, int64_t cols, int64_t width, cudaStream_t s);

// 2-D TMA map over rows of `inner` elements of 1, 2 or 4 bytes.
bool mx_encode_map(CUtensorMap* map, const void* ptr, int elem, int64_t inner, int64_t outer, int64_t pitch_bytes,
                   int box_inner, int box_outer, bool swizzle);

// Launch with a thread-block cluster of `cluster` CTAs along x (0: none) and, unless
// the process turned it off, as a programmatic dependent of the kernel before it:
// the kernel calls pdl_wait before it touches what that one reads or writes, and
// lets its own dependents start only after that, so that a kernel which reads
// weights ahead of its wait finds everything up to two launches back complete.
template <typename... P, typename... A>
int mx_launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 0) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return LORA_ERR_CUDA;
  }
  return LORA_OK;
}

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
