// The LoRA linear with 4-bit base operands: its steps and its entry point.
//
//   out = q(x) W^T + s (x A^T) B^T + bias
//
// q(x): x quantised to W's format; the adapter sees x itself.  Steps: q(x) and, in
// the same pass over x, the rank shrink z = (s / alpha) x A^T as a hi/lo pair
// (alpha: the fp32 factor that the product's epilogue applies); the block-scaled
// GEMM with z B^T as its tail.  Operands that TMA cannot read (rows not 16-byte
// aligned) take the quantisation and the split-K shrink as kernels of their own or,
// at ranks beyond that shrink's, are copied to aligned rows first.
#include <cmath>

#include "mx_shrink.h"

namespace lora {
namespace {

// The most ranks that lora_shrink takes.
constexpr int64_t kShrinkMaxRank = 128;

int64_t r16(int64_t r) { return (r + 15) / 16 * 16; }

struct LinearPlan {
  size_t shrink_bytes, x_codes, x_scales, z, b, x, a, total;
  int split_k;
};

// Workspace: the shrink's (its ticket region first, zeroed once), then scratch.
LinearPlan linear_plan(int64_t M, int64_t N, int64_t K, int64_t R, int fmt) {
  LinearPlan p = {};
  size_t at = kCounterBytes;  // never scratch: calls of other shapes find their tickets zero
  if (R > 0) {
    const size_t fused = kCounterBytes + mx_shrink_part_bytes(M, K, R);
    if (fused > at) at = mx_align(fused);
    if (R <= kShrinkMaxRank) {
      p.split_k = lora_shrink_pick_split_k(M, K, R);
      p.shrink_bytes = lora_shrink_workspace_size(M, R, p.split_k);
    }
    if (p.shrink_bytes > at) at = mx_align(p.shrink_bytes);
  }
  p.x_codes = at;
  at += mx_align(lora_mx_codes_size(M, K, fmt));
  p.x_scales = at;
  at += mx_align(lora_mx_scales_size(M, K, fmt));
  p.z = at;
  if (R > 0) at += mx_align(static_cast<size_t>(M) * 2 * r16(R) * 2);
  p.b = at;
  if (R % 8 != 0) at += mx_align(static_cast<size_t>(N) * ((R + 7) / 8 * 8) * 2);
  // x and A, where rows of a wide adapter's operands may need a copy
  const int64_t k8 = (K + 7) / 8 * 8;
  const bool copies = R > kShrinkMaxRank && K % 8 != 0;
  p.x = at;
  if (copies) at += mx_align(static_cast<size_t>(M) * k8 * 2);
  p.a = at;
  if (copies) at += mx_align(static_cast<size_t>(R) * k8 * 2);
  p.total = at;
  return p;
}

// Rows of `cols` elements to 16-byte aligned rows of `width`, 16 elements a thread.
__global__ void __launch_bounds__(256) mx_widen_kernel(const uint16_t* __restrict__ in, int64_t ldi,
                                                       uint16_t* __restrict__ out, int64_t cols, int64_t width) {
  const int64_t row = blockIdx.x, c = (static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x) * 16;
  if (c >= width) return;
  uint32_t w[8];
  ldg16_any(in + row * ldi, c, cols, w);
  uint4* dst = reinterpret_cast<uint4*>(out + row * width + c);
  dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if (c + 8 < width) dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// B [N, R] with rows padded to a multiple of 8 elements (TMA needs 16-byte rows).
__global__ void mx_pad_rows_kernel(const uint16_t* __restrict__ b, int64_t ldb, uint16_t* __restrict__ out, int64_t N,
                                   int R, int R8) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= N * R8) return;
  const int64_t n = i / R8;
  const int j = static_cast<int>(i - n * R8);
  out[i] = j < R ? b[n * ldb + j] : 0;
}

}  // namespace

// Measured whole calls, r = 16, mxfp4, against 256 x 256 pair tiles: N = K = 4096, 333
// tokens 17.6 against 23.3 us, 512 18.8 against 23.5, 768 (192 tiles) 27.4 against 23.7;
// N = 11008, 256 (172 tiles) 26.9 against 23.5.
bool mx_few_tokens(int64_t M, int64_t N, int num_sms) {
  return M <= 128 || (M + 127) / 128 * ((N + 127) / 128) <= num_sms;
}

int mx_widen_launch(const void* in, int64_t ldi, void* out, int64_t rows, int64_t cols, int64_t width, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((width + 4095) / 4096));
  mx_widen_kernel<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(in), ldi, static_cast<uint16_t*>(out), cols, width);
  return cudaGetLastError() == cudaSuccess ? LORA_OK : LORA_ERR_CUDA;
}

}  // namespace lora

using namespace lora;

extern "C" size_t lora_mx_linear_workspace_size(int64_t M, int64_t N, int64_t K, int64_t R, int fmt) {
  if (M <= 0 || N <= 0 || K <= 0 || R < 0 || (fmt != LORA_MXFP4 && fmt != LORA_NVFP4)) return 0;
  return linear_plan(M, N, K, R, fmt).total;
}

extern "C" float lora_mx_linear_z_scale(float x_global, float w_global, int fmt) {
  float scale = 1.f;
  int shift = 0;
  if (fmt == LORA_NVFP4) mx_split_alpha(static_cast<double>(x_global) * w_global, &scale, &shift);
  return scale;
}

extern "C" int lora_mx_linear(const void* x, int64_t ldx, const void* w_codes, const void* w_scales, float w_global,
                              const void* bias, const void* a, int64_t lda, const void* b, int64_t ldb, void* out,
                              int64_t ldo, void* z_out, int64_t M, int64_t N, int64_t K, int64_t R, float scale,
                              float x_global, int fmt, int dtype, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if ((fmt != LORA_MXFP4 && fmt != LORA_NVFP4) || (dtype != LORA_BF16 && dtype != LORA_F16)) return LORA_ERR_DTYPE;
  if (M < 0 || N < 0 || K < 0 || R < 0 || R > 256 || M > 8388480 || N > 8388480 || K > (int64_t{1} << 24))
    return LORA_ERR_SHAPE;
  if (ldx < K || ldo < N || (R > 0 && (lda < K || ldb < R))) return LORA_ERR_SHAPE;
  if (!mx_global_ok(w_global, fmt) || !mx_global_ok(x_global, fmt)) return LORA_ERR_ARG;
  if (M == 0 || N == 0) return LORA_OK;
  if (K == 0) return LORA_ERR_UNSUPPORTED;
  if (x == nullptr || w_codes == nullptr || w_scales == nullptr || out == nullptr) return LORA_ERR_ARG;
  if (R > 0 && (a == nullptr || b == nullptr)) return LORA_ERR_ARG;
  if (!mx_aligned(w_codes, 16) || !mx_aligned(w_scales, 16) || !mx_aligned(workspace, 256) ||
      (z_out != nullptr && !mx_aligned(z_out, 16)))
    return LORA_ERR_ALIGN;
  const bool served = R > 0 && mx_shrink_serves(x, ldx, a, lda);
  const bool copies = R > kShrinkMaxRank && !served;
  if (copies && K % 8 == 0) return LORA_ERR_ALIGN;  // the workspace has no room for copies
  const int dev = current_device();
  if (dev < 0 || !device_info(dev).is_sm100) return LORA_ERR_DEVICE;
  const LinearPlan p = linear_plan(M, N, K, R, fmt);
  if (workspace == nullptr || workspace_bytes < p.total) return LORA_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  MxLinearOperands o = {};
  o.alpha = 1.f;
  if (fmt == LORA_NVFP4) {
    const double alpha = static_cast<double>(x_global) * w_global;
    if (R > 0) {
      mx_split_alpha(alpha, &o.alpha, &o.dshift);
    } else {
      o.alpha = static_cast<float>(alpha);
    }
  }
  o.b = b;
  o.ldb = ldb;
  // two launches ahead of the kernel that reads B, which may start before its own
  // predecessor on the stream has finished
  if (R > 0 && (ldb % 8 != 0 || !mx_aligned(b, 16))) {
    if (R % 8 == 0) return LORA_ERR_ALIGN;
    const int r8 = static_cast<int>((R + 7) / 8 * 8);
    const int64_t n = N * r8;
    mx_pad_rows_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(
        static_cast<const uint16_t*>(b), ldb, reinterpret_cast<uint16_t*>(ws + p.b), N, static_cast<int>(R),
        r8);
    if (cudaGetLastError() != cudaSuccess) return LORA_ERR_CUDA;
    o.b = ws + p.b;
    o.ldb = r8;
  }
  int rc = LORA_OK;
  const int64_t rp = r16(R);
  char* z = z_out != nullptr ? static_cast<char*>(z_out) : ws + p.z;
  const float zs = scale / o.alpha;
  if (copies) {
    const int64_t k8 = (K + 7) / 8 * 8;
    rc = mx_widen_launch(x, ldx, ws + p.x, M, K, k8, s);
    if (rc == LORA_OK) rc = mx_widen_launch(a, lda, ws + p.a, R, K, k8, s);
    if (rc != LORA_OK) return rc;
    x = ws + p.x;
    a = ws + p.a;
    ldx = lda = k8;
  }
  if (served || copies) {
    MxShrinkOperands sh = {};
    sh.v = x;
    sh.a = a;
    sh.z = z;
    sh.codes = ws + p.x_codes;
    sh.scales = ws + p.x_scales;
    sh.tickets = ws;
    sh.part = ws + kCounterBytes;
    sh.ldv = ldx;
    sh.lda = lda;
    sh.ldz = 2 * rp;
    sh.M = M;
    sh.K = K;
    sh.R = R;
    sh.scale = zs;
    sh.global_scale = x_global;
    rc = mx_shrink_launch(sh, fmt, dtype, s);
  } else {
    rc = mx_quantize_launch(x, ldx, ws + p.x_codes, ws + p.x_scales, M, K, fmt, x_global, dtype, s);
    if (rc == LORA_OK && R > 0)
      rc = lora_shrink(x, ldx, a, lda, z, 2 * rp, dtype, rp, 1, M, K, R, zs, dtype, p.split_k, ws, p.shrink_bytes, s);
  }
  if (rc != LORA_OK) return rc;
  if (R > 0) {
    o.z = z;
    o.ldz = 2 * rp;
    o.z_lo = rp;
  }
  o.x_codes = ws + p.x_codes;
  o.x_scales = ws + p.x_scales;
  o.w_codes = w_codes;
  o.w_scales = w_scales;
  o.bias = bias;
  o.out = out;
  o.ldo = ldo;
  o.M = M;
  o.N = N;
  o.K = K;
  o.R = R;
  if (mx_few_tokens(M, N, device_info(dev).num_sms)) return mx_small_launch(o, fmt, dtype, s);
  return mx_gemm_launch(o, fmt, dtype, s);
}
