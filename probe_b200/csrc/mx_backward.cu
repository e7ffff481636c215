// Backward pass of the LoRA linear from an 8-bit checkpoint of its input.
//
//   g  = s dy B                [M, R]
//   dB = zs dy^T z             [N, R]     z: the forward pass's hi/lo pair
//   dA = g^T X8                [R, K]
//   dx = dy Wq + g A           [M, K]     where asked for
//
// The base weight is frozen; rounding to 4 or 8 bits counts as the identity
// (straight-through).  dx needs W with N as the contraction, against the direction
// of its scale blocks.  Few rows (mx_dx_few): W is decoded on its way into the MMAs
// (mx_dx.cu).  Many: W is decoded once, transposed, into the workspace and the 16-bit
// CTA-pair GEMM takes [g_hi | g_lo] against [A^T | A^T] as its K tail.  Either way W's
// values are exact in 16 bits: nvfp4's tensor scale m 2^p leaves the power of two in the
// values and m in the product's alpha.
#include <cmath>

#include "mx_dx.h"
#include "mx_grad.h"
#include "mx_shrink.h"

namespace lora {
namespace {

// Ranks above this, of enough rows, take g = s dy B from the 16-bit CTA-pair GEMM,
// which halves the shared-memory reads of so wide an adapter (r = 224, 32760 x 5120: 83
// against 109 us).
constexpr int64_t kWideRank = 128, kWideRows = 4096;

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct BackwardPlan {
  bool few;  // dx of few rows
  size_t gemm_bytes, part, part_a, g, bt, at, dy, wt, total;
};

BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int64_t R, bool need_dx) {
  BackwardPlan p = {};
  const int64_t np = up(N, 8), rp = up(R, 16);
  const int dev = current_device();
  p.few = need_dx && mx_dx_few(M, K, dev >= 0 ? device_info(dev).num_sms : 148);
  if (need_dx && !p.few) p.gemm_bytes = lora_gemm_workspace_size(M, K, np, 2 * rp);
  if (R > kWideRank && M >= kWideRows) p.gemm_bytes = std::max(p.gemm_bytes, lora_gemm_workspace_size(M, R, np, 0));
  size_t at = kCounterBytes;  // ticket counters, never scratch; the steps' partials follow them in turn
  at = std::max(at, mx_align(std::max(kCounterBytes + mx_shrink_part_bytes(M, np, R), p.gemm_bytes)));
  p.part = at;
  at += mx_align(mx_grad_part_bytes(M, N, R));
  p.part_a = at;
  at += mx_align(mx_grad_part_bytes(M, K, R));
  p.g = at;
  at += mx_align(static_cast<size_t>(M) * 2 * rp * 2);
  p.bt = at;
  at += mx_align(static_cast<size_t>(R) * np * 2);
  p.at = at;
  if (need_dx) at += mx_align(p.few ? static_cast<size_t>(R) * up(K, 8) * 2 : static_cast<size_t>(K) * 2 * rp * 2);
  p.dy = at;
  at += mx_align(static_cast<size_t>(M) * np * 2);
  p.wt = at;
  if (need_dx && !p.few) at += mx_align(static_cast<size_t>(K) * np * 2);
  p.total = at;
  return p;
}

// out[c, j] = in[j, c] for in [rows, cols], j < width (zeros beyond rows); `copies`
// of the width columns side by side.  32 x 32 a block; the blocks of two matrices
// side by side.
struct TransposeJob {
  const uint16_t* in;
  uint16_t* out;
  int64_t ldi, ldo, rows, cols, width;
  int copies, blocks_c, blocks;
};
struct TransposeJobs {
  TransposeJob of[2];
};

__global__ void __launch_bounds__(256) mx_transpose_kernel(const TransposeJobs jobs) {
  __shared__ uint16_t tile[32][34];
  const bool second = static_cast<int>(blockIdx.x) >= jobs.of[0].blocks;
  const TransposeJob& t = second ? jobs.of[1] : jobs.of[0];
  const int block = second ? blockIdx.x - jobs.of[0].blocks : blockIdx.x;
  const int64_t c0 = static_cast<int64_t>(block % t.blocks_c) * 32, j0 = static_cast<int64_t>(block / t.blocks_c) * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t j = j0 + ty + 8 * i, c = c0 + tx;
    tile[ty + 8 * i][tx] = j < t.rows && c < t.cols ? t.in[j * t.ldi + c] : 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = c0 + ty + 8 * i, j = j0 + tx;
    if (c < t.cols && j < t.width)
      for (int k = 0; k < t.copies; ++k) t.out[c * t.ldo + k * t.width + j] = tile[tx][ty + 8 * i];
  }
}

TransposeJob transpose_job(const void* in, int64_t ldi, void* out, int64_t ldo, int64_t rows, int64_t cols, int64_t width,
                           int copies) {
  TransposeJob t{static_cast<const uint16_t*>(in), static_cast<uint16_t*>(out), ldi, ldo, rows, cols, width, copies};
  t.blocks_c = static_cast<int>(up(cols, 32) / 32);
  t.blocks = t.blocks_c * static_cast<int>(up(width, 32) / 32);
  return t;
}

int transpose(const TransposeJobs& jobs, cudaStream_t s) {
  const int blocks = jobs.of[0].blocks + jobs.of[1].blocks;
  if (blocks == 0) return LORA_OK;
  mx_transpose_kernel<<<blocks, 256, 0, s>>>(jobs);
  return cudaGetLastError() == cudaSuccess ? LORA_OK : LORA_ERR_CUDA;
}

}  // namespace
}  // namespace lora

using namespace lora;

extern "C" size_t lora_mx_backward_workspace_size(int64_t M, int64_t N, int64_t K, int64_t R, int need_dx) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0) return 0;
  return backward_plan(M, N, K, R, need_dx != 0).total;
}

extern "C" int lora_mx_backward(const void* dy, int64_t lddy, const void* x_codes, const void* x_scales, const void* z,
                                float z_scale, const void* a, int64_t lda, const void* b, int64_t ldb,
                                const void* w_codes, const void* w_scales, float w_global, int w_fmt, void* dx,
                                int64_t lddx, void* da, int64_t ldda, void* db, int64_t lddb, int64_t M, int64_t N,
                                int64_t K, int64_t R, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (dtype != LORA_BF16 && dtype != LORA_F16) return LORA_ERR_DTYPE;
  if (dx != nullptr && w_fmt != LORA_MXFP4 && w_fmt != LORA_NVFP4) return LORA_ERR_DTYPE;
  if (M < 0 || N < 0 || K < 0 || R <= 0 || R > 256 || M > 4194240 || N > 4194240 || K > 4194240) return LORA_ERR_SHAPE;
  if (lddy < N || lda < K || ldb < R || ldda < K || lddb < R || (dx != nullptr && lddx < K)) return LORA_ERR_SHAPE;
  if (dx != nullptr && !mx_global_ok(w_global, w_fmt)) return LORA_ERR_ARG;
  if (K == 0) return LORA_ERR_UNSUPPORTED;
  // an empty sum leaves zeros: no operand is read
  const bool empty = M == 0 || N == 0;
  if (da == nullptr || (N > 0 && db == nullptr)) return LORA_ERR_ARG;
  if (!empty && (a == nullptr || b == nullptr || dy == nullptr || x_codes == nullptr || x_scales == nullptr ||
                 z == nullptr || (dx != nullptr && (w_codes == nullptr || w_scales == nullptr))))
    return LORA_ERR_ARG;
  if (!mx_aligned(x_codes, 16) || !mx_aligned(x_scales, 16) || !mx_aligned(z, 16) || !mx_aligned(workspace, 256) ||
      (dx != nullptr && (!mx_aligned(w_codes, 16) || !mx_aligned(w_scales, 16))))
    return LORA_ERR_ALIGN;
  const int dev = current_device();
  if (dev < 0 || !device_info(dev).is_sm100) return LORA_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (empty) {
    if (cudaMemset2DAsync(da, ldda * 2, 0, K * 2, R, s) != cudaSuccess ||
        (N > 0 && cudaMemset2DAsync(db, lddb * 2, 0, R * 2, N, s) != cudaSuccess) ||
        (M > 0 && dx != nullptr && cudaMemset2DAsync(dx, lddx * 2, 0, K * 2, M, s) != cudaSuccess))
      return LORA_ERR_CUDA;
    return LORA_OK;
  }
  const BackwardPlan p = backward_plan(M, N, K, R, dx != nullptr);
  if (workspace == nullptr || workspace_bytes < p.total) return LORA_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  const int64_t np = up(N, 8), rp = up(R, 16);

  // factor m of the tensor scale m 2^q; 2^q goes into the decoded values
  float m = 1.f, pow2 = 1.f;
  if (dx != nullptr && w_fmt == LORA_NVFP4) {
    int e = 0;
    m = 2.f * static_cast<float>(frexp(w_global, &e));
    pow2 = static_cast<float>(ldexp(1.0, e - 1));
  }
  // What the weights give comes first: a kernel that reads it may start before its own
  // predecessor on the stream has finished, so other launches lie between.
  TransposeJobs jobs = {};
  const bool b_rows = mx_aligned(b, 16) && ldb % 8 == 0;  // TMA can read them
  const bool wide = R > kWideRank && M >= kWideRows;
  if (!b_rows || wide) jobs.of[0] = transpose_job(b, ldb, ws + p.bt, np, N, R, np, 1);
  if (dx != nullptr && !p.few) jobs.of[1] = transpose_job(a, lda, ws + p.at, 2 * rp, R, K, rp, 2);
  int rc = transpose(jobs, s);
  if (rc != LORA_OK) return rc;
  const void* ap = a;
  int64_t lda_p = lda;
  if (p.few && (lda % 8 != 0 || !mx_aligned(a, 16))) {
    lda_p = up(K, 8);
    ap = ws + p.at;
    rc = mx_widen_launch(a, lda, ws + p.at, R, K, lda_p, s);
    if (rc != LORA_OK) return rc;
  }
  if (dx != nullptr && !p.few) {
    rc = mx_dequantize_launch(w_codes, w_scales, ws + p.wt, np, N, K, w_fmt, pow2, 2, dtype, s);
    if (rc != LORA_OK) return rc;
  }
  const void* dyp = dy;
  int64_t ldp = lddy;
  if (N % 8 != 0 || lddy % 8 != 0 || !mx_aligned(dy, 16)) {  // TMA needs 16-byte rows
    rc = mx_widen_launch(dy, lddy, ws + p.dy, M, N, np, s);
    if (rc != LORA_OK) return rc;
    dyp = ws + p.dy;
    ldp = np;
  }
  MxGradOperands grads[2] = {};
  MxGradOperands& gr = grads[0];
  gr.v = dyp;
  gr.ldv = ldp;
  gr.p = z;
  gr.ldp = 2 * rp;
  gr.out = db;
  gr.ldo = lddb;
  gr.part = ws + p.part;
  gr.M = M;
  gr.C = N;
  gr.R = R;
  gr.factor = z_scale;

  MxShrinkOperands sh = {};
  sh.v = dyp;
  sh.a = b;
  sh.a_mn = b_rows;
  sh.lda = ldb;
  if (!sh.a_mn) {
    sh.a = ws + p.bt;
    sh.lda = np;
  }
  sh.z = ws + p.g;
  sh.tickets = ws;
  sh.part = ws + kCounterBytes;
  sh.ldv = ldp;
  sh.ldz = 2 * rp;
  sh.M = M;
  sh.K = N;
  sh.R = R;
  sh.scale = scale / m;
  sh.global_scale = 1.f;
  if (wide) {
    if (rp != R && cudaMemsetAsync(ws + p.g, 0, static_cast<size_t>(M) * 2 * rp * 2, s) != cudaSuccess)
      return LORA_ERR_CUDA;
    rc = lora_gemm_ex(dyp, ldp, ws + p.bt, np, nullptr, 0, nullptr, 0, nullptr, ws + p.g, 2 * rp, M, R, np, 0, scale / m,
                      rp, dtype, p.gemm_bytes ? ws : nullptr, p.gemm_bytes, s);
  } else {
    rc = mx_shrink_launch(sh, -1, dtype, s);
  }
  if (rc != LORA_OK) return rc;

  MxGradOperands& ga = grads[1];
  ga = gr;
  ga.v = x_codes;
  ga.v_scales = x_scales;
  ga.p = ws + p.g;
  ga.out = da;
  ga.ldo = ldda;
  ga.part = ws + p.part_a;
  ga.C = K;
  ga.factor = m;
  ga.transposed = true;
  rc = mx_grad_launch(grads, dtype, s);
  if (rc != LORA_OK) return rc;
  rc = mx_grad_reduce_launch(grads, dtype, s);
  if (rc != LORA_OK || dx == nullptr) return rc;

  if (p.few) {
    MxDxOperands o = {};
    o.dy = dyp;
    o.lddy = ldp;
    o.w_codes = w_codes;
    o.w_scales = w_scales;
    o.g = ws + p.g;
    o.ldg = 2 * rp;
    o.g_lo = rp;
    o.a = ap;
    o.lda = lda_p;
    o.dx = dx;
    o.lddx = lddx;
    o.M = M;
    o.N = N;
    o.K = K;
    o.R = R;
    o.alpha = m;
    o.pow2 = pow2;
    return mx_dx_launch(o, w_fmt, dtype, s);
  }
  return lora_gemm_ex(dyp, ldp, ws + p.wt, np, ws + p.g, 2 * rp, ws + p.at, 2 * rp, nullptr, dx, lddx, M, K, np, 2 * rp,
                      m, 0, dtype, p.gemm_bytes ? ws : nullptr, p.gemm_bytes, s);
}
