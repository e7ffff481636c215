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

#include "gemm_pair.cuh"
#include "mx_dx.h"
#include "mx_grad.h"
#include "mx_shrink.h"

namespace lora {
namespace {

// Ranks above this, of enough rows, take g = s dy B from the 16-bit CTA-pair GEMM,
// which halves the shared-memory reads of so wide an adapter; below, its few tiles leave
// SMs idle.  Whole passes without dx, us, GEMM and shrink: 5120 -> 5120, r = 224: 8192 rows
// 149 and 135, 16384 245 and 221, 20000 284 and 277, 24576 319 and 325, 32760 388 and 409;
// r = 256, 24576 rows 325 and 330; r = 192 288 and 282, 32760 348 and 357; r = 144 no gain
// (334 and 337); 4096 -> 11008, r = 224, 4096 rows 159 and 122.
constexpr int64_t kWideRank = 144, kWideRows = 24576;

// g of fp16 activations is kept in three bf16 parts, which never leave its range; beside
// A = Ah + Al the tail of dx takes [gh gm gl gh gm] against [Ah Ah Ah Al Al].
constexpr int kTailHigh = 3, kTailLow = 2, kTailGroups = kTailHigh + kTailLow;

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

struct BackwardPlan {
  bool few;    // dx of few rows
  bool wide;   // g from the pair GEMM
  int parts;   // of g, side by side
  int groups;  // of r16 columns of g: its parts, some of them again for the tail of dx
  size_t gemm_bytes, part, part_a, g, bt, at, dy, wt, total;
};

// dy_rows, b_rows: TMA can read dy, b where they lie.
BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int64_t R, bool need_dx, bool half, bool dy_rows,
                           bool b_rows) {
  BackwardPlan p = {};
  const int64_t np = up(N, 8), rp = up(R, 16);
  const int dev = current_device();
  p.few = need_dx && mx_dx_few(M, K, dev >= 0 ? device_info(dev).num_sms : 148);
  const bool many = need_dx && !p.few;
  p.parts = half ? kTailHigh : 2;
  p.groups = half && many ? kTailGroups : p.parts;
  p.wide = !half && R > kWideRank && M >= kWideRows;
  const int64_t tail = p.groups * rp;
  if (many) p.gemm_bytes = lora_gemm_workspace_size(M, K, np, tail);
  if (p.wide) p.gemm_bytes = std::max(p.gemm_bytes, lora_gemm_workspace_size(M, R, np, 0));
  size_t at = kCounterBytes;  // ticket counters, never scratch; the steps' partials follow them in turn
  at = std::max(at, mx_align(std::max(kCounterBytes + mx_shrink_part_bytes(M, np, R), p.gemm_bytes)));
  p.part = at;
  at += mx_align(mx_grad_part_bytes(M, N, R, p.parts));
  p.part_a = at;
  at += mx_align(mx_grad_part_bytes(M, K, R, p.parts));
  p.g = at;
  at += mx_align(static_cast<size_t>(M) * tail * 2);
  p.bt = at;
  if (p.wide || !b_rows) at += mx_align(static_cast<size_t>(R) * np * 2);
  p.at = at;
  if (many) at += mx_align(static_cast<size_t>(K) * tail * 2);
  if (p.few) at += mx_align(static_cast<size_t>(R) * up(K, 8) * (half ? 4 : 2));
  p.dy = at;
  if (!dy_rows) at += mx_align(static_cast<size_t>(M) * np * 2);
  p.wt = at;
  if (many) at += mx_align(static_cast<size_t>(K) * np * 2);
  p.total = at;
  return p;
}

// An fp16 value as the sum of two bf16 values (exact: 11 bits).
LORA_DEVINL void split_half(uint16_t v, uint16_t& hi, uint16_t& lo) {
  const float f = __half2float(__ushort_as_half(v));
  const __nv_bfloat16 h = __float2bfloat16_rn(f);
  hi = __bfloat16_as_ushort(h);
  lo = __bfloat16_as_ushort(__float2bfloat16_rn(f - __bfloat162float(h)));
}

// out[c, j] = in[j, c] for in [rows, cols], j < width (zeros beyond rows); `copies`
// of the width columns side by side and, of fp16 values in two bf16 parts, `lows` of the
// low part after them.  32 x 32 a block; the blocks of two matrices side by side.
struct TransposeJob {
  const uint16_t* in;
  uint16_t* out;
  int64_t ldi, ldo, rows, cols, width;
  int copies, lows, blocks_c, blocks;
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
    if (c < t.cols && j < t.width) {
      uint16_t hi = tile[tx][ty + 8 * i], lo = 0;
      if (t.lows > 0) split_half(hi, hi, lo);
      for (int k = 0; k < t.copies + t.lows; ++k) t.out[c * t.ldo + k * t.width + j] = k < t.copies ? hi : lo;
    }
  }
}

TransposeJob transpose_job(const void* in, int64_t ldi, void* out, int64_t ldo, int64_t rows, int64_t cols,
                           int64_t width, int copies, int lows) {
  TransposeJob t{static_cast<const uint16_t*>(in), static_cast<uint16_t*>(out), ldi, ldo, rows, cols, width, copies,
                 lows};
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

// fp16 rows of `cols` elements as two bf16 parts, hi [rows, width] and then lo (zeros
// beyond cols), 8 elements a thread.
__global__ void __launch_bounds__(256) mx_split_rows_kernel(const uint16_t* __restrict__ in, int64_t ldi,
                                                            uint16_t* __restrict__ out, int64_t rows, int64_t cols,
                                                            int64_t width) {
  const int64_t row = blockIdx.x, c = (static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x) * 8;
  if (c >= width) return;
  uint16_t h[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) split_half(c + i < cols ? in[row * ldi + c + i] : uint16_t{0}, h[i], l[i]);
  auto word = [](const uint16_t* v) { return v[0] | (static_cast<uint32_t>(v[1]) << 16); };
  uint16_t* dst = out + row * width + c;
  *reinterpret_cast<uint4*>(dst) = make_uint4(word(h), word(h + 2), word(h + 4), word(h + 6));
  *reinterpret_cast<uint4*>(dst + rows * width) = make_uint4(word(l), word(l + 2), word(l + 4), word(l + 6));
}

int split_rows(const void* in, int64_t ldi, void* out, int64_t rows, int64_t cols, int64_t width, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((width + 2047) / 2048));
  mx_split_rows_kernel<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(in), ldi, static_cast<uint16_t*>(out), rows,
                                            cols, width);
  return cudaGetLastError() == cudaSuccess ? LORA_OK : LORA_ERR_CUDA;
}

}  // namespace
}  // namespace lora

using namespace lora;

extern "C" size_t lora_mx_backward_workspace_size(int64_t M, int64_t N, int64_t K, int64_t R, int flags) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0) return 0;
  const bool dx = (flags & LORA_MX_NEED_DX) != 0;
  const bool dy_rows = (flags & LORA_MX_DY_ALIGNED) != 0 && N % 8 == 0, b_rows = (flags & LORA_MX_B_ALIGNED) != 0;
  const size_t bf16 = backward_plan(M, N, K, R, dx, false, dy_rows, b_rows).total;
  if (flags & LORA_MX_ONLY_BF16) return bf16;
  return std::max(bf16, backward_plan(M, N, K, R, dx, true, dy_rows, b_rows).total);
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
  const bool half = dtype == LORA_F16;
  const bool dy_rows = N % 8 == 0 && lddy % 8 == 0 && mx_aligned(dy, 16);
  const bool b_rows = mx_aligned(b, 16) && ldb % 8 == 0;
  const BackwardPlan p = backward_plan(M, N, K, R, dx != nullptr, half, dy_rows, b_rows);
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
  const bool many = dx != nullptr && !p.few;
  const int groups = p.groups;
  if (!b_rows || p.wide) jobs.of[0] = transpose_job(b, ldb, ws + p.bt, np, N, R, np, 1, 0);
  if (many)
    jobs.of[1] = transpose_job(a, lda, ws + p.at, groups * rp, R, K, rp, half ? kTailHigh : 2, half ? kTailLow : 0);
  int rc = transpose(jobs, s);
  if (rc != LORA_OK) return rc;
  const void* ap = a;
  int64_t lda_p = lda;
  if (p.few && (half || lda % 8 != 0 || !mx_aligned(a, 16))) {
    lda_p = up(K, 8);
    ap = ws + p.at;
    rc = half ? split_rows(a, lda, ws + p.at, R, K, lda_p, s) : mx_widen_launch(a, lda, ws + p.at, R, K, lda_p, s);
    if (rc != LORA_OK) return rc;
  }
  if (many) {
    rc = mx_dequantize_launch(w_codes, w_scales, ws + p.wt, np, N, K, w_fmt, pow2, 2, dtype, s);
    if (rc != LORA_OK) return rc;
  }
  const void* dyp = dy;
  int64_t ldp = lddy;
  if (!dy_rows) {
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
  gr.parts = 2;

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
  sh.ldz = groups * rp;
  sh.groups = groups;
  sh.M = M;
  sh.K = N;
  sh.R = R;
  sh.scale = scale / m;
  sh.global_scale = 1.f;
  if (p.wide) {
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
  ga.ldp = groups * rp;
  ga.parts = p.parts;
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
    o.ldg = groups * rp;
    o.r16 = rp;
    o.a = ap;
    if (half) o.a_lo = ws + p.at + R * lda_p * 2;
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
  const int64_t tail = groups * rp;
  return gemm_mixed_tail(dyp, ldp, ws + p.wt, np, ws + p.g, tail, ws + p.at, tail, dx, lddx, M, K, np, tail, m, dtype,
                         LORA_BF16, p.gemm_bytes ? ws : nullptr, p.gemm_bytes, s);
}
