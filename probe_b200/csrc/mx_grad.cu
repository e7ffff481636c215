// Adapter gradients: out[c, j] = factor * sum_t V[t, c] P[t, j], a contraction
// over tokens.
//
//   dB = dy^T z    V = dy (16-bit),            P = z
//   dA = (s dy B)^T X    V = X (mxfp8 checkpoint), P = s dy B, written transposed
//
// tcgen05 with both operands MN-major: TMA brings V and P as they lie in memory
// (tokens as rows, 64-column chunks, 128-byte swizzle) and the transposition is
// the MMA's.  A CTA owns 256 columns of V (two M = 128 accumulators, N = r) and a
// range of tokens, so V is read once from HBM; P, r columns wide, is read once per
// 256 columns of V through L2.  The fp32 partials of the token ranges are summed
// in a fixed order by a second kernel (no atomics).
//
// An mxfp8 V arrives as codes and scale chunks; sixteen warps turn it into 16-bit
// values in the MMA's swizzled layout.  E4M3 times a power of two is exact in
// bf16: the code's exponent and mantissa moved into place, times 2^120, times the
// scale.  Bound: HBM for small ranks (2 or 1.03 bytes an element of V), the MMAs, both of
// whose operands come from shared memory, for large ones.  Both gradients
// of 4097 tokens, 4096 -> 11008, r = 16, 107 MB: 46 us with the partials; of 32760 tokens,
// 5120 -> 5120: 129 at r = 64, 162 at r = 128, 284 to 300 at r = 224 (300 GFLOP, the tensor pipe
// half busy).  They are one launch: the second's blocks start as the
// first's leave, and few tokens' blocks run side by side (256 tokens, 4096 -> 4096: 4.7 us
// instead of 4.0 + 7.8 with waits).
// P is the whole hi/lo pair.  Up to rank 128 its halves lie side by side in one MMA (N = 2 r)
// and are added in the epilogue; above, they meet V one after the other in the same
// accumulator, from stages of half as many tokens.  dA of fp16 activations is computed in
// bf16, where X is exact too, with g in three parts: a gradient beside a B that has just
// left zero lies below fp16's range, a scaled loss's beyond it.  The hi half alone would take 145 us at
// r = 224, but its rounding is as large as that of the 16-bit result.
#include <mutex>

#include "mx_grad.h"

namespace lora {
namespace {

constexpr int kGrCols = 256;  // columns of V a CTA
constexpr int kGrConvWarps = 16;
constexpr int kGrThreads = 64 + 32 * kGrConvWarps;
constexpr int kGrScaleBytes = 2 * 512;  // scale chunks of a stage (128 tokens x 256 columns)
constexpr int kGrSmemMax = 224 * 1024;
constexpr int kGrMaxN = 256;  // columns of one MMA
// TOK tokens a stage.
template <int TOK>
struct GrStage {
  static constexpr int kChunk = TOK * 128;      // TOK tokens x 64 16-bit columns
  static constexpr int kV = 4 * kChunk;         // 16-bit V
  static constexpr int kRaw = TOK * kGrCols;    // codes
};

struct GrMaps {
  CUtensorMap v, p, sc;
};

struct GrArgs {
  float* part;  // [splits][C][ldp]
  int* err;
  int64_t C;
  int r16, parts;
  int n, passes, p_chunks;  // N of an MMA; the runs of P that meet V in turn, 64-column chunks of each
  int stages, stage_bytes, steps_per_split, steps, splits, scale_gb;
};

LORA_DEVINL uint32_t gr_mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 v =
      __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight E4M3 codes times their scale 2^(s - 127), as bf16 values in order.
LORA_DEVINL uint4 gr_decode8(uint2 w, uint32_t s) {
  // two codes in the high bytes of each half: exponent and mantissa moved into
  // bf16's place are 2^-120 of the code's value
  const uint32_t p[4] = {__byte_perm(w.x, 0, 0x1404), __byte_perm(w.x, 0, 0x3424), __byte_perm(w.y, 0, 0x1404),
                         __byte_perm(w.y, 0, 0x3424)};
  uint32_t o[4];
  if (s <= 134) {  // 2^120 and the scale in one factor: 2^(s - 7) is a normal bf16 number
    const uint32_t f = ((s + 120) << 7) * 0x10001u;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = gr_mul_bf16x2((p[i] & 0x80008000u) | ((p[i] >> 4) & 0x07f007f0u), f);
  } else {
    const uint32_t f = (s == 255 ? 0x7fffu : s << 7) * 0x10001u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = gr_mul_bf16x2(gr_mul_bf16x2((p[i] & 0x80008000u) | ((p[i] >> 4) & 0x07f007f0u), 0x7b807b80u), f);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Shared memory: the TMA ring (stage: V or codes + scales, then P), for mxfp8 two
// converted tiles, then the barriers.
template <typename T, bool F8, int TOK>
LORA_DEVINL void gr_job(const GrMaps& maps, const GrArgs& args, int group, int split) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  using S = GrStage<TOK>;
  constexpr int kPOffset = F8 ? S::kRaw + kGrScaleBytes : S::kV;
  uint8_t* conv = smem + args.stages * args.stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(conv + (F8 ? 2 * S::kV : 0));
  uint64_t* empty = full + 8;
  uint64_t* ready = empty + 8;       // [2] converted tile written
  uint64_t* conv_empty = ready + 2;  // [2] converted tile read by its MMAs
  uint64_t* acc_full = conv_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col0 = static_cast<int64_t>(group) * kGrCols;
  const int step0 = split * args.steps_per_split;
  const int step1 = min(step0 + args.steps_per_split, args.steps);
  const uint32_t tmem_cols = args.n <= 16 ? 32u : args.n <= 32 ? 64u : args.n <= 64 ? 128u : args.n <= 128 ? 256u : 512u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ready[s], kGrConvWarps);
      mbar_init(&conv_empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.v);
    tma_prefetch_desc(&maps.p);
    if (F8) tma_prefetch_desc(&maps.sc);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      const uint32_t bytes = kPOffset + args.passes * args.p_chunks * S::kChunk;
      for (int st = step0; st < step1; ++st) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty)) break;
        uint8_t* base = smem + stage * args.stage_bytes;
        mbar_arrive_expect_tx(&full[stage], bytes);
        const int tok = st * TOK;
        if constexpr (F8) {
          tma_load_2d(&maps.v, base, &full[stage], static_cast<int>(col0), tok);
          tma_load_2d(&maps.sc, base + S::kRaw, &full[stage], 0,
                      (tok >> 7) * args.scale_gb + static_cast<int>(col0 >> 7));
        } else {
          for (int c = 0; c < 4; ++c)
            tma_load_2d(&maps.v, base + c * S::kChunk, &full[stage], static_cast<int>(col0) + 64 * c, tok);
        }
        uint8_t* p = base + kPOffset;
        for (int i = 0; i < args.passes; ++i)
          for (int c = 0; c < args.p_chunks; ++c, p += S::kChunk)
            tma_load_2d(&maps.p, p, &full[stage], i * args.r16 + 64 * c, tok);
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the stages (uniform descriptors); one lane issues.  Both
    // operands MN-major (bits 15 and 16), M = 128.
    const uint32_t idesc = (umma_idesc_f16(128, 16, std::is_same<T, __nv_bfloat16>::value ? 1 : 0) & ~(0x3fu << 17)) |
                           (static_cast<uint32_t>(args.n >> 3) << 17) | (1u << 15) | (1u << 16);
    const uint64_t desc0 = mx_desc_mn(smem_u32(smem), S::kChunk);
    const uint64_t conv0 = mx_desc_mn(smem_u32(conv), S::kChunk);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int st = step0; st < step1; ++st) {
      const int n = st - step0;
      if (!warp_wait(&full[stage], phase, abort_flag, args.err, kDevErrTimeoutFull) ||
          (F8 && !warp_wait(&ready[n & 1], (n >> 1) & 1, abort_flag, args.err, kDevErrTimeoutFull))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t base = desc0 + static_cast<uint32_t>((stage * args.stage_bytes) >> 4);
      const uint64_t v = F8 ? conv0 + static_cast<uint32_t>(((n & 1) * S::kV) >> 4) : base;
      if (elect_one()) {
        uint64_t pd = base + static_cast<uint32_t>(kPOffset >> 4);
        for (int i = 0; i < args.passes; ++i, pd += static_cast<uint32_t>((args.p_chunks * S::kChunk) >> 4)) {
#pragma unroll
          for (int k = 0; k < TOK / 16; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m)
              tc_mma_f16(tmem + m * args.n, v + static_cast<uint32_t>((m * 2 * S::kChunk + k * 2048) >> 4),
                         pd + static_cast<uint32_t>((k * 2048) >> 4), idesc, (n > 0 || i > 0 || k > 0) ? 1u : 0u);
        }
        tc_commit(&empty[stage]);
        if (F8) tc_commit(&conv_empty[n & 1]);
      }
      __syncwarp();
      if (++stage == args.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (ok && elect_one()) tc_commit(acc_full);
    __syncwarp();
  } else {
    const int cw = warp - 2;
    if constexpr (F8) {
      int stage = 0;
      uint32_t phase = 0;
      for (int st = step0; st < step1; ++st) {
        const int n = st - step0;
        if (!warp_wait(&full[stage], phase, abort_flag, args.err, kDevErrTimeoutFull) ||
            !warp_wait(&conv_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty))
          break;
        const uint32_t raw = smem_u32(smem) + stage * args.stage_bytes;
        // the scale chunk of this lane's 128 columns, its block
        const uint32_t sc = raw + S::kRaw + (lane >> 4) * 512 + ((lane >> 2) & 3);
        const uint32_t dst = smem_u32(conv) + (n & 1) * S::kV + (lane >> 3) * S::kChunk;
#pragma unroll
        for (int i = 0; i < TOK / kGrConvWarps; ++i) {
          const int t = cw * (TOK / kGrConvWarps) + i;
          const int tr = (st * TOK + t) & 127;  // row within the scale chunk
          const uint2 w = lds64(raw + t * kGrCols + lane * 8);
          const uint32_t s = lds_u8(sc + (tr & 31) * 16 + (tr >> 5) * 4);
          sts128(dst + t * 128 + (((lane & 7) ^ (t & 7)) << 4), gr_decode8(w, s));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ready[n & 1]);
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // epilogue: lane quadrant, accumulator, every other group of 16 ranks
    const int quad = warp & 3, m = (cw >> 2) & 1;
    if (warp_wait(acc_full, 0, abort_flag, args.err, kDevErrTimeoutAccFull)) {
      tc_fence_after();
      const int64_t c = col0 + m * 128 + quad * 32 + lane;
      float* dst = args.part + (static_cast<int64_t>(split) * args.C + c) * args.r16;
      for (int j = (cw >> 3) * 16; j < args.r16; j += 32) {
        const uint32_t src = tmem + (static_cast<uint32_t>(quad * 32) << 16) + m * args.n + j;
        uint32_t r[16], lo[16];
        tmem_ld_32x32b_x16(src, r);
        tmem_wait_ld();
        for (int i = args.passes; i < args.parts; ++i) {  // (passes is 1 or parts)
          tmem_ld_32x32b_x16(src + i * args.r16, lo);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(lo[e]));
        }
        if (c < args.C) {
          st_global_v8(dst + j, r);
          st_global_v8(dst + j + 8, r + 8);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// Both gradients of a call in one launch: the blocks of dB, then those of dA, which
// start as the first leave.
struct GrJobs {
  GrMaps maps[2];
  GrArgs args[2];
  int groups[2], blocks0;
};

template <typename T, int TOK>
__global__ void __launch_bounds__(kGrThreads, 1) mx_grad_kernel(const __grid_constant__ GrJobs jobs) {
  const int b = static_cast<int>(blockIdx.x);
  if (b < jobs.blocks0) {
    gr_job<T, false, TOK>(jobs.maps[0], jobs.args[0], b % jobs.groups[0], b / jobs.groups[0]);
  } else {
    const int c = b - jobs.blocks0;
    gr_job<__nv_bfloat16, true, TOK>(jobs.maps[1], jobs.args[1], c % jobs.groups[1], c / jobs.groups[1]);
  }
}

// Sum of the splits in order, times factor, rounded to T: out[c, j] (ldo) or,
// transposed, out[j, c].  32 columns of V x 32 ranks a block; the blocks of several
// gradients side by side.
struct GrSum {
  const float* part;
  void* out;
  int64_t ldo, C;
  int r, r16, splits, blocks;
  float factor;
  bool transposed;
};
struct GrSums {
  GrSum of[2];
};

template <typename T>
__global__ void __launch_bounds__(256) mx_grad_reduce_kernel(const GrSums sums) {
  __shared__ float tile[32][33];
  pdl_wait();
  pdl_launch_dependents();
  const bool second = static_cast<int>(blockIdx.x) >= sums.of[0].blocks;
  const GrSum& g = second ? sums.of[1] : sums.of[0];
  T* out = static_cast<T*>(g.out);
  const int64_t c0 = static_cast<int64_t>(second ? blockIdx.x - sums.of[0].blocks : blockIdx.x) * 32;
  const int j0 = blockIdx.y * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const int j = j0 + tx;
  for (int s = 0; s < g.splits; ++s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = c0 + ty + 8 * i;
      if (c < g.C && j < g.r) v[i] += g.part[(s * g.C + c) * g.r16 + j];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = c0 + ty + 8 * i;
    if (g.transposed)
      tile[ty + 8 * i][tx] = v[i] * g.factor;
    else if (c < g.C && j < g.r)
      out[c * g.ldo + j] = from_f32<T>(v[i] * g.factor);
  }
  if (g.transposed) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = c0 + tx;
      if (c < g.C && j0 + ty + 8 * i < g.r) out[(j0 + ty + 8 * i) * g.ldo + c] = from_f32<T>(tile[tx][ty + 8 * i]);
    }
  }
}

struct GrPlan {
  int groups, steps, splits, steps_per_split;
};

// Tokens a stage: half of the usual ones where dA's parts of P do not fit one MMA, so
// that three stages or more of them fit beside the decoded tiles.
int grad_tokens(int64_t R, int parts) { return parts * ((R + 15) / 16 * 16) > kGrMaxN ? 32 : 64; }

GrPlan grad_plan(int64_t M, int64_t C, int tok) {
  GrPlan p;
  const int dev = current_device();
  const int sms = dev >= 0 ? device_info(dev).num_sms : 148;
  p.groups = static_cast<int>((C + kGrCols - 1) / kGrCols);
  p.steps = static_cast<int>((M + tok - 1) / tok);
  int splits = std::max(1, sms / p.groups);
  splits = std::min(splits, p.steps);
  p.steps_per_split = (p.steps + splits - 1) / splits;
  p.splits = (p.steps + p.steps_per_split - 1) / p.steps_per_split;
  return p;
}

// Maps and arguments of one gradient; its shared memory through `smem`.
template <int TOK>
bool fill_job(const MxGradOperands& g, const GrPlan& pl, bool f8, int* err, GrMaps* maps, GrArgs* a, size_t* smem) {
  a->part = static_cast<float*>(g.part);
  a->err = err;
  a->C = g.C;
  a->r16 = static_cast<int>((g.R + 15) / 16 * 16);
  // the parts side by side in one MMA, or one after the other
  a->parts = g.parts;
  a->passes = g.parts * a->r16 > kGrMaxN ? g.parts : 1;
  a->n = a->passes == 1 ? g.parts * a->r16 : a->r16;
  a->p_chunks = (a->n + 63) / 64;
  a->steps = pl.steps;
  a->splits = pl.splits;
  a->steps_per_split = pl.steps_per_split;
  a->scale_gb = static_cast<int>(mx_scale_chunks(g.C, LORA_MXFP8));
  using S = GrStage<TOK>;
  a->stage_bytes = (f8 ? S::kRaw + kGrScaleBytes : S::kV) + a->passes * a->p_chunks * S::kChunk;
  const int fixed = (f8 ? 2 * S::kV : 0) + 512 + 1024;
  a->stages = std::min(8, (kGrSmemMax - fixed) / a->stage_bytes);
  *smem = std::max(*smem, static_cast<size_t>(a->stages) * a->stage_bytes + fixed);
  if (f8) {
    const int64_t pitch = mx_padded_k(g.C);
    if (!mx_encode_map(&maps->v, g.v, 1, pitch, g.M, pitch, kGrCols, TOK, false) ||
        !mx_encode_map(&maps->sc, g.v_scales, 4, 128, (g.M + 127) / 128 * a->scale_gb, 512, 128, 2, false))
      return false;
  } else {
    if (!mx_encode_map(&maps->v, g.v, 2, g.C, g.M, g.ldv * 2, 64, TOK, true)) return false;
    maps->sc = maps->v;
  }
  return mx_encode_map(&maps->p, g.p, 2, g.parts * a->r16, g.M, g.ldp * 2, 64, TOK, true);
}

template <typename T, int TOK>
int launch_grads(const MxGradOperands* g, cudaStream_t stream) {
  const int dev = current_device();
  if (dev < 0) return LORA_ERR_DEVICE;
  const DeviceInfo& info = device_info(dev);
  GrJobs jobs;
  size_t smem = 0;
  int blocks = 0;
  for (int i = 0; i < 2; ++i) {
    const GrPlan pl = grad_plan(g[i].M, g[i].C, TOK);
    if (!fill_job<TOK>(g[i], pl, i == 1, info.err_word, &jobs.maps[i], &jobs.args[i], &smem)) return LORA_ERR_CUDA;
    jobs.groups[i] = pl.groups;
    if (i == 1) jobs.blocks0 = blocks;
    blocks += pl.groups * pl.splits;
  }
  auto kernel = mx_grad_kernel<T, TOK>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGrSmemMax);
  });
  if (attr_err[dev] != cudaSuccess) return LORA_ERR_CUDA;
  return mx_launch(kernel, dim3(blocks), kGrThreads, smem, stream, 0, jobs);
}

}  // namespace

size_t mx_grad_part_bytes(int64_t M, int64_t C, int64_t R, int parts) {
  return static_cast<size_t>(grad_plan(M, C, grad_tokens(R, parts)).splits) * C * ((R + 15) / 16 * 16) * sizeof(float);
}

int mx_grad_launch(const MxGradOperands* g, int dtype, cudaStream_t stream) {
  if (grad_tokens(g[1].R, g[1].parts) == 32)
    return dtype == LORA_BF16 ? launch_grads<__nv_bfloat16, 32>(g, stream) : launch_grads<__half, 32>(g, stream);
  return dtype == LORA_BF16 ? launch_grads<__nv_bfloat16, 64>(g, stream) : launch_grads<__half, 64>(g, stream);
}

int mx_grad_reduce_launch(const MxGradOperands* g, int dtype, cudaStream_t stream) {
  const int tok = grad_tokens(g[1].R, g[1].parts);
  GrSums sums = {};
  int blocks = 0, r32 = 0;
  for (int i = 0; i < 2; ++i) {
    GrSum& s = sums.of[i];
    s.part = static_cast<const float*>(g[i].part);
    s.out = g[i].out;
    s.ldo = g[i].ldo;
    s.C = g[i].C;
    s.r = static_cast<int>(g[i].R);
    s.r16 = (s.r + 15) / 16 * 16;
    s.splits = grad_plan(g[i].M, g[i].C, tok).splits;
    s.blocks = static_cast<int>((g[i].C + 31) / 32);
    s.factor = g[i].factor;
    s.transposed = g[i].transposed;
    blocks += s.blocks;
    r32 = std::max(r32, (s.r + 31) / 32);
  }
  return mx_launch(dtype == LORA_BF16 ? mx_grad_reduce_kernel<__nv_bfloat16> : mx_grad_reduce_kernel<__half>,
                   dim3(blocks, r32), 256, 0, stream, 0, sums);
}

}  // namespace lora
