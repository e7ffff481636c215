// 4-bit LoRA linear of few tokens: W streamed once through block-scaled MMAs with
// the tokens as the narrow operand.
//
//   out[t, n] = alpha (2^-d sum_k wq[n,k] sw xq[t,k] sx + sum_j B[n,j] (zh + zl)[t,j]) + bias[n]
//
// tcgen05.mma.kind::mxf4nvf4 with 128 rows of W as M and the tokens (16..128) as N;
// the adapter's products go to an accumulator of their own (kind::f16, B's rows as
// M), so the two kinds never meet and the power of two is taken in the epilogue.
// Bound: HBM, 0.53 (mxfp4) or 0.56 (nvfp4) bytes a weight; for a handful of tokens
// the chain of launches and latencies.  So K is cut over a cluster of up to 8 CTAs
// until about two CTAs an SM stream W; their partial tiles meet in shared memory
// and are summed in rank order over DSMEM.  The kernel starts while its predecessor
// (the shrink that makes xq, sx and z) still runs: W's first stages load before
// griddepcontrol.wait.  Measured, wait included: one token, 4096 -> 11008, mxfp4, 24 MB:
// 7.8 us; 64 tokens, 5120 -> 13824, nvfp4, 40 MB: 11.2.
#include <cmath>
#include <mutex>

#include "mx_tile.cuh"

namespace lora {
namespace {

constexpr int kSmThreads = 192;
// Two CTAs an SM, each with at most half of TMEM, or (128 tokens) one with all of
// it: none of a launch waits for another's.
template <int NB> __host__ __device__ constexpr int sm_smem_max() { return NB == 128 ? 220 * 1024 : 112 * 1024; }
template <int NB> __host__ __device__ constexpr int sm_tmem_max() { return NB == 128 ? 512 : 256; }

struct SmMaps {
  CUtensorMap x, w, sx, sw, zh, zl, b;
};

struct SmArgs {
  MxTileOut tile;
  int* err;
  int num_kb, last_step, rank_kb, last_k16, chunks, stages;
};

LORA_DEVINL void sm_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT, int NB>
struct SmLayout {
  static constexpr int kChunks = 256 / MxFormat<FMT>::kBlock / 4;
  static constexpr int kW = 128 * 128, kX = NB * 128, kSf = kChunks * 512;
  static constexpr int kStage = (kW + kX + 2 * kSf + 1023) / 1024 * 1024;
  static constexpr int kXOffset = kW, kSfOffset = kW + kX;
  static constexpr int kMainBytes = kW + kX + 2 * kSf;
  static constexpr int kSfCols = 2 * kChunks * 4;
  // TMEM: base accumulator, adapter accumulator, scales of every stage
  static constexpr int kFit = (sm_tmem_max<NB>() - 2 * NB) / kSfCols;
  static constexpr int kMaxStages = kFit < 8 ? kFit : 8;
};

template <typename T, int FMT, int NB>
__global__ void __launch_bounds__(kSmThreads)
    mx_small_kernel(const __grid_constant__ SmMaps maps, const SmArgs args) {
  using L = SmLayout<FMT, NB>;
  constexpr uint32_t kCols = 2 * NB + L::kMaxStages * L::kSfCols;
  constexpr uint32_t kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kTmemCols <= sm_tmem_max<NB>(), "TMEM");
  constexpr uint32_t kIdesc = (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NB >> 3) << 17) |
                              ((FMT == LORA_MXFP4 ? 1u : 0u) << 23) | (8u << 24);
  constexpr uint32_t kIdescTail = (1u << 4) | ((std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) << 7) |
                                  ((std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) << 10) |
                                  (static_cast<uint32_t>(NB >> 3) << 17) | (8u << 24);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + args.stages * L::kStage);
  uint64_t* empty = full + 8;
  uint64_t* acc_full = empty + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int splits = 1;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int rank = static_cast<int>(cluster_ctarank());
  const int n0 = static_cast<int>(blockIdx.x) / splits * 128;
  const int t0 = static_cast<int>(blockIdx.y) * NB;
  const int kb0 = args.num_kb * rank / splits, kb1 = args.num_kb * (rank + 1) / splits;
  // the adapter's stages follow the first rank's base stages
  const int tail_kb = rank == 0 ? 2 * args.rank_kb : 0;
  const int total = kb1 - kb0 + tail_kb;

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      auto weights = [&](int i, int stage) {
        uint8_t* base = smem + stage * L::kStage;
        if (i < kb1 - kb0) {
          mbar_arrive_expect_tx(&full[stage], L::kMainBytes);
          tma_load_2d(&maps.w, base, &full[stage], (kb0 + i) * 128, n0);
          tma_load_2d(&maps.sw, base + L::kSfOffset, &full[stage], 0,
                      (n0 >> 7) * args.chunks + (kb0 + i) * L::kChunks);
        } else {
          const int t = i - (kb1 - kb0);
          mbar_arrive_expect_tx(&full[stage], L::kW + L::kX);
          tma_load_2d(&maps.b, base, &full[stage], (t >= args.rank_kb ? t - args.rank_kb : t) * 64, n0);
        }
      };
      auto tokens = [&](int i, int stage) {
        uint8_t* base = smem + stage * L::kStage;
        if (i < kb1 - kb0) {
          tma_load_2d(&maps.x, base + L::kXOffset, &full[stage], (kb0 + i) * 128, t0);
          tma_load_2d(&maps.sx, base + L::kSfOffset + L::kSf, &full[stage], 0,
                      (t0 >> 7) * args.chunks + (kb0 + i) * L::kChunks);
        } else {
          const int t = i - (kb1 - kb0);
          const bool lo = t >= args.rank_kb;
          tma_load_2d(lo ? &maps.zl : &maps.zh, base + L::kXOffset, &full[stage], (lo ? t - args.rank_kb : t) * 64, t0);
        }
      };
      const int pre = min(total, args.stages);
      for (int i = 0; i < pre; ++i) weights(i, i);
      pdl_wait();  // the shrink's codes, scales and z
      pdl_launch_dependents();
      for (int i = 0; i < pre; ++i) tokens(i, i);
      int stage = pre == args.stages ? 0 : pre;
      uint32_t phase = pre == args.stages ? 1 : 0;
      for (int i = pre; i < total; ++i) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty)) break;
        weights(i, stage);
        tokens(i, stage);
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint64_t wd0 = umma_desc_sw128(smem_u32(smem));
    const uint64_t xd0 = umma_desc_sw128(smem_u32(smem) + L::kXOffset);
    const uint64_t sd0 = mx_desc_scales(smem_u32(smem) + L::kSfOffset);
    for (int i = 0; i < total; ++i) {
      if (!warp_wait(&full[stage], phase, abort_flag, args.err, kDevErrTimeoutFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t at = static_cast<uint32_t>(stage * (L::kStage >> 4));
      const uint64_t wd = wd0 + at, xd = xd0 + at, sd = sd0 + at;
      if (i < kb1 - kb0) {
        const uint32_t sfa = tmem + 2 * NB + stage * L::kSfCols, sfb = sfa + L::kChunks * 4;
        const int nk = kb0 + i == args.num_kb - 1 ? args.last_step : 4;
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < L::kChunks; ++j) {
            sm_cp_scales(sfa + 4 * j, sd + static_cast<uint32_t>(32 * j));
            sm_cp_scales(sfb + 4 * j, sd + static_cast<uint32_t>(32 * (L::kChunks + j)));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            constexpr bool kMx = FMT == LORA_MXFP4;
            const int j = kMx ? k >> 1 : k;
            const uint32_t id = kMx ? static_cast<uint32_t>(k & 1) * 2u : 0u;
            if (k < nk)
              mx_mma<FMT, false>(tmem, wd + static_cast<uint32_t>(2 * k), xd + static_cast<uint32_t>(2 * k),
                          kIdesc | (id << 4) | (id << 29), sfa + 4 * j, sfb + 4 * j, (i > 0 || k > 0) ? 1u : 0u);
          }
          tc_commit(&empty[stage]);
        }
      } else {
        const int t = i - (kb1 - kb0);
        const int c = t >= args.rank_kb ? t - args.rank_kb : t;
        const int nk = c == args.rank_kb - 1 ? args.last_k16 : 4;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < nk)
              tc_mma_f16(tmem + NB, wd + static_cast<uint32_t>(2 * k), xd + static_cast<uint32_t>(2 * k), kIdescTail,
                         (t > 0 || k > 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
        }
      }
      __syncwarp();
      if (++stage == args.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (ok && elect_one()) tc_commit(acc_full);
    __syncwarp();
  }

  mx_tile_out<T, NB, kSmThreads, 2, 4, kTmemCols>(args.tile, reinterpret_cast<float*>(smem), tmem,
                                                  tail_kb > 0 ? NB : 0, acc_full, abort_flag, args.err, splits, rank,
                                                  n0, t0);
}

template <typename T, int FMT, int NB>
int launch_small(const MxLinearOperands& o, cudaStream_t stream) {
  using L = SmLayout<FMT, NB>;
  const int dev = current_device();
  if (dev < 0) return LORA_ERR_DEVICE;
  const DeviceInfo& info = device_info(dev);
  SmMaps maps;
  SmArgs a;
  const int64_t pitch = mx_code_pitch(o.K, FMT);
  a.chunks = static_cast<int>(mx_scale_chunks(o.K, FMT));
  if (!mx_encode_map(&maps.x, o.x_codes, 1, pitch, o.M, pitch, 128, NB, true) ||
      !mx_encode_map(&maps.w, o.w_codes, 1, pitch, o.N, pitch, 128, 128, true) ||
      !mx_encode_map(&maps.sx, o.x_scales, 4, 128, (o.M + 127) / 128 * a.chunks, 512, 128, L::kChunks, false) ||
      !mx_encode_map(&maps.sw, o.w_scales, 4, 128, (o.N + 127) / 128 * a.chunks, 512, 128, L::kChunks, false))
    return LORA_ERR_CUDA;
  if (o.R > 0) {
    const char* z = static_cast<const char*>(o.z);
    if (!mx_encode_map(&maps.zh, z, 2, o.R, o.M, o.ldz * 2, 64, NB, true) ||
        !mx_encode_map(&maps.zl, z + o.z_lo * 2, 2, o.R, o.M, o.ldz * 2, 64, NB, true) ||
        !mx_encode_map(&maps.b, o.b, 2, o.R, o.N, o.ldb * 2, 64, 128, true))
      return LORA_ERR_CUDA;
  } else {
    maps.zh = maps.zl = maps.b = maps.x;
  }
  a.tile = {o.out, o.bias, o.ldo, static_cast<int>(o.M), static_cast<int>(o.N), o.alpha, ldexpf(1.f, -o.dshift)};
  a.err = info.err_word;
  const int64_t kp = mx_padded_k(o.K);
  a.num_kb = static_cast<int>((kp + 255) / 256);
  a.last_step = static_cast<int>((kp - static_cast<int64_t>(a.num_kb - 1) * 256 + 63) / 64);
  a.rank_kb = static_cast<int>((o.R + 63) / 64);
  a.last_k16 = a.rank_kb > 0 ? static_cast<int>((o.R - (a.rank_kb - 1) * 64ll + 15) / 16) : 0;
  // The partial tile (NB x 128 fp32) lies over the stages.
  constexpr int kFixed = 1024 + 256;
  a.stages = std::min<int>(L::kMaxStages, (sm_smem_max<NB>() - kFixed) / L::kStage);
  const int n_tiles = static_cast<int>((o.N + 127) / 128), t_tiles = static_cast<int>((o.M + NB - 1) / NB);
  // as many CTAs as are resident at once, each with four or more stages of K
  const int resident = (NB == 128 ? 1 : 2) * info.num_sms;
  int splits = 1;
  while (splits < 8 && n_tiles * t_tiles * splits * 2 <= resident && a.num_kb >= 8 * splits) splits *= 2;
  // over a third (NB 128: half) of an SM's shared memory: no third (second) CTA joins
  size_t smem = static_cast<size_t>(a.stages) * L::kStage;
  static_assert(L::kStage * 2 >= NB * 512 || NB == 128, "the partial tile lies over the stages");
  if (smem < static_cast<size_t>(NB) * 512) return LORA_ERR_UNSUPPORTED;
  smem = std::max<size_t>(smem + kFixed, NB == 128 ? 120 * 1024 : 80 * 1024);
  auto kernel = mx_small_kernel<T, FMT, NB>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sm_smem_max<NB>());
  });
  if (attr_err[dev] != cudaSuccess) return LORA_ERR_CUDA;
  return mx_launch(kernel, dim3(n_tiles * splits, t_tiles), kSmThreads, smem, stream, splits, maps, a);
}

template <typename T, int FMT>
int dispatch(const MxLinearOperands& o, cudaStream_t s) {
  if (o.M <= 16) return launch_small<T, FMT, 16>(o, s);
  if (o.M <= 32) return launch_small<T, FMT, 32>(o, s);
  if (o.M <= 64) return launch_small<T, FMT, 64>(o, s);
  return launch_small<T, FMT, 128>(o, s);
}

}  // namespace

int mx_small_launch(const MxLinearOperands& o, int fmt, int dtype, cudaStream_t s) {
  if (dtype == LORA_BF16)
    return fmt == LORA_MXFP4 ? dispatch<__nv_bfloat16, LORA_MXFP4>(o, s) : dispatch<__nv_bfloat16, LORA_NVFP4>(o, s);
  return fmt == LORA_MXFP4 ? dispatch<__half, LORA_MXFP4>(o, s) : dispatch<__half, LORA_NVFP4>(o, s);
}

}  // namespace lora
