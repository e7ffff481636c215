// Input gradient of the 4-bit LoRA linear for few rows of dy.
//
//   dx[t, k] = alpha (sum_n dy[t,n] Wv[n,k] + sum_j g[t,j] A[j,k])
//
// The contraction runs down W's rows, against the direction of its scale blocks, so
// the block-scaled MMAs do not apply; nor does a decoded copy of W pay for few rows
// (33 MB written and read for 4096 x 4096, four times the codes).  Here W is decoded
// on its way into the MMA: TMA brings the codes of 64 rows x 128 columns and their
// scale chunks, eight warps turn them into 16-bit values in the MN-major layout of
// the MMA's 128-wide operand -- 64-column chunks, token rows 128 bytes apart, the
// 128-byte swizzle -- so the transposition is the MMA's; dy's tile, 16..256 tokens, is
// the other operand.  A's rows, as they lie in memory, have that layout by TMA alone:
// they follow as the last stages, against the hi and then the lo part of g.  For fp16
// these stages are bf16 (g may lie outside fp16's range): A = Ah + Al exactly, g in three
// parts, and the products gh Ah, gm Ah, gl Ah, gh Al, gm Al; gl Al is below 2^-24 of g A.
//
// A code becomes a value in four instructions a pair: E2M1 to f16 by the converter,
// f16's exponent moved into bf16's place (a factor 2^-112, folded into the scale), one
// packed multiplication by the scale.  Codes have two significant bits and scales at
// most four, so the product is exact wherever it is a normal number of the type.
//
// Bound: the chain load -> decode -> MMA of a stage over a ring of four (64 tokens: three),
// whose 16-bit tiles fill the shared memory, then the decode's ALU work.  64 rows of
// 13824 x 5120 (nvfp4, r = 16) take 44 us, of which 11 are the decode's and 6 the MMAs'
// (each left out in turn); 256 rows of 4096 x 4096 18.  HBM's share is small, 0.53 or
// 0.56 bytes a weight.  So a tile takes up to 256 tokens, whose decode is then paid once (256 rows, whole backward pass: two tiles of 128
// 33.8 us, one of 256 28.3; 512 rows 52.8 and 39.5); from 128 tokens on, where one CTA
// fills an SM, two groups of eight warps decode stages in turn (128 rows, 4096 x 11008:
// 53.3 to 49.3), below, two CTAs of one group each share it (64 rows, 13824 x 5120: 55.8
// against 58.5 for a CTA of two groups).  The contraction is cut over a cluster as in the
// few-token linear, and W's first stages are loaded and decoded before
// griddepcontrol.wait.
#include <mutex>

#include "mx_dx.h"
#include "mx_tile.cuh"

namespace lora {
namespace {

constexpr int kDxGroupWarps = 8;       // decode a stage
constexpr int kDxRows = 64;            // of W (or A) a stage
constexpr int kDxHalf = kDxRows * 128;  // 64 rows x 64 16-bit columns
constexpr int kDxW = 2 * kDxHalf;      // the operand tile
constexpr int kDxRaw = kDxRows * 64;   // codes of a stage
// Two CTAs an SM, or (128 tokens and more) one, with two groups of decoding warps that
// take stages in turn.
template <int NB> __host__ __device__ constexpr int dx_ctas() { return NB >= 128 ? 1 : 2; }
template <int NB> __host__ __device__ constexpr int dx_smem_max() { return NB >= 128 ? 220 * 1024 : 112 * 1024; }
template <int NB> __host__ __device__ constexpr int dx_groups() { return NB >= 128 ? 2 : 1; }
template <int NB> __host__ __device__ constexpr int dx_threads() { return 64 + 32 * kDxGroupWarps * dx_groups<NB>(); }

struct DxMaps {
  CUtensorMap x, w, sw, g, a, al;
};

struct DxArgs {
  MxTileOut tile;
  int* err;
  int num_kb, last_step, rank_kb, last_k16, r16, gb;
  float pow2;
};

template <int FMT, int NB>
struct DxLayout {
  static constexpr int kChunks = 128 / MxFormat<FMT>::kBlock / 4;  // scale chunks of 128 columns
  static constexpr int kSf = kChunks * 512;
  static constexpr int kX = NB * 128;
  static constexpr int kXOffset = kDxW, kRawOffset = kDxW + kX, kSfOffset = kRawOffset + kDxRaw;
  static constexpr int kStage = (kSfOffset + kSf + 1023) / 1024 * 1024;
  static constexpr int kFixed = 1024 + 512;  // alignment, barriers
  // As many as fit, divided by the groups: a stage always goes to the same group, so that
  // a warp which waits for a stage's next tile has seen its last one -- a barrier's
  // parity says no more than that.
  static constexpr int kStages = (dx_smem_max<NB>() - kFixed) / kStage / dx_groups<NB>() * dx_groups<NB>();
  static constexpr size_t kBytes = static_cast<size_t>(kStages) * kStage + kFixed;
  static_assert(kStages == (NB == 64 ? 3 : 4), "the depth that the measurements are of");
  static_assert(kStages * kStage >= NB * 512, "the partial tile lies over the stages");
};

// Factor of a block of codes as a pair of the type, where one packed multiplication
// is exact: bf16 with 2^112 (see dx_decode8); fp16 in its normal range or zero.
template <typename T> LORA_DEVINL bool dx_factor(float f, uint32_t& pair);
template <> LORA_DEVINL bool dx_factor<__nv_bfloat16>(float f, uint32_t& pair) {
  pair = (__float_as_uint(f * 5.1922969e33f) >> 16) * 0x10001u;  // 2^112; at most four significant bits
  return f < 65536.f;
}
template <> LORA_DEVINL bool dx_factor<__half>(float f, uint32_t& pair) {
  pair = static_cast<uint32_t>(__half_as_ushort(__float2half_rn(f))) * 0x10001u;
  return f == 0.f || (f >= 6.1035156e-5f && f < 65536.f);
}

// Eight codes times an exact factor.
template <typename T> LORA_DEVINL uint4 dx_decode8(uint32_t w, uint32_t f);
template <> LORA_DEVINL uint4 dx_decode8<__nv_bfloat16>(uint32_t w, uint32_t f) {
  uint32_t h[4], o[4];
  mx_from_e2m1x8(w, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = (h[i] & 0x80008000u) | ((h[i] >> 3) & 0x0fff0fffu);
    const __nv_bfloat162 v =
        __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&f));
    o[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
template <> LORA_DEVINL uint4 dx_decode8<__half>(uint32_t w, uint32_t f) {
  uint32_t h[4], o[4];
  mx_from_e2m1x8(w, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hmul2_rn(*reinterpret_cast<const __half2*>(&h[i]), *reinterpret_cast<const __half2*>(&f));
    o[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// The same in fp32, rounded once, for every other factor (NaN, and results that are
// subnormal or out of range).
template <typename T>
LORA_DEVINL uint4 dx_decode8_any(uint32_t w, float f) {
  uint32_t h[4], o[4];
  mx_from_e2m1x8(w, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    o[i] = pack2<T>(q.x * f, q.y * f);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename T, int FMT, int NB>
__global__ void __launch_bounds__(dx_threads<NB>(), dx_ctas<NB>())
    mx_dx_kernel(const __grid_constant__ DxMaps maps, const DxArgs args) {
  using L = DxLayout<FMT, NB>;
  constexpr uint32_t kTmemCols = NB <= 32 ? 32 : NB;
  constexpr uint32_t kAb = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  // M = 128, W's operand MN-major (bit 15)
  constexpr uint32_t kIdesc =
      (1u << 4) | (kAb << 7) | (kAb << 10) | (1u << 15) | (static_cast<uint32_t>(NB >> 3) << 17) | (8u << 24);
  constexpr uint32_t kIdescTail = kIdesc | (1u << 7) | (1u << 10);
  constexpr int kTails = kAb ? 2 : 5;  // products of g's parts and A's

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full_w = reinterpret_cast<uint64_t*>(smem + L::kStages * L::kStage);
  uint64_t* full_x = full_w + 8;
  uint64_t* ready = full_x + 8;  // W decoded
  uint64_t* empty = ready + 8;
  uint64_t* acc_full = empty + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int splits = 1;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int rank = static_cast<int>(cluster_ctarank());
  const int k0 = static_cast<int>(blockIdx.x) / splits * 128;  // columns of dx
  const int t0 = static_cast<int>(blockIdx.y) * NB;
  const int kb0 = args.num_kb * rank / splits, base = args.num_kb * (rank + 1) / splits - kb0;
  // the adapter's stages follow the first rank's
  const int total = base + (rank == 0 ? kTails * args.rank_kb : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full_w[s], 1);
      mbar_init(&full_x[s], 1);
      mbar_init(&ready[s], kDxGroupWarps);
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
        uint8_t* at = smem + stage * L::kStage;
        if (i < base) {
          const int n = (kb0 + i) * kDxRows;
          mbar_arrive_expect_tx(&full_w[stage], kDxRaw + L::kSf);
          tma_load_2d(&maps.w, at + L::kRawOffset, &full_w[stage], k0 / 2, n);
          tma_load_2d(&maps.sw, at + L::kSfOffset, &full_w[stage], 0, (n >> 7) * args.gb + (k0 >> 7) * L::kChunks);
        } else {
          const int tail = (i - base) / args.rank_kb, j = ((i - base) % args.rank_kb) * kDxRows;
          const CUtensorMap* a = tail < 3 ? &maps.a : &maps.al;
          mbar_arrive_expect_tx(&full_w[stage], kDxW);
          tma_load_2d(a, at, &full_w[stage], k0, j);
          tma_load_2d(a, at + kDxHalf, &full_w[stage], k0 + 64, j);
        }
      };
      auto rows = [&](int i, int stage) {
        uint8_t* at = smem + stage * L::kStage + L::kXOffset;
        mbar_arrive_expect_tx(&full_x[stage], L::kX);
        if (i < base) {
          tma_load_2d(&maps.x, at, &full_x[stage], (kb0 + i) * kDxRows, t0);
        } else {
          // (columns beyond a part's, the next part's, meet rows of zeros)
          const int tail = (i - base) / args.rank_kb, c = (i - base) % args.rank_kb;
          tma_load_2d(&maps.g, at, &full_x[stage], (tail < 3 ? tail : tail - 3) * args.r16 + c * 64, t0);
        }
      };
      const int pre = min(total, L::kStages);
      for (int i = 0; i < pre; ++i) weights(i, i);
      pdl_wait();  // g
      pdl_launch_dependents();
      for (int i = 0; i < pre; ++i) rows(i, i);
      int stage = pre == L::kStages ? 0 : pre;
      uint32_t phase = pre == L::kStages ? 1 : 0;
      for (int i = pre; i < total; ++i) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty)) break;
        weights(i, stage);
        rows(i, stage);
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint64_t wd0 = mx_desc_mn(smem_u32(smem), kDxHalf);
    const uint64_t xd0 = umma_desc_sw128(smem_u32(smem) + L::kXOffset);
    for (int i = 0; i < total; ++i) {
      if (!warp_wait(&full_w[stage], phase, abort_flag, args.err, kDevErrTimeoutFull) ||
          !warp_wait(&full_x[stage], phase, abort_flag, args.err, kDevErrTimeoutFull) ||
          !warp_wait(&ready[stage], phase, abort_flag, args.err, kDevErrTimeoutFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t at = static_cast<uint32_t>(stage * (L::kStage >> 4));
      const int nk = i < base ? (kb0 + i == args.num_kb - 1 ? args.last_step : 4)
                              : ((i - base) % args.rank_kb == args.rank_kb - 1 ? args.last_k16 : 4);
      const uint32_t idesc = i < base ? kIdesc : kIdescTail;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < nk)
            tc_mma_f16(tmem, wd0 + at + static_cast<uint32_t>((k * 16 * 128) >> 4), xd0 + at + static_cast<uint32_t>(2 * k),
                       idesc, (i > 0 || k > 0) ? 1u : 0u);
        tc_commit(&empty[stage]);
      }
      __syncwarp();
      if (++stage == L::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (ok && elect_one()) tc_commit(acc_full);
    __syncwarp();
  } else {
    // a thread decodes 32 columns of a row; the upper 64 columns' threads take their
    // 16-byte units in another order, so that eight lanes' stores meet eight banks
    const int group = (warp - 2) / kDxGroupWarps, id = (threadIdx.x - 64) % (32 * kDxGroupWarps);
    const int r = id >> 2, seg = id & 3, swap = seg >> 1;
    const uint32_t src = smem_u32(smem) + L::kRawOffset + id * 16;
    const uint32_t dst = smem_u32(smem) + swap * kDxHalf + r * 128;
    const uint32_t sf = smem_u32(smem) + L::kSfOffset + (r & 31) * 16 + (r >> 5) * 4 +
                        (FMT == LORA_NVFP4 ? swap * 512 + (seg & 1) * 2 : seg);
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < total; ++i) {
      if (i % dx_groups<NB>() == group) {
        if (!warp_wait(&full_w[stage], phase, abort_flag, args.err, kDevErrTimeoutFull)) break;
        if (i < base) {
          const uint32_t at = static_cast<uint32_t>(stage * L::kStage);
          const uint32_t sa = sf + at + ((kb0 + i) & 1) * 8;  // odd stages: rows 64..127 of their scale chunk
          const uint4 q = lds128(src + at);
          const uint32_t w[4] = {swap ? q.z : q.x, swap ? q.w : q.y, swap ? q.x : q.z, swap ? q.y : q.w};
          float f[2];
          if constexpr (FMT == LORA_NVFP4) {
            f[0] = mx_e4m3(lds_u8(sa + swap)) * args.pow2;
            f[1] = mx_e4m3(lds_u8(sa + 1 - swap)) * args.pow2;
          } else {
            f[0] = f[1] = mx_e8m0(lds_u8(sa)) * args.pow2;
          }
  #pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pair;
            const bool exact = dx_factor<T>(f[h], pair);
  #pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = 2 * h + e;  // unit j ^ (2 swap) of this thread's four
              const uint4 v = exact ? dx_decode8<T>(w[j], pair) : dx_decode8_any<T>(w[j], f[h]);
              sts128(dst + at + (((((seg & 1) << 2) + (j ^ (2 * swap))) ^ (r & 7)) << 4), v);
            }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ready[stage]);
      }
      if (++stage == L::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }

  mx_tile_out<T, NB, dx_threads<NB>(), 2, kDxGroupWarps * dx_groups<NB>(), kTmemCols>(
      args.tile, reinterpret_cast<float*>(smem), tmem, 0, acc_full, abort_flag, args.err, splits, rank, k0, t0);
}

template <typename T, int FMT, int NB>
int launch_dx(const MxDxOperands& o, cudaStream_t stream) {
  using L = DxLayout<FMT, NB>;
  const int dev = current_device();
  if (dev < 0) return LORA_ERR_DEVICE;
  const DeviceInfo& info = device_info(dev);
  DxMaps maps;
  DxArgs a;
  const int64_t pitch = mx_code_pitch(o.K, FMT);
  a.gb = static_cast<int>(mx_scale_chunks(o.K, FMT));
  if (!mx_encode_map(&maps.x, o.dy, 2, o.N, o.M, o.lddy * 2, 64, NB, true) ||
      !mx_encode_map(&maps.w, o.w_codes, 1, pitch, o.N, pitch, 64, kDxRows, false) ||
      !mx_encode_map(&maps.sw, o.w_scales, 4, 128, (o.N + 127) / 128 * a.gb, 512, 128, L::kChunks, false) ||
      !mx_encode_map(&maps.g, o.g, 2, o.ldg, o.M, o.ldg * 2, 64, NB, true) ||
      !mx_encode_map(&maps.a, o.a, 2, o.K, o.R, o.lda * 2, 64, kDxRows, true))
    return LORA_ERR_CUDA;
  maps.al = maps.a;
  if (o.a_lo != nullptr && !mx_encode_map(&maps.al, o.a_lo, 2, o.K, o.R, o.lda * 2, 64, kDxRows, true))
    return LORA_ERR_CUDA;
  a.tile = {o.dx, nullptr, o.lddx, static_cast<int>(o.M), static_cast<int>(o.K), o.alpha, 1.f};
  a.err = info.err_word;
  a.num_kb = static_cast<int>((o.N + kDxRows - 1) / kDxRows);
  a.last_step = static_cast<int>((o.N - (a.num_kb - 1) * 64ll + 15) / 16);
  a.rank_kb = static_cast<int>((o.R + 63) / 64);
  a.last_k16 = static_cast<int>((o.R - (a.rank_kb - 1) * 64ll + 15) / 16);
  a.r16 = static_cast<int>(o.r16);
  a.pow2 = o.pow2;
  const int k_tiles = static_cast<int>((o.K + 127) / 128), t_tiles = static_cast<int>((o.M + NB - 1) / NB);
  // as many CTAs as are resident at once, each with eight or more stages
  const int resident = dx_ctas<NB>() * info.num_sms;
  int splits = 1;
  while (splits < 8 && k_tiles * t_tiles * splits * 2 <= resident && a.num_kb >= 16 * splits) splits *= 2;
  auto kernel = mx_dx_kernel<T, FMT, NB>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(L::kBytes));
  });
  if (attr_err[dev] != cudaSuccess) return LORA_ERR_CUDA;
  return mx_launch(kernel, dim3(k_tiles * splits, t_tiles), dx_threads<NB>(), L::kBytes, stream, splits, maps, a);
}

template <typename T, int FMT>
int dispatch(const MxDxOperands& o, cudaStream_t s) {
  if (o.M <= 16) return launch_dx<T, FMT, 16>(o, s);
  if (o.M <= 32) return launch_dx<T, FMT, 32>(o, s);
  if (o.M <= 64) return launch_dx<T, FMT, 64>(o, s);
  return o.M <= 128 ? launch_dx<T, FMT, 128>(o, s) : launch_dx<T, FMT, 256>(o, s);
}

}  // namespace

// Measured whole backward passes (us), r = 16, against the decoded copy of W and the
// pair GEMM: 256 rows, 4096 -> 4096 28.3 against 54.3, 4096 -> 32000 92 against 164;
// 1024 rows, 4096 -> 4096 (128 tiles of 256 x 128) 55 against 64; 1500 rows (192 tiles)
// 89.8 against 88.5.
bool mx_dx_few(int64_t M, int64_t K, int num_sms) {
  return M <= 256 || (M + 255) / 256 * ((K + 127) / 128) <= num_sms;
}

int mx_dx_launch(const MxDxOperands& o, int fmt, int dtype, cudaStream_t s) {
  if (dtype == LORA_BF16)
    return fmt == LORA_MXFP4 ? dispatch<__nv_bfloat16, LORA_MXFP4>(o, s) : dispatch<__nv_bfloat16, LORA_NVFP4>(o, s);
  return fmt == LORA_MXFP4 ? dispatch<__half, LORA_MXFP4>(o, s) : dispatch<__half, LORA_NVFP4>(o, s);
}

}  // namespace lora
