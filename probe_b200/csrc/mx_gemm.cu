// 4-bit block-scaled GEMM with the LoRA expand folded in.
//
//   out[M,N] = alpha ( 2^-d sum_k xq[m,k] sx[m,k/b] wq[n,k] sw[n,k/b]
//                      + sum_j (zh[m,j] + zl[m,j]) B[n,j] ) + bias[n]
//
// xq, wq: E2M1 codes, sx, sw: their block scales (mx.cuh), multiplied inside
// tcgen05.mma.kind::mxf4nvf4 as the products are formed.  z = [zh | zl] is the
// 16-bit hi/lo pair of the adapter's shrink; its products with B are kind::f16
// MMAs into the same fp32 accumulator, after the base ones.  nvfp4 has
// alpha 2^-d = the product of the two tensor scales with alpha in [1, 2): the
// power of two is taken off the accumulator by the first tail MMA (scale-input-d,
// exact, at most 2^-15; beyond that a stage of zeros takes off the first 2^-15),
// so z stays within the range of fp16.
//
// Bound: the tensor pipe (K = 64 steps of M 256 x N 256 a pair) and, with it,
// the operand intake of each SM: a 256-deep stage brings 32 KB of codes and 3
// to 6 KB of scales for 4 MMAs, the byte ratio of a 16-bit GEMM with 256 x 256
// tiles.  Layout: a cluster of two CTAs per 256 x 256 tile, persistent; warp 0
// TMA (codes in 128-byte swizzled rows, scale chunks as they are stored), warp
// 1 of the leader copies the stage's scales to TMEM (tcgen05.cp, each CTA from
// its own shared memory) and issues the MMAs, warps 2..9 the epilogue, warp 10 the
// scales' loads.
// TMEM holds a buffer of scales per pipeline stage, so that a stage's full barrier
// already says that its scale buffer is free: the MMA warp has 512 cycles a stage
// and every further wait costs it 100 to 200.  Beside those 144 (mxfp4) or 240
// (nvfp4) columns two 256-column accumulators do not fit: they overlap in as many,
// the epilogue takes the shared columns to registers first and only that holds up
// the next tile's MMAs.  Measured: 4095 tokens, 5120 -> 13824, mxfp4, r = 16: 5.5 PFLOP/s;
// 32760 tokens, 5120 -> 5120, nvfp4, r = 224: 417 us.
#include <cudaTypedefs.h>

#include <cmath>
#include <mutex>

#include "mx_linear.h"

namespace lora {
namespace {

constexpr int kMxEpiWarps = 8;  // two of each TMEM lane quadrant, taking 16-column groups in turn
constexpr int kMxScaleWarp = 2 + kMxEpiWarps;  // loads the scales
constexpr int kMxGemmThreads = 64 + 32 * kMxEpiWarps + 32;

struct MxGemmArgs {
  void* out;
  const void* bias;
  int* err;
  int64_t ldo;
  int M, N;
  int num_kb;         // 256-deep base stages
  int last_k64;       // MMA steps of the last one
  int rank_kb;        // 64-deep tail stages of each z part (0: no adapter)
  int last_k16;       // MMA steps of the last of them
  int fused_tail;     // 1: [zh | zl] in one stage (up to rank 32)
  int zero_kb;        // 1: a tail stage of zeros comes first
  int chunks;         // scale chunks of a block of 128 rows
  int num_m_tiles, num_n_tiles, num_tiles, group_m;
  int dshift;         // 0..30
  float alpha;
};

template <int FMT>
struct MxSmem {
  static constexpr int kChunks = 256 / MxFormat<FMT>::kBlock / 4;  // scale chunks of 128 rows a stage
  static constexpr int kStages = FMT == LORA_MXFP4 ? 6 : 5;
  static constexpr int kOpBytes = 128 * 128;                       // codes (or z, B) of 128 rows
  static constexpr int kSfBytes = 3 * kChunks * 512;               // x rows, then the W rows of both CTAs
  static constexpr int kMainBytes = 2 * kOpBytes + kSfBytes;
  static constexpr int kSfOffset = kStages * 2 * kOpBytes;
  static constexpr int kBarOffset = kSfOffset + kStages * kSfBytes;
  static constexpr int kEpiOffset = kBarOffset + 256;                 // 32 rows x 16 columns an epilogue warp
  static constexpr int kBytes = kEpiOffset + kMxEpiWarps * 1024 + 1024;
  // TMEM columns
  static constexpr int kSfCols = 3 * kChunks * 4;
  static constexpr int kSfBase = 512 - kStages * kSfCols;
  static constexpr int kAcc1 = kSfBase - 256;  // accumulator 1; accumulator 0 starts at 0
  static constexpr int kOverlap = 256 - kAcc1;
  static_assert(kOverlap % 16 == 0 && kBytes <= 227 * 1024, "layout");
};

LORA_DEVINL void mx_cp_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D = A B^T + D 2^-S
template <int S>
LORA_DEVINL void mx_mma_f16_pair_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, %4;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "n"(S)
      : "memory");
}
LORA_DEVINL void mx_mma_f16_pair_shift(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int shift) {
  switch (shift) {
#define LORA_MX_CASE(S) \
  case S: mx_mma_f16_pair_scaled<S>(d, a, b, idesc); break;
    LORA_MX_CASE(1) LORA_MX_CASE(2) LORA_MX_CASE(3) LORA_MX_CASE(4) LORA_MX_CASE(5) LORA_MX_CASE(6) LORA_MX_CASE(7)
    LORA_MX_CASE(8) LORA_MX_CASE(9) LORA_MX_CASE(10) LORA_MX_CASE(11) LORA_MX_CASE(12) LORA_MX_CASE(13)
    LORA_MX_CASE(14) LORA_MX_CASE(15)
#undef LORA_MX_CASE
    default: tc_mma_f16_pair(d, a, b, idesc, 1u);
  }
}

// Block-scaled instruction descriptor: E2M1 operands, K-major, fp32 accumulator;
// the scale ids (the pair of bytes of a 32-bit scale word) are added per MMA.
template <int FMT>
__host__ __device__ constexpr uint32_t mx_idesc(int m, int n) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | ((FMT == LORA_MXFP4 ? 1u : 0u) << 23) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

LORA_DEVINL void mx_tile_coords(int tile, const MxGemmArgs& a, int& mt, int& nt) {
  const int group_size = a.group_m * a.num_n_tiles;
  const int group = tile / group_size;
  const int first_m = group * a.group_m;
  const int gm = min(a.num_m_tiles - first_m, a.group_m);
  const int in_group = tile - group * group_size;
  mt = first_m + in_group % gm;
  nt = in_group / gm;
}

struct MxMaps {
  CUtensorMap x, w, sx, sw, zh, zl, b;
};

// 16 columns of 32 rows, a row a lane: alpha, bias, rounding, then one 32-byte store
// or two of 16 bytes (align: the rows' alignment), or (ANY), for rows of any alignment
// and the last columns, 4-byte words through `stage` (1 KB of shared memory), eight lanes
// a row -- 16 two-byte stores a lane made such a call five times as long.
template <typename T, bool ANY>
LORA_DEVINL void mx_store16(const MxGemmArgs& args, int row0, int lane, int col0, int align, uint32_t stage,
                            const uint32_t* r) {
  if (col0 >= args.N || row0 >= args.M) return;
  const T* bias = static_cast<const T*>(args.bias);
  const int row = row0 + lane;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) * args.alpha;
  if (bias != nullptr) {
    if (col0 + 16 <= args.N && (reinterpret_cast<uintptr_t>(bias) & 15) == 0) {
      const uint4 b0 = __ldg(reinterpret_cast<const uint4*>(bias + col0));
      const uint4 b1 = __ldg(reinterpret_cast<const uint4*>(bias + col0 + 8));
      const uint32_t bw[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = unpack2<T>(bw[i]);
        v[2 * i] += f.x;
        v[2 * i + 1] += f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (col0 + i < args.N) v[i] += to_f32(bias[col0 + i]);
    }
  }
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  T* out = static_cast<T*>(args.out) + col0;
  if (align >= 16 && col0 + 16 <= args.N) {
    if (row >= args.M) return;
    T* dst = out + static_cast<int64_t>(row) * args.ldo;
    if (align == 32) {
      st_global_v8(dst, w);
    } else {
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    return;
  }
  if constexpr (!ANY) return;
  sts128(stage + lane * 32, make_uint4(w[0], w[1], w[2], w[3]));
  sts128(stage + lane * 32 + 16, make_uint4(w[4], w[5], w[6], w[7]));
  __syncwarp();
  // lane: word `lane % 8` of rows 4 i + lane / 8; where a row starts on an odd element
  // the words lie one element on, and the eighth lane stores the two left over
  const int n = min(16, args.N - col0), word = lane & 7;
  const uint32_t src = stage + (lane >> 3) * 32 + word * 4;
  uint32_t lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = lds32(src + i * 128);
    hi[i] = lds32(word < 7 ? src + i * 128 + 4 : src + i * 128 - 28);  // the next word; the eighth lane: the first
  }
  uint16_t* base = reinterpret_cast<uint16_t*>(out + static_cast<int64_t>(row0 + (lane >> 3)) * args.ldo);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint16_t* dst = base + static_cast<int64_t>(4 * i) * args.ldo;
    if (row0 + 4 * i + (lane >> 3) >= args.M) continue;
    if ((reinterpret_cast<uintptr_t>(dst) & 2) == 0) {
      if (2 * word + 1 < n)
        *reinterpret_cast<uint32_t*>(dst + 2 * word) = lo[i];
      else if (2 * word < n)
        dst[2 * word] = static_cast<uint16_t>(lo[i]);
    } else if (word < 7) {
      if (2 * word + 2 < n)
        *reinterpret_cast<uint32_t*>(dst + 2 * word + 1) = __funnelshift_r(lo[i], hi[i], 16);
      else if (2 * word + 1 < n)
        dst[2 * word + 1] = static_cast<uint16_t>(lo[i] >> 16);
    } else {
      if (n == 16) dst[15] = static_cast<uint16_t>(lo[i] >> 16);
      dst[0] = static_cast<uint16_t>(hi[i]);
    }
  }
  __syncwarp();
}

// ANY: rows that are not 16-byte aligned, or N no multiple of 16.
template <typename T, int FMT, bool ANY>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMxGemmThreads, 1)
    mx_gemm_pair_kernel(const __grid_constant__ MxMaps maps, const MxGemmArgs args) {
  using L = MxSmem<FMT>;
  constexpr uint32_t kIdesc = mx_idesc<FMT>(256, 256);
  constexpr uint32_t kIdescTail = umma_idesc_f16(256, 256, std::is_same<T, __nv_bfloat16>::value ? 1 : 0);
  constexpr uint16_t kBoth = 0x3;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sm_a = smem;
  uint8_t* sm_b = smem + L::kStages * L::kOpBytes;
  uint8_t* sm_sf = smem + L::kSfOffset;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
  uint64_t* empty = full + L::kStages;
  uint64_t* acc_full = empty + L::kStages;  // a tile's MMAs are complete
  uint64_t* acc_free = acc_full + 1;        // its shared columns are drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 2 * kMxEpiWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
    tma_prefetch_desc(&maps.sx);
    tma_prefetch_desc(&maps.sw);
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();  // the codes, scales and z of the kernels before
  pdl_launch_dependents();
  const int tail_kb = (args.fused_tail ? 1 : 2 * args.rank_kb) + args.zero_kb;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < args.num_tiles; tile += npairs) {
        int mt, nt;
        mx_tile_coords(tile, args, mt, nt);
        const int row_a = mt * 256 + static_cast<int>(rank) * 128;
        const int row_b = nt * 256 + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < args.num_kb + tail_kb; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
          uint8_t* a = sm_a + stage * L::kOpBytes;
          uint8_t* b = sm_b + stage * L::kOpBytes;
          if (kb < args.num_kb) {
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * L::kMainBytes);
            tma_load_2d_pair(&maps.x, a, bar, kb * 128, row_a);
            tma_load_2d_pair(&maps.w, b, bar, kb * 128, row_b);
          } else {
            if (leader) mbar_arrive_expect_tx(&full[stage], 4 * L::kOpBytes);
            // (the stage of zeros lies beyond the operands' columns)
            const int t = kb - args.num_kb - args.zero_kb;
            const bool lo = t >= args.rank_kb;
            const int c = (t < 0 ? args.rank_kb : lo ? t - args.rank_kb : t) * 64;
            tma_load_2d_pair(lo ? &maps.zl : &maps.zh, a, bar, c, row_a);
            tma_load_2d_pair(&maps.b, b, bar, c, row_b);
          }
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == kMxScaleWarp) {
    // Five loads a stage are more than one thread issues in the stage's 512 cycles of
    // MMAs (618 measured): the scales' two come from here.  Their bytes are part of
    // the stage's expected ones.
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < args.num_tiles; tile += npairs) {
        int mt, nt;
        mx_tile_coords(tile, args, mt, nt);
        for (int kb = 0; kb < args.num_kb + tail_kb; ++kb) {
          // (the tail's stages are waited for too: a phase further on would read as free)
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          if (kb < args.num_kb) {
            const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
            uint8_t* sf = sm_sf + stage * L::kSfBytes;
            tma_load_2d_pair(&maps.sx, sf, bar, 0,
                             (mt * 2 + static_cast<int>(rank)) * args.chunks + kb * L::kChunks);
            tma_load_3d_pair(&maps.sw, sf + L::kChunks * 512, bar, 0, kb * L::kChunks, nt * 2);
          }
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the stages, so that descriptors and addresses live in
    // uniform registers; one elected lane waits and issues.
    if (leader) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true, ready = false;
      const uint64_t ad0 = umma_desc_sw128(smem_u32(sm_a));
      const uint64_t bd0 = umma_desc_sw128(smem_u32(sm_b));
      const uint64_t sd0 = mx_desc_scales(smem_u32(sm_sf));
      for (int tile = pair; ok && tile < args.num_tiles; tile += npairs, ++local) {
        if (local > 0 &&
            !warp_wait(acc_free, (local - 1) & 1, abort_flag, args.err, kDevErrTimeoutAccEmpty))
          break;
        tc_fence_after();
        const uint32_t d = tmem + ((local & 1) ? L::kAcc1 : 0);
        for (int kb = -args.num_kb; kb < tail_kb; ++kb) {  // base stages below 0, then the tail's
          if (!ready && !warp_wait(&full[stage], phase, abort_flag, args.err, kDevErrTimeoutFull)) {
            ok = false;
            break;
          }
          if (kb == 0) {  // the tile's base MMAs finish before MMAs of the other kind start
            const int last = stage == 0 ? L::kStages - 1 : stage - 1;
            if (!warp_wait(&empty[last], stage == 0 ? phase ^ 1 : phase, abort_flag, args.err,
                           kDevErrTimeoutEmpty)) {
              ok = false;
              break;
            }
          }
          tc_fence_after();
          const uint64_t ad = ad0 + static_cast<uint32_t>(stage * (L::kOpBytes >> 4));
          const uint64_t bd = bd0 + static_cast<uint32_t>(stage * (L::kOpBytes >> 4));
          const uint64_t sd = sd0 + static_cast<uint32_t>(stage * (L::kSfBytes >> 4));
          const int next = stage + 1 == L::kStages ? 0 : stage + 1;
          const uint32_t next_phase = next == 0 ? phase ^ 1 : phase;
          // asked now, used after the MMAs are issued
          ready = mbar_try_wait(&full[next], next_phase);
          if (kb < 0) {
            const uint32_t sf = tmem + L::kSfBase + stage * L::kSfCols;
            const uint32_t sfb = sf + L::kChunks * 4;
            const int nk = kb == -1 ? args.last_k64 : 4;
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < L::kChunks; ++j) {
                mx_cp_scales_pair(sf + 4 * j, sd + static_cast<uint64_t>(32 * j));
                mx_cp_scales_pair(sfb + 8 * j, sd + static_cast<uint64_t>(32 * (L::kChunks + j)));
                mx_cp_scales_pair(sfb + 8 * j + 4, sd + static_cast<uint64_t>(32 * (2 * L::kChunks + j)));
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                constexpr bool kMx = FMT == LORA_MXFP4;
                const int j = kMx ? k >> 1 : k;
                const uint32_t id = kMx ? static_cast<uint32_t>(k & 1) * 2u : 0u;
                if (k < nk)
                  mx_mma<FMT, true>(d, ad + static_cast<uint64_t>(2 * k), bd + static_cast<uint64_t>(2 * k),
                                   kIdesc | (id << 4) | (id << 29), sf + 4 * j, sfb + 8 * j,
                                   (kb > -args.num_kb || k > 0) ? 1u : 0u);
              }
              tc_commit_pair(&empty[stage], kBoth);
            }
          } else {
            const int t = kb - args.zero_kb;
            const int c = t >= args.rank_kb ? t - args.rank_kb : t;
            const int nk = t < 0 ? 1 : c == args.rank_kb - 1 ? args.last_k16 << args.fused_tail : 4;
            const int shift = t < 0 ? 15 : t == 0 ? args.dshift - 15 * args.zero_kb : 0;
            // one stage of [zh | zl]: the lo part's steps meet the same columns of B
            const int wrap = args.fused_tail ? args.last_k16 : 4;
            if (elect_one()) {
              mx_mma_f16_pair_shift(d, ad, bd, kIdescTail, shift);
#pragma unroll
              for (int k = 1; k < 4; ++k)
                if (k < nk)
                  tc_mma_f16_pair(d, ad + static_cast<uint64_t>(2 * k),
                                  bd + static_cast<uint64_t>(2 * (k >= wrap ? k - wrap : k)), kIdescTail, 1u);
              tc_commit_pair(&empty[stage], kBoth);
            }
          }
          ready = __all_sync(0xffffffffu, ready);
          stage = next;
          phase = next_phase;
        }
        if (ok && elect_one()) tc_commit_pair(acc_full, kBoth);
        __syncwarp();
      }
    }
  } else {
    const int quad = warp & 3;
    const int part = (warp - 2) >> 2;  // takes the 16-column groups of this parity
    const uintptr_t at = reinterpret_cast<uintptr_t>(args.out) | static_cast<uintptr_t>(args.ldo * 2);
    const int align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 2;
    const uint32_t stage = smem_u32(smem) + L::kEpiOffset + (warp - 2) * 1024;
    constexpr int kFirst = (L::kOverlap / 16 + 1) / 2;  // most shared groups of one warp
    int local = 0;
    for (int tile = pair; tile < args.num_tiles; tile += npairs, ++local) {
      int mt, nt;
      mx_tile_coords(tile, args, mt, nt);
      if (!warp_wait(acc_full, local & 1, abort_flag, args.err, kDevErrTimeoutAccFull)) break;
      tc_fence_after();
      const int row = mt * 256 + static_cast<int>(rank) * 128 + quad * 32;
      const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + ((local & 1) ? L::kAcc1 : 0);
      // Groups in the order: columns shared with the other accumulator, then the
      // rest.  The shared ones go to registers first, and the next tile may start.
      const int first = (local & 1) ? 0 : L::kAcc1;
      {
        uint32_t r[kFirst][16];
#pragma unroll
        for (int q = 0; q < kFirst; ++q)
          if (2 * q + part < L::kOverlap / 16) tmem_ld_32x32b_x16(t_row + first + (2 * q + part) * 16, r[q]);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(acc_free), 0));
#pragma unroll
        for (int q = 0; q < kFirst; ++q)
          if (2 * q + part < L::kOverlap / 16)
            mx_store16<T, ANY>(args, row, lane, nt * 256 + first + (2 * q + part) * 16, align, stage, r[q]);
      }
#pragma unroll 1
      for (int g = (L::kOverlap / 16 - part + 1) / 2 * 2 + part; g < 16; g += 4) {
        uint32_t r[2][16];
        const int c0 = (first + g * 16) & 255, c1 = (first + g * 16 + 32) & 255;
        tmem_ld_32x32b_x16(t_row + c0, r[0]);
        if (g + 2 < 16) tmem_ld_32x32b_x16(t_row + c1, r[1]);
        tmem_wait_ld();
        mx_store16<T, ANY>(args, row, lane, nt * 256 + c0, align, stage, r[0]);
        if (g + 2 < 16) mx_store16<T, ANY>(args, row, lane, nt * 256 + c1, align, stage, r[1]);
      }
    }
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Scale chunks of two neighbouring blocks of 128 rows in one box: 128 words x
// `box_chunks` chunks x 2 row blocks.
bool encode_scale_pairs(CUtensorMap* map, const void* ptr, int64_t chunks, int64_t blocks, int box_chunks) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(chunks), static_cast<cuuint64_t>(blocks)};
  const cuuint64_t strides[2] = {512, static_cast<cuuint64_t>(chunks) * 512};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_chunks), 2};
  const cuuint32_t one[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(ptr), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int FMT, bool ANY>
int launch_pair(const MxLinearOperands& o, cudaStream_t stream) {
  using L = MxSmem<FMT>;
  const int dev = current_device();
  if (dev < 0) return LORA_ERR_DEVICE;
  const DeviceInfo& info = device_info(dev);
  MxMaps maps;
  MxGemmArgs a;
  const int64_t pitch = mx_code_pitch(o.K, FMT);
  a.chunks = static_cast<int>(mx_scale_chunks(o.K, FMT));
  if (!mx_encode_map(&maps.x, o.x_codes, 1, pitch, o.M, pitch, 128, 128, true) ||
      !mx_encode_map(&maps.w, o.w_codes, 1, pitch, o.N, pitch, 128, 128, true) ||
      !mx_encode_map(&maps.sx, o.x_scales, 4, 128, (o.M + 127) / 128 * a.chunks, 512, 128, L::kChunks, false) ||
      !encode_scale_pairs(&maps.sw, o.w_scales, a.chunks, (o.N + 127) / 128, L::kChunks))
    return LORA_ERR_CUDA;
  if (o.R > 0) {
    const char* z = static_cast<const char*>(o.z);
    a.fused_tail = o.z_lo * 2 <= 64 ? 1 : 0;
    if (!mx_encode_map(&maps.zh, z, 2, a.fused_tail ? 2 * o.z_lo : o.R, o.M, o.ldz * 2, 64, 128, true) ||
        !mx_encode_map(&maps.zl, z + o.z_lo * 2, 2, o.R, o.M, o.ldz * 2, 64, 128, true) ||
        !mx_encode_map(&maps.b, o.b, 2, o.R, o.N, o.ldb * 2, 64, 128, true))
      return LORA_ERR_CUDA;
  } else {
    a.fused_tail = 0;
    maps.zh = maps.zl = maps.b = maps.x;
  }
  a.out = o.out;
  a.bias = o.bias;
  a.err = info.err_word;
  a.ldo = o.ldo;
  a.M = static_cast<int>(o.M);
  a.N = static_cast<int>(o.N);
  const int64_t kp = mx_padded_k(o.K);
  a.num_kb = static_cast<int>((kp + 255) / 256);
  a.last_k64 = static_cast<int>((kp - (a.num_kb - 1) * 256ll + 63) / 64);
  a.rank_kb = static_cast<int>((o.R + 63) / 64);
  a.last_k16 = a.rank_kb > 0 ? static_cast<int>((o.R - (a.rank_kb - 1) * 64ll + 15) / 16) : 0;
  a.zero_kb = o.dshift > 15 ? 1 : 0;
  a.num_m_tiles = static_cast<int>((o.M + 255) / 256);
  a.num_n_tiles = static_cast<int>((o.N + 255) / 256);
  a.num_tiles = a.num_m_tiles * a.num_n_tiles;
  a.group_m = 8;
  a.dshift = o.dshift;
  a.alpha = o.alpha;
  auto kernel = mx_gemm_pair_kernel<T, FMT, ANY>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  static int capacity[64];
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    int clusters = 0;
    if (attr_err[dev] == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * info.num_sms);
      cfg.blockDim = dim3(kMxGemmThreads);
      cfg.dynamicSmemBytes = L::kBytes;
      if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        clusters = 0;
      }
    }
    capacity[dev] = clusters > 0 ? clusters : info.num_sms / 2;
  });
  if (attr_err[dev] != cudaSuccess) return LORA_ERR_CUDA;
  const int pairs = std::min(a.num_tiles, capacity[dev]);
  return mx_launch(kernel, dim3(2 * pairs), kMxGemmThreads, L::kBytes, stream, 0, maps, a);
}

}  // namespace

bool mx_encode_map(CUtensorMap* map, const void* ptr, int elem, int64_t inner, int64_t outer, int64_t pitch_bytes,
                   int box_inner, int box_outer, bool swizzle) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const CUtensorMapDataType type = elem == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT32;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch_bytes)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
  const cuuint32_t one[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int mx_gemm_launch(const MxLinearOperands& o, int fmt, int dtype, cudaStream_t stream) {
  const bool any = o.N % 16 != 0 || o.ldo % 8 != 0 || !mx_aligned(o.out, 16);
#define LORA_MXG(T, F) (any ? launch_pair<T, F, true>(o, stream) : launch_pair<T, F, false>(o, stream))
  if (dtype == LORA_BF16)
    return fmt == LORA_MXFP4 ? LORA_MXG(__nv_bfloat16, LORA_MXFP4) : LORA_MXG(__nv_bfloat16, LORA_NVFP4);
  return fmt == LORA_MXFP4 ? LORA_MXG(__half, LORA_MXFP4) : LORA_MXG(__half, LORA_NVFP4);
#undef LORA_MXG
}

}  // namespace lora
