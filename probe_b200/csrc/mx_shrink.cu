// Rank shrink  z = s v A^T  with, in the same pass over v, v's quantisation to a
// 4-bit format.
//
//   z [M, 2 r16] = [hi | lo], hi = round(z), lo = round(z - hi)
//
// (without a format, of fp16 operands: bf16 parts [hi | mid | lo], whose range is fp32's)
//
// A is [R, K] (rows along K, an adapter's down projection) or, for gradients,
// [K, R] (an up projection, multiplied from the other side); tcgen05 takes either
// as the N operand, K-major or MN-major, with 128 tokens as M.  While the MMAs of
// a 128 x 128 tile of v run (x 64 for ranks above 64, whose adapter tile is larger),
// eight warps quantise the same tile from shared memory (two lanes a row: conflict-free
// with the 128-byte swizzle, whole 32-byte sectors of codes out).  A second group of
// eight takes every other tile; a third made it slower (4095 x 5120 mxfp4, r = 16: 26.7
// against 25.9 us; r = 224 of 32760 tokens, nvfp4: 219 against 176).  Up to 64 tokens
// there are four groups of four (whole calls of 1, 16 and 64 tokens, N = 4096, both formats,
// r = 16, 96, 224: 4096 columns 3 to 9 % faster, 13824 columns 5 to 20 %; one token of 13824,
// nvfp4, r = 16, 21.7 to 17.4 us).
//
// Bound: the floor is HBM (v once, codes out); what is measured is the ALU pipe of the
// quantisation -- 4095 x 5120 mxfp4 with r = 16, 53 MB, takes 18 to 25 us, issue slots
// 0.44 and the ALU pipe 0.43 used on average, start and end included -- and for large
// ranks the adapter's tile through L2 into shared memory.
// Work split: the (token block, chunk of columns) pairs in one sequence, cut into
// equal runs, one per SM, so that any M fills the machine; a token block cut by a
// run boundary leaves fp32 partials that its last contributor (a ticket) adds in
// run order, so the result does not depend on timing.  Where token blocks are no more
// than SMs (18944 tokens), a cluster of 8, 4, 2 or 1 CTAs takes each block instead and
// its partial sums meet in shared memory: no ticket, fence and reload, whose latencies
// would be half of a short call.
#include <mutex>

#include "mx_shrink.h"

namespace lora {
namespace {

constexpr int kShWorkers = 16;  // two groups of eight (or four of four), taking stages in turn
constexpr int kShThreads = 64 + 32 * kShWorkers;
constexpr int kShBoxBytes = 128 * 128;  // 128 tokens x 64 columns
constexpr int kShSmemMax = 224 * 1024;
constexpr int kNoFormat = -1;

struct ShMaps {
  CUtensorMap v, a;
};

struct ShArgs {
  void* z;
  uint8_t *codes, *scales;
  float* part;   // [2 runs' ends][128][r16] per CTA
  int* tickets;  // kShWorkers per CTA, zero between calls
  int* err;
  int64_t M, K, Kp, ldz;
  int chunks_total;
  int kc, r16, a_boxes, a_box_bytes, stages, stage_bytes, gb;
  int groups;   // of r16 columns of a three-part result
  int cluster;  // CTAs of a token block's cluster; 0: runs
  int group_shift;  // log2 of the warps of a group, which takes 16 rows a warp
  float scale;
  MxGlobal gl;
};

// First chunk of a run (chunks x runs fit 31 bits).
LORA_DEVINL int sh_start(const ShArgs& a, int cta) {
  return static_cast<int>(static_cast<uint32_t>(a.chunks_total) * static_cast<uint32_t>(cta) / gridDim.x);
}

// hi/lo pair of 16 values to a row of z.
template <typename T>
LORA_DEVINL void sh_store_pair(T* z, int r16, const float* v) {
  uint32_t h[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    const float2 f = unpack2<T>(h[i]);
    l[i] = pack2<T>(v[2 * i] - f.x, v[2 * i + 1] - f.y);
  }
  uint4* d = reinterpret_cast<uint4*>(z);
  d[0] = make_uint4(h[0], h[1], h[2], h[3]);
  d[1] = make_uint4(h[4], h[5], h[6], h[7]);
  d = reinterpret_cast<uint4*>(z + r16);
  d[0] = make_uint4(l[0], l[1], l[2], l[3]);
  d[1] = make_uint4(l[4], l[5], l[6], l[7]);
}

// N values as bf16 parts, v = hi + mid + lo to 24 bits, `groups` groups of columns.
template <int N>
LORA_DEVINL void sh_store_three(uint16_t* z, int r16, int groups, const float* v) {
  using B = __nv_bfloat16;
  uint32_t p[3][N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float2 rest = make_float2(v[2 * i], v[2 * i + 1]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      p[k][i] = pack2<B>(rest.x, rest.y);
      const float2 f = unpack2<B>(p[k][i]);
      rest.x -= f.x, rest.y -= f.y;
    }
  }
#pragma unroll
  for (int g = 0; g < 5; ++g) {
    if (g >= groups) break;
    const uint32_t* w = p[g % 3];
    if constexpr (N == 4) {
      *reinterpret_cast<uint2*>(z + g * r16) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 8; ++i)
        reinterpret_cast<uint4*>(z + g * r16)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
}

template <typename T, int FMT, bool AMN, int KB>
__global__ void __launch_bounds__(kShThreads, 1)
    mx_shrink_kernel(const __grid_constant__ ShMaps maps, const ShArgs args) {
  // the gradient g of fp16 activations, which leaves fp16's range on either side
  constexpr bool kThree = FMT == kNoFormat && std::is_same<T, __half>::value;
  auto store16 = [&](T* z, const float* v) {
    if constexpr (kThree)
      sh_store_three<16>(reinterpret_cast<uint16_t*>(z), args.r16, args.groups, v);
    else
      sh_store_pair<T>(z, args.r16, v);
  };
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + args.stages * args.stage_bytes);
  uint64_t* empty = full + 8;
  uint64_t* acc_full = empty + 8;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* recip = reinterpret_cast<float*>(tmem_slot + 4);  // 128 entries (nvfp4)
  const uint32_t csum = smem_u32(smem);  // cluster mode: [128][r16] partial sums, over the drained stages

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int crank = args.cluster ? static_cast<int>(cluster_ctarank()) : 0;
  const int cblock = args.cluster ? static_cast<int>(blockIdx.x) / args.cluster * args.kc : 0;  // its first chunk
  const int c_begin = args.cluster ? cblock + args.kc * crank / args.cluster : sh_start(args, blockIdx.x);
  const int c_end = args.cluster ? cblock + args.kc * (crank + 1) / args.cluster : sh_start(args, blockIdx.x + 1);
  const uint32_t need = 2 * args.r16;
  const uint32_t tmem_cols = need <= 32 ? 32u : need <= 64 ? 64u : need <= 128 ? 128u : need <= 256 ? 256u : 512u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], FMT == kNoFormat ? 1 : 1 + (1 << args.group_shift));  // the MMAs, a group of workers
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kShWorkers);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.v);
    tma_prefetch_desc(&maps.a);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  if constexpr (FMT == LORA_NVFP4) {
    if (threadIdx.x >= 64 && threadIdx.x < 192)
      recip[threadIdx.x - 64] = mx_recip_entry(static_cast<int>(threadIdx.x) - 64, args.gl.g);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();  // v, and the buffers that the kernels before may still read
  pdl_launch_dependents();  // after the wait: a dependent may take what came before this kernel as done

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      const uint32_t bytes = KB * kShBoxBytes + args.a_boxes * args.a_box_bytes;
      int tb = c_begin / args.kc, kc = c_begin - tb * args.kc;
      for (int c = c_begin; c < c_end; ++c) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, args.err, kDevErrTimeoutEmpty)) break;
        uint8_t* base = smem + stage * args.stage_bytes;
        mbar_arrive_expect_tx(&full[stage], bytes);
        for (int b = 0; b < KB; ++b)
          tma_load_2d(&maps.v, base + b * kShBoxBytes, &full[stage], (kc * KB + b) * 64, tb * 128);
        for (int b = 0; b < args.a_boxes; ++b)
          tma_load_2d(&maps.a, base + KB * kShBoxBytes + b * args.a_box_bytes, &full[stage],
                      AMN ? b * 64 : (kc * KB + b) * 64, AMN ? kc * KB * 64 : 0);
        if (++kc == args.kc) {
          kc = 0;
          ++tb;
        }
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // the whole warp walks the chunks (uniform descriptors); one lane issues
    const uint32_t idesc = (umma_idesc_f16(128, 16, std::is_same<T, __nv_bfloat16>::value ? 1 : 0) & ~(0x3fu << 17)) |
                           (static_cast<uint32_t>(args.r16 >> 3) << 17) | (AMN ? 1u << 16 : 0u);
    const uint64_t x0 = umma_desc_sw128(smem_u32(smem));
    const uint64_t a0 = AMN ? mx_desc_mn(smem_u32(smem) + KB * kShBoxBytes, args.a_box_bytes)
                            : umma_desc_sw128(smem_u32(smem) + KB * kShBoxBytes);
    int stage = 0, seg = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int c = c_begin; ok && c < c_end; ++seg) {
      const int seg_end = min(c_end, (c / args.kc + 1) * args.kc);
      if (!warp_wait(&acc_empty[seg & 1], ((seg >> 1) & 1) ^ 1, abort_flag, args.err, kDevErrTimeoutAccEmpty))
        break;
      tc_fence_after();
      const uint32_t d = tmem + (seg & 1) * args.r16;
      for (bool first = true; c < seg_end; ++c, first = false) {
        if (!warp_wait(&full[stage], phase, abort_flag, args.err, kDevErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at = static_cast<uint32_t>((stage * args.stage_bytes) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4 * KB; ++k) {
            const uint64_t xd = x0 + (at + static_cast<uint32_t>((k >> 2) * (kShBoxBytes >> 4) + 2 * (k & 3)));
            const uint64_t ad =
                a0 + (at + (AMN ? static_cast<uint32_t>(k * (2048 >> 4))
                                : static_cast<uint32_t>((k >> 2) * (args.a_box_bytes >> 4) + 2 * (k & 3))));
            tc_mma_f16(d, xd, ad, idesc, (!first || k > 0) ? 1u : 0u);
          }
          tc_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok && elect_one()) tc_commit(&acc_full[seg & 1]);
      __syncwarp();
    }
  } else {
    const int w = warp - 2, quad = warp & 3, part = w >> 2;
    const uint32_t recip_addr = smem_u32(recip), smem_addr = smem_u32(smem);
    int stage = 0, seg = 0, turn = w >> args.group_shift;
    uint32_t phase = 0;
    bool ok = true;
    for (int c = c_begin; ok && c < c_end; ++seg) {
      const int tb = c / args.kc;
      const int seg_begin = c, seg_end = min(c_end, (tb + 1) * args.kc);
      if constexpr (FMT != kNoFormat) {
        // rows 16 (w % group) .. + 15 of the block, 32 columns a lane; rows that no warp takes
        // are beyond M, where codes read as zeros and no result is stored
        const int r = 16 * (w & ((1 << args.group_shift) - 1)) + (lane >> 1);
        const int64_t row = static_cast<int64_t>(tb) * 128 + r;
        uint8_t* sc = args.scales + static_cast<int64_t>(tb) * args.gb * 512 + (r & 31) * 16 + (r >> 5) * 4;
        for (; c < seg_end; ++c) {
          const int kc = c - tb * args.kc;
          if (turn-- == 0) {
            turn = (kShWorkers >> args.group_shift) - 1;
            if (!warp_wait(&full[stage], phase, abort_flag, args.err, kDevErrTimeoutFull)) {
              ok = false;
              break;
            }
            const uint32_t xs = smem_addr + stage * args.stage_bytes + r * 128;
            uint32_t bytes = 0;  // scale bytes of this lane, in block order
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              uint32_t x[16];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint4 q = lds128(xs + b * kShBoxBytes + ((((lane & 1) * 4 + i) ^ (r & 7)) << 4));
                x[4 * i] = q.x, x[4 * i + 1] = q.y, x[4 * i + 2] = q.z, x[4 * i + 3] = q.w;
              }
              if (b == KB - 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
              }
              const int64_t col = static_cast<int64_t>(kc * KB + b) * 64 + (lane & 1) * 32;
              uint32_t cd[4];
              const uint32_t t0 = mx_amax16(x), t1 = mx_amax16(x + 8);
              if constexpr (FMT == LORA_NVFP4) {
                const MxScale<T, FMT> s0(t0, args.gl, recip_addr), s1(t1, args.gl, recip_addr);
                mx_codes16<T, FMT>(x, s0, cd);
                mx_codes16<T, FMT>(x + 8, s1, cd + 2);
                bytes |= (s0.byte | (s1.byte << 8)) << (16 * b);
              } else {
                const MxScale<T, FMT> s(max(t0, t1), args.gl, recip_addr);
                mx_codes16<T, FMT>(x, s, cd);
                mx_codes16<T, FMT>(x + 8, s, cd + 2);
                bytes |= s.byte << (16 * b);
              }
              if (row < args.M && col < args.Kp)
                *reinterpret_cast<uint4*>(args.codes + row * (args.Kp >> 1) + (col >> 1)) =
                    make_uint4(cd[0], cd[1], cd[2], cd[3]);
            }
            const uint32_t other = __shfl_xor_sync(0xffffffffu, bytes, 1);
            if constexpr (FMT == LORA_NVFP4) {
              // blocks 0, 1 of 64 columns (a chunk of scales) are the even lane's, 2, 3
              // the odd one's; the even lane stores the first chunk, the odd one a second
              const uint32_t word =
                  (lane & 1) ? (other >> 16) | (bytes & 0xffff0000u) : (bytes & 0xffffu) | (other << 16);
              const int chunk = KB * kc + (lane & 1);
              if ((lane & 1) < KB && chunk < args.gb) *reinterpret_cast<uint32_t*>(sc + chunk * 512) = word;
            } else if ((lane & 1) == 0) {
              const uint32_t word = bytes | (other << 8);
              if constexpr (KB == 2)
                *reinterpret_cast<uint32_t*>(sc + kc * 512) = word;
              else
                *reinterpret_cast<uint16_t*>(sc + (kc >> 1) * 512 + (kc & 1) * 2) = static_cast<uint16_t>(word);
            }
          }
          if (++stage == args.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
      }
      c = seg_end;
      if (args.cluster) break;  // below
      // ---- the block's sum (or this run's part of it); a warp takes its 32 rows and
      // every fourth group of 16 columns
      if (!warp_wait(&acc_full[seg & 1], (seg >> 1) & 1, abort_flag, args.err, kDevErrTimeoutAccFull)) break;
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(tb) * 128 + quad * 32 + lane;
      const bool whole = seg_begin == tb * args.kc && seg_end == (tb + 1) * args.kc;
      T* zrow = static_cast<T*>(args.z) + row * args.ldz;
      float* slot = args.part + (static_cast<int64_t>(blockIdx.x) * 2 + (seg_begin == c_begin ? 0 : 1)) * 128 * args.r16 +
                    (quad * 32 + lane) * args.r16;
      for (int j = part * 16; j < args.r16; j += 64) {
        uint32_t u[16];
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(quad * 32) << 16) + (seg & 1) * args.r16 + j, u);
        tmem_wait_ld();
        if (row >= args.M) continue;
        if (whole) {
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(u[e]) * args.scale;
          store16(zrow + j, v);
        } else {
          st_global_v8(slot + j, u);
          st_global_v8(slot + j + 8, u + 8);
        }
      }
      __syncwarp();
      tc_fence_before();
      if (lane == 0) mbar_arrive(&acc_empty[seg & 1]);
      if (!whole && part * 16 < args.r16) {
        // first and last run with a chunk of this block
        const int first_chunk = tb * args.kc, end_chunk = first_chunk + args.kc;
        int j0 = static_cast<int>(static_cast<int64_t>(first_chunk) * gridDim.x / args.chunks_total);
        while (sh_start(args, j0 + 1) <= first_chunk) ++j0;
        while (sh_start(args, j0) > first_chunk) --j0;
        int j1 = static_cast<int>(static_cast<int64_t>(end_chunk - 1) * gridDim.x / args.chunks_total);
        while (sh_start(args, j1 + 1) < end_chunk) ++j1;
        while (sh_start(args, j1) >= end_chunk) --j1;
        // each warp has a ticket of its own for its rows and columns; j0 is the first
        // run of no other cut block
        __threadfence();
        __syncwarp();
        int last = 0;
        if (lane == 0) {
          int* ticket = args.tickets + j0 * kShWorkers + w;
          last = atomicAdd(ticket, 1) == j1 - j0;
          if (last) *ticket = 0;
        }
        if (__shfl_sync(0xffffffffu, last, 0)) {
          __threadfence();
          // run j0's part lies in its last slot unless the run starts with this block;
          // every later run starts inside it
          const int slot0 = sh_start(args, j0) >= first_chunk ? 0 : 1;
          const float* base = args.part + (quad * 32 + lane) * args.r16;
          const int64_t pitch = static_cast<int64_t>(2 * 128) * args.r16;
          if (row < args.M)
            for (int j = part * 16; j < args.r16; j += 64) {
              float v[16];
#pragma unroll
              for (int h = 0; h < 2; ++h) {  // 8 columns at a time, four runs' loads in flight
                float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int i = j0; i <= j1; i += 4) {
                  float4 q[4][2];
#pragma unroll
                  for (int n = 0; n < 4; ++n)
                    if (i + n <= j1) {
                      const float4* p = reinterpret_cast<const float4*>(
                          base + (i + n) * pitch + (i + n == j0 && slot0 ? 128 * args.r16 : 0) + j + 8 * h);
                      q[n][0] = __ldcg(p);
                      q[n][1] = __ldcg(p + 1);
                    }
#pragma unroll
                  for (int n = 0; n < 4; ++n)
                    if (i + n <= j1) {
                      acc[0] += q[n][0].x, acc[1] += q[n][0].y, acc[2] += q[n][0].z, acc[3] += q[n][0].w;
                      acc[4] += q[n][1].x, acc[5] += q[n][1].y, acc[6] += q[n][1].z, acc[7] += q[n][1].w;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * h + e] = acc[e] * args.scale;
              }
              store16(zrow + j, v);
            }
        }
      }
    }
    if (args.cluster) {
      // every worker has read its tiles, every MMA has: the sums may take their place
      ok = warp_wait(&acc_full[0], 0, abort_flag, args.err, kDevErrTimeoutAccFull);
      named_bar_sync(1, 32 * kShWorkers);
      tc_fence_after();
      for (int j = part * 16; ok && j < args.r16; j += 64) {
        uint32_t u[16];
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(quad * 32) << 16) + j, u);
        tmem_wait_ld();
        const uint32_t dst = csum + ((quad * 32 + lane) * args.r16 + j) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sts128(dst + 16 * e, make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]));
      }
    }
  }
  if (args.cluster) {
    // every CTA's partial sums are in its shared memory
    cluster_sync_free_tmem(tmem, tmem_cols, warp, warp >= 2, kShWorkers);
    // rows are dealt to the ranks, groups of four columns to the threads
    const int per = 128 / args.cluster, quads = args.r16 / 4;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / args.cluster) * 128 + crank * per;
    for (int i = threadIdx.x; i < per * quads; i += kShThreads) {
      const int r = i / quads, j = (i - r * quads) * 4;
      if (row0 + r >= args.M) break;
      const uint32_t src = csum + ((crank * per + r) * args.r16 + j) * 4;
      float4 p[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < args.cluster) p[q] = ld_dsmem_f4(mapa_shared(src, q));
      float4 v = p[0];
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < args.cluster) v.x += p[q].x, v.y += p[q].y, v.z += p[q].z, v.w += p[q].w;
      v.x *= args.scale, v.y *= args.scale, v.z *= args.scale, v.w *= args.scale;
      T* z = static_cast<T*>(args.z) + (row0 + r) * args.ldz + j;
      if constexpr (kThree) {
        const float f[4] = {v.x, v.y, v.z, v.w};
        sh_store_three<4>(reinterpret_cast<uint16_t*>(z), args.r16, args.groups, f);
        continue;
      }
      const uint2 h = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
      const float2 h0 = unpack2<T>(h.x), h1 = unpack2<T>(h.y);
      *reinterpret_cast<uint2*>(z) = h;
      *reinterpret_cast<uint2*>(z + args.r16) =
          make_uint2(pack2<T>(v.x - h0.x, v.y - h0.y), pack2<T>(v.z - h1.x, v.w - h1.y));
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
  } else {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, tmem_cols);
    }
  }
}

// 64-column boxes a chunk: the adapter's part of a stage grows with the rank.
int shrink_boxes(int64_t R) { return R > 64 ? 1 : 2; }

// Runs: one per SM, but no shorter than two chunks.
int shrink_ctas(int64_t M, int64_t K, int64_t R) {
  const int dev = current_device();
  const int sms = dev >= 0 ? device_info(dev).num_sms : 148;
  const int64_t total = (M + 127) / 128 * ((K + 64 * shrink_boxes(R) - 1) / (64 * shrink_boxes(R)));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms, total / 2)));
}

// CTAs of a token block's cluster where that fills no more than the machine: a
// power of two up to 8, each with a chunk or more.  0: equal runs over all blocks.
int shrink_cluster(int64_t M, int64_t K, int64_t R) {
  const int dev = current_device();
  const int sms = dev >= 0 ? device_info(dev).num_sms : 148;
  const int64_t blocks = (M + 127) / 128, kc = (K + 64 * shrink_boxes(R) - 1) / (64 * shrink_boxes(R));
  int c = 8;
  while (c > 1 && (c > kc || blocks * c > sms)) c /= 2;
  if (blocks * c > sms) return 0;
  return c;
}

template <typename T, int FMT, bool AMN, int KB>
int launch_shrink(const MxShrinkOperands& o, cudaStream_t stream) {
  const int dev = current_device();
  if (dev < 0) return LORA_ERR_DEVICE;
  const DeviceInfo& info = device_info(dev);
  ShMaps maps;
  ShArgs a;
  a.r16 = static_cast<int>((o.R + 15) / 16 * 16);
  a.a_boxes = AMN ? (a.r16 + 63) / 64 : KB;
  a.a_box_bytes = AMN ? KB * 64 * 128 : a.r16 * 128;
  if (!mx_encode_map(&maps.v, o.v, 2, o.K, o.M, o.ldv * 2, 64, 128, true)) return LORA_ERR_CUDA;
  if (AMN ? !mx_encode_map(&maps.a, o.a, 2, o.R, o.K, o.lda * 2, 64, KB * 64, true)
          : !mx_encode_map(&maps.a, o.a, 2, o.K, o.R, o.lda * 2, 64, a.r16, true))
    return LORA_ERR_CUDA;
  a.z = o.z;
  a.codes = static_cast<uint8_t*>(o.codes);
  a.scales = static_cast<uint8_t*>(o.scales);
  a.tickets = static_cast<int*>(o.tickets);
  a.part = static_cast<float*>(o.part);
  a.err = info.err_word;
  a.M = o.M;
  a.K = o.K;
  a.Kp = mx_padded_k(o.K);
  a.ldz = o.ldz;
  a.groups = o.groups;
  a.kc = static_cast<int>((o.K + 64 * KB - 1) / (64 * KB));
  a.chunks_total = static_cast<int>((o.M + 127) / 128 * a.kc);
  a.stage_bytes = KB * kShBoxBytes + a.a_boxes * a.a_box_bytes;
  a.gb = FMT == kNoFormat ? 0 : static_cast<int>(mx_scale_chunks(o.K, FMT == kNoFormat ? 0 : FMT));
  a.scale = o.scale;
  a.gl = mx_global(o.global_scale);
  constexpr int kFixed = 1024 + 1024;  // alignment, barriers and reciprocals
  a.cluster = shrink_cluster(o.M, o.K, o.R);
  a.stages = std::min(8, (kShSmemMax - kFixed) / a.stage_bytes);
  a.group_shift = 3;
  if (FMT != kNoFormat) {
    // A stage always goes to the same group -- the groups divide the ring -- so that a
    // warp which waits for a stage's next tile has seen its last one: a barrier's parity
    // says no more than that.
    a.stages &= ~1;
    if (o.M <= 64) {
      a.group_shift = 2;
      a.stages &= ~3;
    }
  }
  auto kernel = mx_shrink_kernel<T, FMT, AMN, KB>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShSmemMax);
  });
  if (attr_err[dev] != cudaSuccess) return LORA_ERR_CUDA;
  size_t smem = static_cast<size_t>(a.stages) * a.stage_bytes + kFixed;
  // All of tensor memory: no CTA that takes some may share the SM.  A cluster's CTA that
  // holds it while its peer waits for another cluster's, and the other way round on another
  // SM, would wait for good (kernels of two streams).
  if (2 * a.r16 > 256) smem = kShSmemMax;
  if (a.cluster && a.stages * a.stage_bytes < 128 * a.r16 * 4) return LORA_ERR_UNSUPPORTED;  // never: 167 KB and more
  const int64_t ctas = a.cluster ? (o.M + 127) / 128 * a.cluster : shrink_ctas(o.M, o.K, o.R);
  return mx_launch(kernel, dim3(static_cast<unsigned>(ctas)), kShThreads, smem, stream, a.cluster, maps, a);
}

template <typename T, int KB>
int dispatch(const MxShrinkOperands& o, int fmt, cudaStream_t s) {
  if (fmt == kNoFormat)
    return o.a_mn ? launch_shrink<T, kNoFormat, true, KB>(o, s) : launch_shrink<T, kNoFormat, false, KB>(o, s);
  if (fmt == LORA_MXFP4) return launch_shrink<T, LORA_MXFP4, false, KB>(o, s);
  return launch_shrink<T, LORA_NVFP4, false, KB>(o, s);
}

}  // namespace

size_t mx_shrink_part_bytes(int64_t M, int64_t K, int64_t R) {
  return static_cast<size_t>(shrink_ctas(M, K, R)) * 2 * 128 * ((R + 15) / 16 * 16) * sizeof(float);
}

bool mx_shrink_serves(const void* v, int64_t ldv, const void* a, int64_t lda) {
  return mx_aligned(v, 16) && ldv % 8 == 0 && mx_aligned(a, 16) && lda % 8 == 0;
}

int mx_shrink_launch(const MxShrinkOperands& o, int fmt, int dtype, cudaStream_t stream) {
  if (shrink_boxes(o.R) == 1)
    return dtype == LORA_BF16 ? dispatch<__nv_bfloat16, 1>(o, fmt, stream) : dispatch<__half, 1>(o, fmt, stream);
  return dtype == LORA_BF16 ? dispatch<__nv_bfloat16, 2>(o, fmt, stream) : dispatch<__half, 2>(o, fmt, stream);
}

}  // namespace lora
