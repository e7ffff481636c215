// Epilogue of the kernels whose tile has 128 columns of the result as its TMEM lanes
// and tokens as its TMEM columns, the contraction cut over a cluster: the partial
// tiles meet in shared memory and are summed in rank order over DSMEM.
#pragma once

#include "mx_linear.h"

namespace lora {

struct MxTileOut {
  void* out;
  const void* bias;
  int64_t ldo;
  int M, N;
  float alpha, base_scale;  // out = alpha (base_scale acc + second acc) + bias
};

// Threads of the block: THREADS; warps FIRST .. FIRST + WARPS - 1 read TMEM (WARPS a
// multiple of 4), whose COLS columns warp 1 gives back.  part: NB x 128 fp32 over the drained stages.  second: TMEM column of the second
// accumulator, 0 for none.
template <typename T, int NB, int THREADS, int FIRST, int WARPS, int COLS>
LORA_DEVINL void mx_tile_out(const MxTileOut& args, float* part, uint32_t tmem, uint32_t second, uint64_t* acc_full,
                             volatile int* abort_flag, int* err, int splits, int rank, int n0, int t0) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // one result column a thread into [token][128]; then a warp sums and stores one
  // token's 128 columns at a time
  const int count = min(NB, args.M - t0);
  if (warp >= FIRST && warp < FIRST + WARPS && warp_wait(acc_full, 0, abort_flag, err, kDevErrTimeoutAccFull)) {
    tc_fence_after();
    const int quad = warp & 3;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t dst = smem_u32(part) + (quad * 32 + lane) * 4;
#pragma unroll 1
    for (int c = ((warp - FIRST) >> 2) * 16; c < count; c += 4 * WARPS) {
      uint32_t u[16], l[16];
      tmem_ld_32x32b_x16(t_row + c, u);
      if (second) tmem_ld_32x32b_x16(t_row + second + c, l);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = __uint_as_float(u[e]) * args.base_scale;
        if (second) v += __uint_as_float(l[e]);
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + (c + e) * 512), "f"(v) : "memory");
      }
    }
  }
  if (splits > 1) {  // every rank's partial tile is in its shared memory
    cluster_sync_free_tmem(tmem, COLS, warp, warp >= FIRST && warp < FIRST + WARPS, WARPS);
  } else {
    tc_fence_before();
    __syncthreads();
  }
  {
    const int b = count * rank / splits, e = count * (rank + 1) / splits;
    const int n = n0 + 4 * lane;
    const bool vec = args.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(args.out) & 7) == 0 && n + 4 <= args.N;
    const T* bias = static_cast<const T*>(args.bias);
    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (bias != nullptr && n + i < args.N) add[i] = to_f32(bias[n + i]);
    const uint32_t src = smem_u32(part) + lane * 16;
    for (int t = b + warp; t < e; t += THREADS / 32) {
      float4 v;
      if (splits == 1) {
        const uint4 u = lds128(src + t * 512);
        v = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
      } else {
        float4 p[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < splits) p[q] = ld_dsmem_f4(mapa_shared(src + t * 512, q));
        v = p[0];
#pragma unroll
        for (int q = 1; q < 8; ++q)
          if (q < splits) v.x += p[q].x, v.y += p[q].y, v.z += p[q].z, v.w += p[q].w;
      }
      v.x = v.x * args.alpha + add[0], v.y = v.y * args.alpha + add[1];
      v.z = v.z * args.alpha + add[2], v.w = v.w * args.alpha + add[3];
      T* o = static_cast<T*>(args.out) + static_cast<int64_t>(t0 + t) * args.ldo + n;
      if (vec) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
      } else {
        if (n < args.N) o[0] = from_f32<T>(v.x);
        if (n + 1 < args.N) o[1] = from_f32<T>(v.y);
        if (n + 2 < args.N) o[2] = from_f32<T>(v.z);
        if (n + 3 < args.N) o[3] = from_f32<T>(v.w);
      }
    }
  }
  if (splits > 1) {
    cluster_sync_all();  // no CTA leaves while another reads its partial tile
  } else if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

}  // namespace lora
