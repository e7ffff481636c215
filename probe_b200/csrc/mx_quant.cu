// Quantisation to the microscaled formats and back.
//
// mxfp4 / mxfp8: e = max(floor(log2 amax) - top, -127) over a block of 32
// (top: the exponent of the largest code, 2 for E2M1 and 8 for E4M3), the scale
// byte is e + 127 and a code is x 2^-e rounded to nearest even, saturating.
// Every step before the rounding is exact.
// nvfp4: s = E4M3(amax / (6 g)) over a block of 16, a code is x / (s g) rounded
// to nearest even; both quotients are correctly rounded fp32.
// A block that holds an infinity or a NaN gets a NaN scale and zero codes: all
// its values read back as NaN, and so does every product with it.
//
// Bound: HBM (2 bytes read, 0.53 to 1.03 written an element).  A CTA takes 128
// rows x 128 columns, the extent of whole scale chunks: 8 threads a row with 16
// elements each, in four passes of 32 rows, two of them loaded ahead: 48 registers, so
// five CTAs an SM, whose 80 KB in flight cover the latency (all four ahead and four
// CTAs: 13824 x 5120 nvfp4 39.1 us, not 37.2; one ahead and six 39.6); the 512 scale
// bytes of a chunk go through shared memory and leave as 16-byte stores.  A thread's 32
// bytes are one access: as two 16-byte stores, half a sector each, decoding
// 32760 x 5120 mxfp8 took 93 us, not 77.
#include "mx.cuh"

namespace lora {
namespace {

constexpr int kMxTile = 128;
constexpr int kMxThreads = 256;
constexpr int kMxAhead = 2;  // passes of 32 rows loaded ahead

// Scale byte and codes of one thread's 16 elements.
template <typename T, int FMT>
LORA_DEVINL uint32_t mx_encode16(const uint32_t* w, const MxGlobal& gl, uint32_t recip, uint32_t* codes) {
  uint32_t top = mx_amax16(w);
  if constexpr (MxFormat<FMT>::kBlock == 32) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const MxScale<T, FMT> s(top, gl, recip);
  mx_codes16<T, FMT>(w, s, codes);
  return s.byte;
}

// ALIGN: of the rows, in bytes (32, 16, 2).
template <typename T, int FMT, int ALIGN>
__global__ void __launch_bounds__(kMxThreads, 5)
    mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes,
                       uint8_t* __restrict__ scales, int64_t M, int64_t K, int64_t Kp, int chunks, MxGlobal gl) {
  constexpr int kChunks = kMxTile / MxFormat<FMT>::kBlock / 4;  // scale chunks of this tile
  __shared__ alignas(16) uint8_t sc[kChunks * 512];
  const int seg = threadIdx.x & 7;   // 16-column segment of the tile
  const int sub = threadIdx.x >> 3;  // row within a pass
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kMxTile;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kMxTile + seg * 16;
  __shared__ float recip[FMT == LORA_NVFP4 ? 128 : 1];
  uint32_t w[kMxAhead][8];
  auto load = [&](int p) {
    uint32_t* v = w[p % kMxAhead];
    const int64_t row = row0 + 32 * p + sub;
    if (row < M) {
      const T* src = x + row * ldx + col;
      if (ALIGN == 32 && col + 16 <= K) {
        ldg_stream_v8(src, v);
      } else if (ALIGN == 16 && col + 16 <= K) {
        const uint4 a = ldg_stream(src), b = ldg_stream(src + 8);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        ldg16_any(x + row * ldx, col, K, v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0u;
    }
  };
#pragma unroll
  for (int p = 0; p < kMxAhead; ++p) load(p);
  if constexpr (FMT == LORA_NVFP4) {
    if (threadIdx.x < 128) recip[threadIdx.x] = mx_recip_entry(static_cast<int>(threadIdx.x), gl.g);
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = row0 + 32 * p + sub;
    uint32_t c[4];
    uint32_t byte = mx_encode16<T, FMT>(w[p % kMxAhead], gl, smem_u32(recip), c);
    if (p + kMxAhead < 4) load(p + kMxAhead);
    if (col >= Kp || row >= M) byte = 0;
    if (row < M && col < Kp) {
      if constexpr (MxFormat<FMT>::kBits == 4)
        *reinterpret_cast<uint2*>(codes + row * (Kp >> 1) + (col >> 1)) = make_uint2(c[0], c[1]);
      else
        *reinterpret_cast<uint4*>(codes + row * Kp + col) = make_uint4(c[0], c[1], c[2], c[3]);
    }
    if constexpr (MxFormat<FMT>::kBlock == 16)
      sc[(seg >> 2) * 512 + sub * 16 + p * 4 + (seg & 3)] = static_cast<uint8_t>(byte);
    else if ((seg & 1) == 0)
      sc[sub * 16 + p * 4 + (seg >> 1)] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
  if (threadIdx.x < kChunks * 32) {
    const int chunk = static_cast<int>(blockIdx.x) * kChunks + (threadIdx.x >> 5);
    if (chunk < chunks)
      reinterpret_cast<uint4*>(scales + (static_cast<int64_t>(blockIdx.y) * chunks + chunk) * 512)[threadIdx.x & 31] =
          reinterpret_cast<const uint4*>(sc)[threadIdx.x];
  }
}

// Values of one thread's 16 codes: (code x scale) x g, rounded once to T.
template <typename T, int FMT>
LORA_DEVINL void mx_decode16(const uint32_t* c, uint32_t byte, float g, uint32_t* out) {
  const float s = FMT == LORA_NVFP4 ? mx_e4m3(byte) : mx_e8m0(byte);
  uint32_t h[8];
  if constexpr (MxFormat<FMT>::kBits == 4) {
    mx_from_e2m1x8(c[0], h);
    mx_from_e2m1x8(c[1], h + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = mx_from_e4m3x2((c[i >> 1] >> (16 * (i & 1))) & 0xffffu);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 q = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    out[i] = pack2<T>(q.x * s * g, q.y * s * g);
  }
}

// A CTA decodes 128 x 128 values: straight to rows aligned to 16 or (vec) 32 bytes; to rows of any
// alignment, through shared memory, in 4-byte words; or transposed through shared
// memory (column c of the tensor becomes row c of out, Mw >= M values wide: zeros
// beyond M).
enum { kDqRows, kDqAnyRows, kDqTransposed };
template <typename T, int FMT, int MODE>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
                         int64_t ldo, int64_t M, int64_t Mw, int64_t K, int64_t Kp, int chunks, float g, bool vec) {
  constexpr bool TR = MODE == kDqTransposed;
  // Transposed: rows of sixteen 16-byte units, unit u of row r at u ^ f(r), f(r) =
  // 2 (r / 8 % 4) + r % 2, so that the eight rows an 8 x 8 matrix is gathered from
  // below lie in different banks.
  __shared__ alignas(128) uint16_t tile[MODE != kDqRows ? kMxTile * kMxTile : 8];
  const int seg = threadIdx.x & 7;
  const int sub = threadIdx.x >> 3;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kMxTile;
  const int64_t col0 = static_cast<int64_t>(blockIdx.x) * kMxTile;
  const int64_t col = col0 + seg * 16;
  const int block = static_cast<int>(col / MxFormat<FMT>::kBlock);
  const uint8_t* sc =
      scales + (static_cast<int64_t>(blockIdx.y) * chunks + (block >> 2)) * 512 + sub * 16 + (block & 3);
  uint32_t c[4][4], byte[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = row0 + 32 * p + sub;
    c[p][0] = c[p][1] = c[p][2] = c[p][3] = byte[p] = 0u;
    if (row < M && col < Kp) {
      byte[p] = sc[p * 4];
      if constexpr (MxFormat<FMT>::kBits == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(codes + row * (Kp >> 1) + (col >> 1));
        c[p][0] = v.x, c[p][1] = v.y;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(codes + row * Kp + col);
        c[p][0] = v.x, c[p][1] = v.y, c[p][2] = v.z, c[p][3] = v.w;
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = row0 + 32 * p + sub;
    uint32_t o[8];
    mx_decode16<T, FMT>(c[p], byte[p], g, o);
    if constexpr (TR) {
      const int r = 32 * p + sub;
      const int f = ((r >> 3) & 3) * 2 + (r & 1);
      const uint32_t base = smem_u32(tile) + r * 256;
      const uint4 h0 = make_uint4(o[0], o[1], o[2], o[3]), h1 = make_uint4(o[4], o[5], o[6], o[7]);
      // the upper segments store their second unit first: eight lanes, eight banks
      const int swap = seg >> 2;
      sts128(base + (((2 * seg + swap) ^ f) << 4), swap ? h1 : h0);
      sts128(base + (((2 * seg + 1 - swap) ^ f) << 4), swap ? h0 : h1);
    } else if constexpr (MODE == kDqAnyRows) {
      const uint32_t base = smem_u32(tile) + (32 * p + sub) * 256 + seg * 32;
      sts128(base, make_uint4(o[0], o[1], o[2], o[3]));
      sts128(base + 16, make_uint4(o[4], o[5], o[6], o[7]));
    } else if (row < M && col < K) {
      T* dst = out + row * ldo + col;
      if (col + 16 <= K && vec) {
        st_global_v8(dst, o);
      } else if (col + 16 <= K) {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
      } else {
        uint16_t* d = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (col + i < K) d[i] = static_cast<uint16_t>(o[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
  if constexpr (MODE == kDqAnyRows) {
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = static_cast<int>(min(static_cast<int64_t>(kMxTile), K - col0));
    for (int r = warp; r < kMxTile && row0 + r < M; r += kMxThreads / 32) {
      uint16_t* dst = reinterpret_cast<uint16_t*>(out) + (row0 + r) * ldo + col0;
      const uint16_t* src = tile + r * kMxTile;
      const int odd = (reinterpret_cast<uintptr_t>(dst) >> 1) & 1;  // elements ahead of the first whole word
      for (int e = odd + 2 * lane; e + 1 < n; e += 64)
        *reinterpret_cast<uint32_t*>(dst + e) = src[e] | (static_cast<uint32_t>(src[e + 1]) << 16);
      if (odd && lane == 0) dst[0] = src[0];
      if (((n - odd) & 1) && n > odd && lane == 1) dst[n - 1] = src[n - 1];
    }
  }
  if constexpr (TR) {
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint16_t* o16 = reinterpret_cast<uint16_t*>(out);
    // 32 rows x 8 columns at a time: matrix i takes rows 8 q + 2 i + {0, 1} as its slots
    // 2 q + {0, 1}, so that transposed lane (c, q) holds rows 8 q .. 8 q + 7 of column c
    // -- 16 bytes of the output's row c
    const int slot = lane & 7, mat = lane >> 3;
    const int cc = lane >> 2, q = lane & 3;
    for (int t = warp; t < 4 * (kMxTile / 8); t += kMxThreads / 32) {
      const int rb = (t & 3) * 32, u = t >> 2;  // row block, unit of eight columns
      const int r = rb + 8 * (slot >> 1) + 2 * mat + (slot & 1);
      uint32_t v[4];
      __syncwarp();
      ldmatrix_x4_trans(v, smem_u32(tile) + r * 256 + ((u ^ (((r >> 3) & 3) * 2 + (r & 1))) << 4));
      const int64_t c = col0 + u * 8 + cc, row = row0 + rb + 8 * q;
      uint16_t* dst = o16 + c * ldo + row;
      if (c < K && vec && row + 8 <= Mw) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
      } else if (c < K) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (row + i < Mw) dst[i] = static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename T, int FMT>
int quantize_t(const void* x, int64_t ldx, void* codes, void* scales, int64_t M, int64_t K, float g,
               cudaStream_t stream) {
  const int64_t Kp = mx_padded_k(K);
  const dim3 grid(static_cast<unsigned>((Kp + kMxTile - 1) / kMxTile), static_cast<unsigned>((M + kMxTile - 1) / kMxTile));
  auto kernel = aligned(x, 32) && ldx % 16 == 0  ? mx_quantize_kernel<T, FMT, 32>
                : aligned(x, 16) && ldx % 8 == 0 ? mx_quantize_kernel<T, FMT, 16>
                                                 : mx_quantize_kernel<T, FMT, 2>;
  kernel<<<grid, kMxThreads, 0, stream>>>(static_cast<const T*>(x), ldx, static_cast<uint8_t*>(codes),
                                          static_cast<uint8_t*>(scales), M, K, Kp,
                                          static_cast<int>(mx_scale_chunks(K, FMT)), mx_global(g));
  return cudaGetLastError() == cudaSuccess ? LORA_OK : LORA_ERR_CUDA;
}

template <typename T, int FMT>
int dequantize_t(const void* codes, const void* scales, void* out, int64_t ldo, int64_t M, int64_t K, float g,
                 int transpose, cudaStream_t stream) {
  const int64_t Kp = mx_padded_k(K);
  // the composite operators ask for rows padded to 16 bytes (transpose == 2)
  const int64_t Mw = transpose == 2 ? (M + 7) / 8 * 8 : M;
  const dim3 grid(static_cast<unsigned>((Kp + kMxTile - 1) / kMxTile), static_cast<unsigned>((M + kMxTile - 1) / kMxTile));
  const int chunks = static_cast<int>(mx_scale_chunks(K, FMT));
  const bool vec = transpose ? aligned(out, 16) && ldo % 8 == 0 : aligned(out, 32) && ldo % 16 == 0;
  auto kernel = transpose ? mx_dequantize_kernel<T, FMT, kDqTransposed>
                : aligned(out, 16) && ldo % 8 == 0 ? mx_dequantize_kernel<T, FMT, kDqRows>
                                                   : mx_dequantize_kernel<T, FMT, kDqAnyRows>;
  kernel<<<grid, kMxThreads, 0, stream>>>(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
                                          static_cast<T*>(out), ldo, M, Mw, K, Kp, chunks, g, vec);
  return cudaGetLastError() == cudaSuccess ? LORA_OK : LORA_ERR_CUDA;
}

}  // namespace

int mx_quantize_launch(const void* x, int64_t ldx, void* codes, void* scales, int64_t M, int64_t K, int fmt, float g,
                       int dtype, cudaStream_t s) {
#define LORA_MXQ(T)                                                                                    \
  (fmt == LORA_MXFP4   ? quantize_t<T, LORA_MXFP4>(x, ldx, codes, scales, M, K, g, s)                  \
   : fmt == LORA_NVFP4 ? quantize_t<T, LORA_NVFP4>(x, ldx, codes, scales, M, K, g, s)                  \
                       : quantize_t<T, LORA_MXFP8>(x, ldx, codes, scales, M, K, g, s))
  return dtype == LORA_BF16 ? LORA_MXQ(__nv_bfloat16) : LORA_MXQ(__half);
#undef LORA_MXQ
}

int mx_dequantize_launch(const void* codes, const void* scales, void* out, int64_t ldo, int64_t M, int64_t K, int fmt,
                         float g, int transpose, int dtype, cudaStream_t s) {
#define LORA_MXD(T)                                                                                    \
  (fmt == LORA_MXFP4   ? dequantize_t<T, LORA_MXFP4>(codes, scales, out, ldo, M, K, g, transpose, s)   \
   : fmt == LORA_NVFP4 ? dequantize_t<T, LORA_NVFP4>(codes, scales, out, ldo, M, K, g, transpose, s)   \
                       : dequantize_t<T, LORA_MXFP8>(codes, scales, out, ldo, M, K, g, transpose, s))
  return dtype == LORA_BF16 ? LORA_MXD(__nv_bfloat16) : LORA_MXD(__half);
#undef LORA_MXD
}

}  // namespace lora

using namespace lora;

// Sizes a CTA grid of 128 x 128 tiles can cover (grid.y <= 65535).
static bool mx_shape_ok(int64_t M, int64_t K) {
  return M >= 0 && K >= 0 && M <= 65535ll * 128 && K <= (int64_t{1} << 30);
}

extern "C" size_t lora_mx_codes_size(int64_t M, int64_t K, int fmt) {
  if (!mx_format_ok(fmt) || M <= 0 || K <= 0) return 0;
  return static_cast<size_t>(M) * static_cast<size_t>(mx_code_pitch(K, fmt));
}

extern "C" size_t lora_mx_scales_size(int64_t M, int64_t K, int fmt) {
  if (!mx_format_ok(fmt) || M <= 0 || K <= 0) return 0;
  return static_cast<size_t>((M + 127) / 128) * static_cast<size_t>(mx_scale_chunks(K, fmt)) * 512;
}

extern "C" int lora_mx_quantize(const void* x, int64_t ldx, void* codes, void* scales, int64_t M, int64_t K, int fmt,
                                float global_scale, int dtype, void* stream) {
  if (!mx_format_ok(fmt) || (dtype != LORA_BF16 && dtype != LORA_F16)) return LORA_ERR_DTYPE;
  if (!mx_shape_ok(M, K) || ldx < K) return LORA_ERR_SHAPE;
  if (!mx_global_ok(global_scale, fmt)) return LORA_ERR_ARG;
  if (M == 0 || K == 0) return LORA_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr) return LORA_ERR_ARG;
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(x, 2)) return LORA_ERR_ALIGN;
  const int dev = current_device();
  if (dev < 0 || !device_info(dev).is_sm100) return LORA_ERR_DEVICE;
  return mx_quantize_launch(x, ldx, codes, scales, M, K, fmt, global_scale, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int lora_mx_dequantize(const void* codes, const void* scales, void* out, int64_t ldo, int64_t M, int64_t K,
                                  int fmt, float global_scale, int transpose, int dtype, void* stream) {
  if (!mx_format_ok(fmt) || (dtype != LORA_BF16 && dtype != LORA_F16)) return LORA_ERR_DTYPE;
  if (!mx_shape_ok(M, K) || ldo < (transpose ? M : K)) return LORA_ERR_SHAPE;
  if (!mx_global_ok(global_scale, fmt)) return LORA_ERR_ARG;
  if (M == 0 || K == 0) return LORA_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr) return LORA_ERR_ARG;
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(out, 2)) return LORA_ERR_ALIGN;
  const int dev = current_device();
  if (dev < 0 || !device_info(dev).is_sm100) return LORA_ERR_DEVICE;
  return mx_dequantize_launch(codes, scales, out, ldo, M, K, fmt, global_scale, transpose, dtype,
                              static_cast<cudaStream_t>(stream));
}
