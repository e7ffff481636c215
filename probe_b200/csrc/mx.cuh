// Microscaled formats (4- and 8-bit floating point with a scale per block).
//
//   mxfp4   E2M1 codes, a power of two (E8M0 byte) per 32 values of a row
//   nvfp4   E2M1 codes, an E4M3 scale per 16 values, one fp32 scale per tensor
//   mxfp8   E4M3 codes, a power of two (E8M0 byte) per 32 values
//
// Storage of an [M, K] tensor, Kp = K rounded up to 32:
//   codes   row-major, Kp/2 bytes a row (two E2M1 codes a byte, the even column
//           in the low half) or Kp bytes (E4M3); columns K..Kp-1 hold zeros
//   scales  512-byte chunks of 128 rows x 4 blocks, chunk (row / 128) * GB +
//           block / 4 with GB = ceil(blocks / 4); row r and block g of a chunk
//           at byte 16 (r % 32) + 4 (r / 32) + g; rows and blocks beyond the
//           tensor hold zeros.  One chunk is what tcgen05.cp.32x128b copies
//           into 4 columns of TMEM for a block-scaled MMA, so neither the
//           product nor its loads rearrange a byte.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace lora {

template <int FMT> struct MxFormat;
template <> struct MxFormat<LORA_MXFP4> {
  static constexpr int kBlock = 32, kBits = 4, kTop = 2;  // kTop: exponent of the largest code
};
template <> struct MxFormat<LORA_NVFP4> {
  static constexpr int kBlock = 16, kBits = 4, kTop = 2;
};
template <> struct MxFormat<LORA_MXFP8> {
  static constexpr int kBlock = 32, kBits = 8, kTop = 8;
};

inline int mx_block(int fmt) { return fmt == LORA_NVFP4 ? 16 : 32; }
inline int mx_bits(int fmt) { return fmt == LORA_MXFP8 ? 8 : 4; }
inline int64_t mx_padded_k(int64_t k) { return (k + 31) / 32 * 32; }
inline int64_t mx_code_pitch(int64_t k, int fmt) { return mx_padded_k(k) * mx_bits(fmt) / 8; }
inline int64_t mx_scale_chunks(int64_t k, int fmt) { return (mx_padded_k(k) / mx_block(fmt) + 3) / 4; }
inline bool mx_format_ok(int fmt) { return fmt == LORA_MXFP4 || fmt == LORA_NVFP4 || fmt == LORA_MXFP8; }
// The tensor-wide scale of nvfp4 (1 for the others): in this range scale x block
// scale and its reciprocal are normal fp32 numbers.
inline bool mx_global_ok(float g, int fmt) {
  return fmt == LORA_NVFP4 ? (g >= 5.4210109e-20f && g <= 1.8446744e19f) : g == 1.0f;  // [2^-64, 2^64]
}

// Shared-memory accesses by 32-bit address: behind the dynamic buffer's aligned
// base the compiler only sees generic pointers, whose loads take the global path.
LORA_DEVINL uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
LORA_DEVINL uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
LORA_DEVINL float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
LORA_DEVINL uint32_t lds_u8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
LORA_DEVINL uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
LORA_DEVINL void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 32-byte global accesses (32-byte aligned).
LORA_DEVINL void ldg_stream_v8(const void* p, uint32_t* w) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
LORA_DEVINL void st_global_v8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 16 elements of 2 bytes of a row from column c, zeros at and beyond k, at any
// 2-byte alignment: the aligned 16-byte words that hold them, funnelled into place
// (no word is read that holds none of the 16).
LORA_DEVINL void ldg16_any(const void* row, int64_t c, int64_t k, uint32_t* w) {
  const uint16_t* p = static_cast<const uint16_t*>(row) + c;
  if (c + 16 <= k) {
    const uint32_t sh = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
    const uint4 a = ldg_stream(base), b = ldg_stream(base + 1);
    uint4 d = make_uint4(0u, 0u, 0u, 0u);
    if (sh != 0) d = ldg_stream(base + 2);
    uint32_t v[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, d.x, d.y, d.z, d.w};
    if (sh & 8) {
#pragma unroll
      for (int i = 0; i < 10; ++i) v[i] = v[i + 2];
    }
    if (sh & 4) {
#pragma unroll
      for (int i = 0; i < 9; ++i) v[i] = v[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = (sh & 2) ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t lo = c + 2 * i < k ? p[2 * i] : 0u;
    const uint32_t hi = c + 2 * i + 1 < k ? p[2 * i + 1] : 0u;
    w[i] = lo | (hi << 16);
  }
}

// Two fp32 operations an instruction.
LORA_DEVINL uint64_t f32x2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
LORA_DEVINL void unpack_f32x2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
LORA_DEVINL uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
LORA_DEVINL uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}

// MN-major operand in 64-wide chunks `lbo` bytes apart: rows of the contraction 128 bytes
// apart, 8-row groups 1024 bytes apart, 128-byte swizzle.
LORA_DEVINL uint64_t mx_desc_mn(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// A scale chunk in shared memory: 32 rows of 16 bytes, no swizzle, 8-row groups 128
// bytes apart.
LORA_DEVINL uint64_t mx_desc_scales(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(128 >> 4) << 16;
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}

// D (+)= A B^T of 4-bit codes with their block scales in TMEM, by one CTA (PAIR false) or a
// pair of them.
template <int FMT, bool PAIR>
LORA_DEVINL void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                        uint32_t accumulate) {
#define LORA_MX_MMA(GROUP, VEC)                                                                                  \
  asm volatile(                                                                                                  \
      "{\n\t.reg .pred p;\n\t"                                                                                  \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                               \
      "tcgen05.mma.cta_group::" GROUP ".kind::mxf4nvf4.block_scale.scale_vec::" VEC                              \
      " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                                        \
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                            \
      : "memory")
  if constexpr (FMT == LORA_MXFP4 && PAIR) LORA_MX_MMA("2", "2X");
  if constexpr (FMT == LORA_MXFP4 && !PAIR) LORA_MX_MMA("1", "2X");
  if constexpr (FMT == LORA_NVFP4 && PAIR) LORA_MX_MMA("2", "4X");
  if constexpr (FMT == LORA_NVFP4 && !PAIR) LORA_MX_MMA("1", "4X");
#undef LORA_MX_MMA
}

// One lane of a converged warp.  Asked anew in front of each block that one lane
// executes, never kept: the code generator may repeat the election where a kept
// answer is used, and in diverged code that elects several lanes.
LORA_DEVINL bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// mbar_wait_bounded by a whole warp: every lane waits for itself (an elected lane
// and a broadcast measured slower), every lane gets the same answer.
LORA_DEVINL bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int code) {
  const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort, err, code));
  __syncwarp();
  return ok;
}

// The two halves of cluster_sync_all, and the arrival half of a named barrier.
LORA_DEVINL void cluster_arrive_all() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
LORA_DEVINL void cluster_wait_all() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
LORA_DEVINL void named_bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The cluster meets.  Warp 1 gives its CTA's tensor memory back in between, once the
// reading warps (`readers`) are done with it: a CTA that held it and waited for a peer, which
// may be waiting for another kernel's, could wait for good.  Barrier 2.
LORA_DEVINL void cluster_sync_free_tmem(uint32_t tmem, uint32_t cols, int warp, bool reads, int readers) {
  if (reads) {
    tc_fence_before();
    named_bar_arrive(2, 32 * (readers + 1));
  }
  cluster_arrive_all();
  if (warp == 1) {
    named_bar_sync(2, 32 * (readers + 1));
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
  __syncwarp();
  cluster_wait_all();
}

// 2^(byte - 127) of an E8M0 scale byte; 255 is NaN.
LORA_DEVINL float mx_e8m0(uint32_t byte) {
  const uint32_t bits = byte == 0 ? 0x00400000u : (byte == 255 ? 0x7fffffffu : byte << 23);
  return __uint_as_float(bits);
}
// One E4M3 byte.
LORA_DEVINL float mx_e4m3(uint32_t byte) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(byte)));
  return __low2float(*reinterpret_cast<__half2*>(&h2));
}
// Two floats -> two E4M3 codes (lo in the low byte), nearest even, saturating.
LORA_DEVINL uint32_t mx_to_e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// Eight floats -> eight E2M1 codes, the first in the low bits.
LORA_DEVINL uint32_t mx_to_e2m1x8(const float* v) {
  uint32_t d;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(d)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return d;
}
// Eight E2M1 codes -> four f16 pairs (exact).
LORA_DEVINL void mx_from_e2m1x8(uint32_t w, uint32_t* h2) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h2[0]), "=r"(h2[1]), "=r"(h2[2]), "=r"(h2[3])
      : "r"(w));
}
// Two E4M3 codes -> one f16 pair (exact).
LORA_DEVINL uint32_t mx_from_e4m3x2(uint32_t w) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(w)));
  return h2;
}

// Largest magnitude, as the 16-bit pattern without its sign: infinities and
// NaN compare above every number.
LORA_DEVINL uint32_t mx_amax16(const uint32_t* w) {
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

template <typename T> LORA_DEVINL float mx_bits16_to_f32(uint32_t b);
template <> LORA_DEVINL float mx_bits16_to_f32<__nv_bfloat16>(uint32_t b) { return __uint_as_float(b << 16); }
template <> LORA_DEVINL float mx_bits16_to_f32<__half>(uint32_t b) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
}

// Tensor-wide constants of a quantisation: 6 g and its reciprocal, both rounded.
struct MxGlobal {
  float g, g6, r6;
};
inline MxGlobal mx_global(float g) {
  const float g6 = 6.0f * g;
  return MxGlobal{g, g6, 1.0f / g6};
}

// Correctly rounded quotients by one divisor: with r the correctly rounded
// reciprocal of d, one residual step makes x r the rounded x / d (Markstein,
// 1990).  |x r| is kept below 2^20 so that the residual stays finite; every
// quotient that large saturates.
LORA_DEVINL float mx_div_far(float x, float d, float r) {
  const float q = fminf(fmaxf(x * r, -1048576.f), 1048576.f);
  return fmaf(fmaf(-q, d, x), r, q);
}

// Scale of a block from its amax16: the byte to store and what turns a value
// into units of the scale (mxfp4 / mxfp8: mul; nvfp4: divisor and reciprocal).
template <typename T, int FMT>
struct MxScale {
  uint32_t byte;
  float d, r;
  bool far;
  // recip: shared address of the reciprocals of (E4M3 code x g), 128 entries (nvfp4)
  LORA_DEVINL MxScale(uint32_t top, const MxGlobal& gl, uint32_t recip) {
    constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    const bool bad = top >= kInf;
    const float amax = mx_bits16_to_f32<T>(top);
    if constexpr (FMT == LORA_NVFP4) {
      byte = bad ? 0x7fu : mx_to_e4m3x2(mx_div_far(amax, gl.g6, gl.r6), 0.f) & 0xffu;
      d = mx_e4m3(byte) * gl.g;
      r = lds_f32(recip + byte * 4);  // 0 for a zero or NaN scale
      far = amax * r > 1048576.f;
    } else {
      const int e = max(static_cast<int>(__float_as_uint(amax) >> 23) - MxFormat<FMT>::kTop, 0);  // biased by 127
      byte = bad ? 255u : static_cast<uint32_t>(e);
      r = bad ? 0.f : __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      d = 0.f;
      far = false;
    }
  }
};

// Entry `code` of the reciprocals: correctly rounded, 0 for zero and NaN scales
// (whose codes are zero).
LORA_DEVINL float mx_recip_entry(int code, float g) {
  return code == 0 || code >= 127 ? 0.f : __frcp_rn(mx_e4m3(static_cast<uint32_t>(code)) * g);
}

// Codes of 16 values: 8 (4-bit) or 16 bytes.
template <typename T, int FMT>
LORA_DEVINL void mx_codes16(const uint32_t* w, const MxScale<T, FMT>& s, uint32_t* codes) {
  float v[16];
  if constexpr (FMT == LORA_NVFP4) {
    if (s.r == 0.f) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    } else if (s.far) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 x = unpack2<T>(w[i]);
        v[2 * i] = mx_div_far(x.x, s.d, s.r);
        v[2 * i + 1] = mx_div_far(x.y, s.d, s.r);
      }
    } else {  // mx_div_far without its clamp, on pairs
      const uint64_t r = f32x2(s.r, s.r), nd = f32x2(-s.d, -s.d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 x = unpack2<T>(w[i]);
        const uint64_t xx = f32x2(x.x, x.y);
        const uint64_t q = mul_f32x2(xx, r);
        unpack_f32x2(fma_f32x2(fma_f32x2(q, nd, xx), r, q), v[2 * i], v[2 * i + 1]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = unpack2<T>(s.byte == 255u ? 0u : w[i]);
      unpack_f32x2(mul_f32x2(f32x2(x.x, x.y), f32x2(s.r, s.r)), v[2 * i], v[2 * i + 1]);
    }
  }
  if constexpr (MxFormat<FMT>::kBits == 4) {
    codes[0] = mx_to_e2m1x8(v);
    codes[1] = mx_to_e2m1x8(v + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      codes[i] = mx_to_e4m3x2(v[4 * i], v[4 * i + 1]) | (mx_to_e4m3x2(v[4 * i + 2], v[4 * i + 3]) << 16);
  }
}

// Device entry points of the parts (host launchers), used by the C ABI and by
// the composite operators.  transpose: 0, 1, or 2 for [K, M rounded up to 8] with
// zeros in the padding.
int mx_quantize_launch(const void* x, int64_t ldx, void* codes, void* scales, int64_t M, int64_t K, int fmt,
                       float global_scale, int dtype, cudaStream_t stream);
int mx_dequantize_launch(const void* codes, const void* scales, void* out, int64_t ldo, int64_t M, int64_t K, int fmt,
                         float global_scale, int transpose, int dtype, cudaStream_t stream);

}  // namespace lora
