// Host interface of the rank shrink with its fused quantisation (mx_shrink.cu).
#pragma once

#include "mx_linear.h"

namespace lora {

struct MxShrinkOperands {
  const void* v;  // [M, K], ldv
  const void* a;  // [R, K] or, a_mn, [K, R]
  bool a_mn;
  // [M, ldz]: hi at column 0, lo at r16.  fmt -1 of fp16 operands: `groups` columns groups of
  // bf16, r16 wide, the parts of an exact sum of three (3) and the first two again (5)
  void* z;
  int groups;
  void *codes, *scales;   // of v in the format, where one is asked for
  void *part, *tickets;   // mx_shrink_part_bytes; the zeroed ticket region
  int64_t ldv, lda, ldz, M, K, R;
  float scale, global_scale;
};

size_t mx_shrink_part_bytes(int64_t M, int64_t K, int64_t R);
// TMA needs 16-byte rows.
bool mx_shrink_serves(const void* v, int64_t ldv, const void* a, int64_t lda);
// fmt: LORA_MXFP4 / LORA_NVFP4 (a_mn false) or -1 for the shrink alone.
int mx_shrink_launch(const MxShrinkOperands& o, int fmt, int dtype, cudaStream_t stream);

}  // namespace lora
