// Shared by the attention kernels' translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200q.h"

namespace b200q {

// Tokens of a call: a tile beyond stays within 32 bits.
constexpr int kMostTokens = 0x7fffffff - 1024;

// b200q_view's rules.
inline int check_view(const b200q_view& x) {
  if (x.data == nullptr) return B200Q_ERR_NULL_POINTER;
  for (int64_t s : {x.page, x.token, x.head})
    if (s % 8 != 0 || s < 0 || s >= (int64_t{1} << 39)) return B200Q_ERR_UNSUPPORTED_SHAPE;
  return (reinterpret_cast<uintptr_t>(x.data) & 15u) != 0 ? B200Q_ERR_MISALIGNED : B200Q_OK;
}

// gemm_umma.cu: TMA descriptor of 16-bit elements with 2 to 5 dimensions, strides in elements (of dimensions 1 on), the
// 128-byte swizzle, zeros outside.  Encoded on every call.
bool make_tensor_map_16(const void* base, int dims, const uint64_t* size, const int64_t* stride, const uint32_t* box,
                        CUtensorMap* out);

// Rows of a view that one TMA box brings: [box_rows] positions of one head, 64 dimensions each.  Packed
// keys are one page of key_tokens positions.
bool make_key_map(const b200q_view& x, const b200q_attention& a, uint32_t box_rows, CUtensorMap* out);

// attn_decode.cu, attn_prefill.cu; return B200Q_* codes
int launch_attn_decode(const b200q_attention& a, void* workspace, int* status, cudaStream_t stream);
size_t attn_decode_workspace(const b200q_attention& a);
int launch_attn_prefill(const b200q_attention& a, void* workspace, int* status, cudaStream_t stream);
size_t attn_prefill_workspace(const b200q_attention& a);

}  // namespace b200q
