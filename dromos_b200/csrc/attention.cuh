// What the attention kernels share: arguments, exponentials, the scale of a query row, the store of results.
#pragma once

#include "kv.cuh"
#include "tc.cuh"

namespace b200 {
namespace {

struct AttentionArgs {
  KvView kv;
  const void* q;
  uint16_t* out;
  float* partial;
  int64_t ld_q, ld_out;
  int q_dtype, q_heads, group, window, min_tiles;
  float scale_log2;  // the softmax's scale times log2 e
  bool out_vec;      // rows of `out` go on in pieces of four values
};

// 2^x, 2^-22 relative, results below f32's normal range 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The power of two that brings a row's largest magnitude to 2^14 .. 2^15, inside f16's range.
__device__ __forceinline__ float f16_scale(float most) { return scale_of<kActF16>(most); }

__device__ __forceinline__ void store_out(const AttentionArgs& A, int64_t at, const float4& v, float factor) {
  const uint32_t w[4] = {f32_to_bf16_bits(v.x * factor), f32_to_bf16_bits(v.y * factor), f32_to_bf16_bits(v.z * factor), f32_to_bf16_bits(v.w * factor)};
  if (A.out_vec) {
    *reinterpret_cast<uint2*>(A.out + at) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) A.out[at + j] = static_cast<uint16_t>(w[j]);
  }
}

}  // namespace
}  // namespace b200
