// What the attention kernels share: arguments, exponentials, the scale of a query row, the store of results.
#pragma once

#include "kv.cuh"
#include "tc.cuh"

namespace b200 {

// What a CTA of the stream kernel leaves for the join: the unit that begins in its share and goes on into the next one's, rows 0 where there is none.
struct JoinInfo {
  int row0, row_block, rows, head, last, pad[3];  // last: the share that holds the unit's end
};

struct AttentionArgs {
  KvView kv;
  const void* q;
  uint16_t* out;
  float* partial;
  JoinInfo* join;
  int64_t ld_q, ld_out;
  int q_dtype, q_heads, group, window, min_tiles;
  float scale_log2;  // the softmax's scale times log2 e
  bool out_vec, q_vec;  // rows of `out` and of `q` go on in pieces of four values
  bool pad;             // rows past the last sequence become zeros
  int most;             // the query rows per key head up to which a sequence is the stream kernel's; the tiles take those with more
};

namespace {

// The first slot seen by a row that sees the slots before `past` (0 or less: none). `past` is as far below 0 as a
// sequence is shorter than its new tokens, and a window as wide as an int: their difference need not be one.
__device__ __forceinline__ int first_seen(int past, int window) { return window > 0 ? max(0, max(0, past) - window) : 0; }
// Tiles that hold the slots before `past`, which may be the largest int: such sums are unsigned, here and where slots are compared with it.
__device__ __forceinline__ int tiles_before(int past, int tile) { return past <= 0 ? 0 : static_cast<int>((static_cast<uint32_t>(past) + tile - 1) / tile); }

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

// Zeros in the rows of no sequence, which begin at row `from`: all threads of a CTA, one of `ctas`.
__device__ __forceinline__ void zero_rows_from(const AttentionArgs& A, int from, int head_dim, int cta, int ctas) {
  if (from < 0) return;
  for (int64_t row = static_cast<int64_t>(from) + cta; row < A.kv.tokens; row += ctas)
    for (int c = 4 * threadIdx.x; c < A.q_heads * head_dim; c += 4 * blockDim.x) store_out(A, row * A.ld_out + c, make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f);
}

// ---- codes to f16 pairs, exact ------------------------------------------------------------------------------------------
template <bool kInt8>
__device__ __forceinline__ void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {  // codes 0, 1 and codes 2, 3
  if constexpr (kInt8) {
    const uint32_t u = w ^ 0x80808080u;  // code + 128, placed in the digits of 1024
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x), hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

}  // namespace

// attention_tile.cu: sequences of more than `limit` query rows per key head, in tiles of 128 rows on tcgen05. The workspace is its own.
int64_t tile_attention_workspace(int head_dim, int kv_heads, int group, int tokens, int sequences);
int tile_attention(AttentionArgs A, int head_dim, bool int8, int limit, void* workspace, cudaStream_t stream);

}  // namespace b200
