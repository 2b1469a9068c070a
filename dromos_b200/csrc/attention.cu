// lx_b200_attention: causal attention of new tokens' queries over a paged 8-bit cache.
#include <algorithm>

#include "kv.cuh"

namespace b200 {
namespace {

struct AttentionArgs {
  KvView kv;
  const void* q;
  uint16_t* out;
  int64_t ld_q, ld_out;
  int q_dtype, q_heads, group, window, int8;
  float scale_log2;  // the softmax's scale times log2 e
};

__device__ __forceinline__ float code_value(uint32_t code, int int8) {
  return int8 ? static_cast<float>(static_cast<int8_t>(code)) : e4m3_to_f32(code);
}

// One warp per query row and head: a running maximum and sum over the slots it sees, one slot after the other.
template <int D>
__global__ void __launch_bounds__(128) attention_rows_kernel(const __grid_constant__ AttentionArgs A) {
  pdl_wait();
  const KvView& C = A.kv;
  const int lane = threadIdx.x & 31, h = blockIdx.y;
  const int64_t row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= C.tokens) return;
  int s = -1, slot = 0;
  for (int i = 0; i < C.sequences && s < 0; ++i) {
    bool bad;
    const Span q = span_of(C, i, bad);
    if (bad && lane == 0) report_batch(C);
    if (row >= q.row0 && row < q.row0 + q.n) s = i, slot = q.length - q.n + static_cast<int>(row) - q.row0;
  }
  if (s < 0) return;
  constexpr int V = D / 32;
  float q[V], o[V] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) q[i] = load_f32(A.q, A.q_dtype, row * A.ld_q + h * D + lane * V + i) * A.scale_log2;
  const int kvh = h / A.group, P = C.page_tokens;
  for (int j = A.window > 0 ? max(0, slot - A.window + 1) : 0; j <= slot; ++j) {
    const int page = page_of(C, s, j / P);
    if (page < 0 && lane == 0) report_batch(C);
    const int64_t at = max(page, 0) * C.page_stride + (static_cast<int64_t>(kvh) * P + j % P) * D + lane * V;
    const int64_t sc = static_cast<int64_t>(max(page, 0)) * C.kv_heads + kvh;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) dot = fmaf(q[i], code_value(C.k[at + i], A.int8), dot);
    dot = page < 0 ? __uint_as_float(0x7fffffffu) : warp_sum(dot) * C.k_scale[sc];
    const float top = fmaxf(m, dot), shrink = m == -INFINITY ? 0.0f : exp2f(m - top), p = exp2f(dot - top), pv = p * C.v_scale[sc];
    l = l * shrink + p;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = fmaf(pv, code_value(C.v[at + i], A.int8), o[i] * shrink);
    m = top;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) A.out[row * A.ld_out + h * D + lane * V + i] = static_cast<uint16_t>(f32_to_bf16_bits(slot < 0 ? 0.0f : o[i] / l));
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int64_t lx_b200_attention_workspace_bytes(const lx_b200_kv_cache* cache, int q_heads, int max_new) {
  if (check_cache(cache) || q_heads < 1 || q_heads % cache->kv_heads || max_new < 0) return -1;
  return 0;
}

extern "C" int lx_b200_attention(const lx_b200_kv_cache* cache, const lx_b200_kv_batch* batch, const void* q, lx_dtype q_dtype, int ld_q, int q_heads,
                                 float scale, int window, void* out, int ld_out, void* workspace, void* stream) {
  if (int e = check_cache(cache)) return e;
  if (int e = check_batch(batch)) return e;
  const int64_t width = static_cast<int64_t>(q_heads) * cache->head_dim;
  if (!valid_dtype(q_dtype) || q_heads < 1 || q_heads % cache->kv_heads || window < 0 || width > INT_MAX) return kInvalid;
  if (batch->sequences == 0 || batch->tokens == 0) return kOk;
  if (!q || !out || ld_q < width || ld_out < width) return kInvalid;
  AttentionArgs A;
  A.kv = view_of(*cache, *batch);
  A.q = q, A.out = static_cast<uint16_t*>(out), A.ld_q = ld_q, A.ld_out = ld_out;
  A.q_dtype = q_dtype, A.q_heads = q_heads, A.group = q_heads / cache->kv_heads, A.window = window, A.int8 = cache->type == LX_W_INT8;
  A.scale_log2 = scale * 1.4426950408889634f;
  auto kernel = cache->head_dim == 64 ? attention_rows_kernel<64> : cache->head_dim == 128 ? attention_rows_kernel<128> : attention_rows_kernel<256>;
  return launch_kernel(kernel, dim3((batch->tokens + 3) / 4, q_heads), dim3(128), 0, static_cast<cudaStream_t>(stream), A);
}
