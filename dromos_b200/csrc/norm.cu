// lx_b200_norm_residual: the norm after a block, its gate, the scaled residual and the norm before the next block, one pass over the
// rows.
//
//   u = y rsqrt(mean y^2 + eps) post;   h' = residual_scale h + block_scale gate u;   x = h' rsqrt(mean h'^2 + eps) pre
//
// A row is one CTA's; a thread keeps its values in registers from the one read of y, h and gate to the writes of h' and x. Few rows are
// a chain of latencies: all loads, the weights' among them, are issued at once (one row of 4096: 2.8 us). Many rows are bound by HBM,
// and what counts is that one row of an SM loads while another one is summed: then the weights, which the caches hold, are read
// where they are used, so that two CTAs of 512 threads fit the SM's registers. The same threads have the same values either way, and
// every product and sum of a value is written out, so that the compiler does not round once here and twice there.
#include <algorithm>

#include "tc.cuh"

namespace b200 {
namespace {

struct NormArgs {
  const void *y, *h, *gate, *post, *pre;
  void *h_out, *x;
  int64_t ld_y, ld_h, ld_gate, ld_h_out, ld_x;
  int y_dtype, h_dtype, gate_dtype, weight_dtype, x_dtype;
  int gate_sigmoid, C;
  float residual_scale, block_scale, eps;
};

// Eight values of a row as they lie in memory; the conversion is apart so that every load of a row is issued before the first is used.
struct Raw8 {
  uint4 a, b;
};
__device__ __forceinline__ Raw8 load_raw8(const void* p, int dtype, int64_t i) {
  Raw8 r;
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * (dtype == LX_BF16 ? 2 : 4));
  r.a = q[0];
  r.b = dtype == LX_BF16 ? make_uint4(0, 0, 0, 0) : q[1];
  return r;
}
__device__ __forceinline__ void values_of(const Raw8& r, int dtype, float (&v)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dtype == LX_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  }
}
__device__ __forceinline__ void store8(void* p, int dtype, int64_t i, const float (&v)[8]) {
  if (dtype == LX_BF16) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = f32_to_bf16_bits(v[2 * q]) | f32_to_bf16_bits(v[2 * q + 1]) << 16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}
// The sum over a CTA, the same bits in every thread. `part`: 32 words, used by one sum only.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
  if (lane == 0) part[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? part[lane] : 0.0f);
}
__device__ __forceinline__ float gate_of(float g, int sigmoid) { return sigmoid ? 1.0f / (1.0f + expf(-g)) : g; }

// Rows of whole 16-byte-aligned pieces of eight values: thread t has the pieces t, t + blockDim.x, ... (PIECES of them at most).
template <int PIECES, bool LATE>
__global__ void __launch_bounds__(512, LATE ? (PIECES == 1 ? 3 : PIECES == 2 ? 2 : 1) : 1) norm_kernel(const __grid_constant__ NormArgs A) {
  __shared__ float part[2][32];
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int pieces = A.C / 8;
  Raw8 y[PIECES], h[PIECES], g[LATE ? 1 : PIECES], wp[LATE ? 1 : PIECES], wn[LATE ? 1 : PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int p = threadIdx.x + i * blockDim.x;
    if (p >= pieces) continue;
    if (A.y) y[i] = load_raw8(A.y, A.y_dtype, row * A.ld_y + 8 * p);
    h[i] = load_raw8(A.h, A.h_dtype, row * A.ld_h + 8 * p);
    if (!LATE && A.y && A.gate) g[i] = load_raw8(A.gate, A.gate_dtype, row * A.ld_gate + 8 * p);
    if (!LATE && A.y && A.post) wp[i] = load_raw8(A.post, A.weight_dtype, 8 * p);
    if (!LATE && A.pre) wn[i] = load_raw8(A.pre, A.weight_dtype, 8 * p);
  }
  float scale = A.block_scale;
  if (A.y && A.post) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (threadIdx.x + i * blockDim.x >= pieces) continue;
      float v[8];
      values_of(y[i], A.y_dtype, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
    }
    scale *= rsqrtf(block_sum(sum, part[0]) / static_cast<float>(A.C) + A.eps);
  }
  float next[PIECES][8], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int p = threadIdx.x + i * blockDim.x;
    if (p >= pieces) continue;
    float u[8], v[8];
    values_of(h[i], A.h_dtype, next[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) next[i][j] = __fmul_rn(next[i][j], A.residual_scale);
    if (A.y) {
      values_of(y[i], A.y_dtype, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = __fmul_rn(u[j], scale);
      if (A.post) {
        values_of(LATE ? load_raw8(A.post, A.weight_dtype, 8 * p) : wp[LATE ? 0 : i], A.weight_dtype, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = __fmul_rn(u[j], v[j]);
      }
      if (A.gate) {
        values_of(LATE ? load_raw8(A.gate, A.gate_dtype, row * A.ld_gate + 8 * p) : g[LATE ? 0 : i], A.gate_dtype, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = __fmul_rn(u[j], gate_of(v[j], A.gate_sigmoid));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) next[i][j] = __fadd_rn(next[i][j], u[j]);
    }
    if (A.h_out) store8(A.h_out, A.h_dtype, row * A.ld_h_out + 8 * p, next[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(next[i][j], next[i][j], sum);
  }
  if (!A.pre) return;
  const float rms = rsqrtf(block_sum(sum, part[1]) / static_cast<float>(A.C) + A.eps);
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int p = threadIdx.x + i * blockDim.x;
    if (p >= pieces) continue;
    float v[8];
    values_of(LATE ? load_raw8(A.pre, A.weight_dtype, 8 * p) : wn[LATE ? 0 : i], A.weight_dtype, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], __fmul_rn(next[i][j], rms));
    store8(A.x, A.x_dtype, row * A.ld_x + 8 * p, v);
  }
}

// Any width, stride and alignment: three passes over the row, which the caches hold. h_out may be h: the thread that writes a value
// is the one that reads it, in the last pass.
__global__ void __launch_bounds__(1024) norm_any_kernel(const __grid_constant__ NormArgs A) {
  __shared__ float part[2][32];
  pdl_wait();
  const int64_t row = blockIdx.x;
  float scale = A.block_scale;
  if (A.y && A.post) {
    float sum = 0.0f;
    for (int c = threadIdx.x; c < A.C; c += blockDim.x) {
      const float v = load_f32(A.y, A.y_dtype, row * A.ld_y + c);
      sum = fmaf(v, v, sum);
    }
    scale *= rsqrtf(block_sum(sum, part[0]) / static_cast<float>(A.C) + A.eps);
  }
  auto next_of = [&](int c) {
    float v = A.residual_scale * load_f32(A.h, A.h_dtype, row * A.ld_h + c);
    if (A.y) {
      float u = load_f32(A.y, A.y_dtype, row * A.ld_y + c) * scale;
      if (A.post) u *= load_f32(A.post, A.weight_dtype, c);
      if (A.gate) u *= gate_of(load_f32(A.gate, A.gate_dtype, row * A.ld_gate + c), A.gate_sigmoid);
      v += u;
    }
    return v;
  };
  float rms = 0.0f;
  if (A.pre) {
    float sum = 0.0f;
    for (int c = threadIdx.x; c < A.C; c += blockDim.x) {
      const float v = next_of(c);
      sum = fmaf(v, v, sum);
    }
    rms = rsqrtf(block_sum(sum, part[1]) / static_cast<float>(A.C) + A.eps);
  }
  for (int c = threadIdx.x; c < A.C; c += blockDim.x) {
    const float v = next_of(c);
    if (A.h_out) store_from_f32(A.h_out, A.h_dtype, row * A.ld_h_out + c, v);
    if (A.pre) store_from_f32(A.x, A.x_dtype, row * A.ld_x + c, v * rms * load_f32(A.pre, A.weight_dtype, c));
  }
}

// Whether rows `ld` elements apart start on 16 bytes.
bool whole(const void* p, int dtype, int64_t ld) { return !p || (aligned(p, 16) && ld * (dtype == LX_BF16 ? 2 : 4) % 16 == 0); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int lx_b200_norm_residual(const void* y, lx_dtype y_dtype, int ld_y, const void* h, lx_dtype h_dtype, int ld_h, const void* gate,
                                     lx_dtype gate_dtype, int ld_gate, int gate_sigmoid, const void* post, const void* pre,
                                     lx_dtype weight_dtype, float residual_scale, float block_scale, float eps, void* h_out, int ld_h_out,
                                     void* x, lx_dtype x_dtype, int ld_x, int T, int C, void* stream) {
  if (T < 0 || C < 1 || !valid_dtype(y_dtype) || !valid_dtype(h_dtype) || !valid_dtype(gate_dtype) || !valid_dtype(weight_dtype) || !valid_dtype(x_dtype))
    return kInvalid;
  if (T == 0) return kOk;
  if (!h || (!x && pre) || (!h_out && !pre)) return kInvalid;
  if (ld_h < C || (y && ld_y < C) || (gate && ld_gate != 0 && ld_gate < C) || (h_out && ld_h_out < C) || (pre && ld_x < C)) return kInvalid;
  NormArgs A{y, h, gate, post, pre, h_out, x, ld_y, ld_h, ld_gate, ld_h_out, ld_x, y_dtype, h_dtype, gate_dtype, weight_dtype, x_dtype,
             gate_sigmoid, C, residual_scale, block_scale, eps};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool pieces = C % 8 == 0 && whole(y, y_dtype, ld_y) && whole(h, h_dtype, ld_h) && whole(gate, gate_dtype, ld_gate) && whole(post, weight_dtype, 0) &&
                      whole(pre, weight_dtype, 0) && whole(h_out, h_dtype, ld_h_out) && whole(pre ? x : nullptr, x_dtype, ld_x);
  // how a row is dealt to threads goes by C alone, so a row's bits do not depend on the other rows
  const bool late = T > 2 * sm_count();  // two rows for each SM: from here on rows wait for one another and not for their own loads
  auto threads = [&](int per) { return dim3(((C / 8 + per - 1) / per + 31) / 32 * 32); };
  if (pieces && C <= 8 * 512) return launch_kernel(late ? norm_kernel<1, true> : norm_kernel<1, false>, dim3(T), threads(1), 0, s, A);
  if (pieces && C <= 16 * 512) return launch_kernel(late ? norm_kernel<2, true> : norm_kernel<2, false>, dim3(T), threads(2), 0, s, A);
  if (pieces && C <= 32 * 512) return launch_kernel(late ? norm_kernel<4, true> : norm_kernel<4, false>, dim3(T), threads(4), 0, s, A);
  return launch_kernel(norm_any_kernel, dim3(T), dim3(std::min(1024, (C + 31) / 32 * 32)), 0, s, A);
}
