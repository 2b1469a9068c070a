// The paged 8-bit cache of keys and values as its kernels see it: arguments, checks of them, the rule of its scales.
#pragma once

#include <climits>

#include "launch.cuh"

namespace b200 {

struct KvView {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int64_t pages, page_stride;
  int kv_heads, page_tokens;
  const int32_t *starts, *lengths, *table;
  int sequences, tokens, ld_pages;
  int* status;
};

namespace {

// Smallest and largest exponent of a scale the append writes. The lower end is for the sum of a softmax's weights, which are held divided
// by these scales: at most 2^100 for a key where few rows are attended (2^120 for a million of them, inside f32), 2^108 where many are (the
// weights' 2^15, less 2^7), whose sums pass f32 with a million keys that are all next to the lower end, such as values of zeros: the
// results are then 0 for numbers below 2^-91. No f32 needs a scale above the upper end.
constexpr int kScaleMin = -100, kScaleMax = 122;

// A sequence's rows and slots, 0 new tokens where what the arrays say cannot be.
struct Span {
  int row0, n, length;
};
__device__ __forceinline__ Span span_of(const KvView& A, int s, bool& bad) {
  const int r0 = A.starts[s], r1 = A.starts[s + 1], len = A.lengths[s];
  bad = r0 < 0 || r1 < r0 || r1 > A.tokens || len < 0;
  return bad ? Span{0, 0, 0} : Span{r0, r1 - r0, len};
}
// The page that holds a sequence's slots page_tokens * i and on, or -1.
__device__ __forceinline__ int page_of(const KvView& A, int s, int i) {
  if (i < 0 || i >= A.ld_pages) return -1;
  const int p = A.table[static_cast<int64_t>(s) * A.ld_pages + i];
  return p < 0 || p >= A.pages ? -1 : p;
}
__device__ __forceinline__ void report_batch(const KvView& A) {
  if (A.status) atomicExch(A.status, kStatusBatch);
}

// Four values of a row; vec: they lie on a boundary of their size.
__device__ __forceinline__ float4 load_row4(const void* p, int dtype, int64_t i, bool vec) {
  if (vec) {
    if (dtype == LX_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  }
  return make_float4(load_f32(p, dtype, i), load_f32(p, dtype, i + 1), load_f32(p, dtype, i + 2), load_f32(p, dtype, i + 3));
}

// The same of N rows at once: every load is issued before one is waited for, which a choice of the type within each does not do.
template <int N>
__device__ __forceinline__ void load_rows4(const void* p, int dtype, const int64_t (&at)[N], bool vec, float4 (&x)[N]) {
  if (vec && dtype == LX_BF16) {
    uint2 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at[i]);
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = make_float4(__uint_as_float(w[i].x << 16), __uint_as_float(w[i].x & 0xffff0000u), __uint_as_float(w[i].y << 16), __uint_as_float(w[i].y & 0xffff0000u));
  } else if (vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = load_row4(p, dtype, at[i], false);
  }
}
// a / b of counts: 64-bit division is a hundred instructions, and hardly ever needed.
__device__ __forceinline__ int64_t divide(int64_t a, int b) {
  return a >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}

// ---- host -----------------------------------------------------------------------------------------------------------
inline int check_cache(const lx_b200_kv_cache* c) {
  if (!c || c->kv_heads < 1 || c->pages < 1 || !c->k || !c->v || !c->k_scale || !c->v_scale) return kInvalid;
  if (c->type != LX_W_FP8 && c->type != LX_W_INT8) return kNotSupported;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return kNotSupported;
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) return kNotSupported;
  if (c->kv_heads > 1024 || c->pages > INT_MAX) return kNotSupported;
  const int64_t page = static_cast<int64_t>(c->kv_heads) * c->page_tokens * c->head_dim;
  if (c->page_stride < page || c->page_stride % 16 || !aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
    return kInvalid;
  return kOk;
}
inline int check_batch(const lx_b200_kv_batch* b) {
  if (!b || b->sequences < 0 || b->tokens < 0 || b->max_new < 0 || b->ld_pages < 0) return kInvalid;
  if (b->sequences > (1 << 30)) return kNotSupported;  // loops over them count past the last one, in 32 bits
  if (b->sequences > 0 && (!b->starts || !b->lengths || (b->ld_pages > 0 && !b->pages))) return kInvalid;
  return kOk;
}
inline KvView view_of(const lx_b200_kv_cache& c, const lx_b200_kv_batch& b) {
  KvView A;
  A.k = static_cast<uint8_t*>(c.k), A.v = static_cast<uint8_t*>(c.v), A.k_scale = c.k_scale, A.v_scale = c.v_scale;
  A.pages = c.pages, A.page_stride = c.page_stride, A.kv_heads = c.kv_heads, A.page_tokens = c.page_tokens;
  A.starts = b.starts, A.lengths = b.lengths, A.table = b.pages;
  A.sequences = b.sequences, A.tokens = b.tokens, A.ld_pages = b.ld_pages;
  A.status = status_word();
  return A;
}

}  // namespace
}  // namespace b200
