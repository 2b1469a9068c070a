// lx_b200_kv_append: new keys and values into a paged 8-bit cache, rotated on the way, and the rotated queries.
//
// A CTA has the new tokens of one page for one key head: it alone decides the page's scales for that head, so there are no atomics and
// the codes do not depend on the order of anything. It reads its rows twice: once for their largest magnitudes, once (from the
// caches) for their codes. The queries of the heads that share the key head are other CTAs'.
#include <algorithm>

#include "kv.cuh"

namespace b200 {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAnglePairs = 4096;  // cosines and sines held at once: 32 KB

struct AppendArgs {
  KvView kv;
  const void *k, *v, *q;
  void* q_out;
  int64_t ld_k, ld_v, ld_q, ld_q_out;
  int kv_dtype, q_dtype, q_out_dtype, group, head_dim, rotary, interleaved, int8, splits;
  bool k_vec, v_vec, q_vec, q_out_vec;  // rows in whole pieces of four values
  const int32_t* positions;
  const double* frequencies;
};

__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, const float* v, bool vec) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) store_from_f32(p, dtype, i + j, v[j]);
  } else if (dtype == LX_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        make_uint2(f32_to_bf16_bits(v[0]) | f32_to_bf16_bits(v[1]) << 16, f32_to_bf16_bits(v[2]) | f32_to_bf16_bits(v[3]) << 16);
  }
}

// A piece of a head is eight values that turn together: two runs of four, `first` and `second`, that begin at lo and hi.
struct Piece {
  int lo, hi, pair;  // pair: the first of its four pairs, -1 where nothing turns
};
__device__ __forceinline__ Piece piece_of(const AppendArgs& A, int u) {
  const int r = A.rotary;
  if (8 * u >= r) return {8 * u, 8 * u + 4, -1};
  return A.interleaved ? Piece{8 * u, 8 * u + 4, 4 * u} : Piece{4 * u, 4 * u + r / 2, 4 * u};
}
// The eight values of a piece, turned by the angles at cs.
__device__ __forceinline__ void turn(const AppendArgs& A, const float4& a, const float4& b, const Piece& u, const float2* cs, float (&x)[8]) {
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  if (u.pair < 0 || !cs) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 c = cs[u.pair + j];
    if (A.interleaved) {
      const float s = x[2 * j], t = x[2 * j + 1];
      x[2 * j] = s * c.x - t * c.y, x[2 * j + 1] = t * c.x + s * c.y;
    } else {
      const float s = x[j], t = x[j + 4];
      x[j] = s * c.x - t * c.y, x[j + 4] = t * c.x + s * c.y;
    }
  }
}
// Four codes of values already divided by their scale.
__device__ __forceinline__ uint32_t codes4(const float* v, int int8) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = int8 ? static_cast<uint32_t>(static_cast<int>(rintf(fminf(fmaxf(v[j], -127.0f), 127.0f)))) & 0xffu : e4m3_encode(v[j]) & 0xffu;
    w |= b << (8 * j);
  }
  return w;
}
// The smallest power of two, within the limits, that brings a magnitude (its bits) to 448 (0.875 * 2^9) or 127 ((1 - 2^-7) * 2^7) or less.
__device__ __forceinline__ float scale_for(uint32_t magnitude, int int8) {
  if (magnitude >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  if (magnitude < 0x00800000u) return __uint_as_float(static_cast<uint32_t>(127 + kScaleMin) << 23);
  const int e = static_cast<int>(magnitude >> 23) - 126;  // magnitude = m 2^e, m in [0.5, 1)
  const uint32_t m = magnitude & 0x7fffffu;
  const int want = int8 ? e - 7 + (m > 0x7e0000u) : e - 9 + (m > 0x600000u);
  return __uint_as_float(static_cast<uint32_t>(127 + min(max(want, kScaleMin), kScaleMax)) << 23);
}

// Which pages a CTA has. With splits > 0 (batches whose sequences have about equally many new tokens) CTA x has the pages x % splits,
// + splits, ... of sequence x / splits. Else it has place x of the batch: sequence s has starts[s] / P + 2 s .. starts[s + 1] / P +
// 2 s + 1 of these, no fewer than the pages that its new tokens can touch, whatever slot they begin in. (A decode step of 64 sequences
// takes 7.4 us the first way and 10.7 the second; a long prompt among 63 of them would leave 8,000 CTAs idle the first way.)
__device__ __forceinline__ int places_before(const KvView& C, int s) { return min(max(C.starts[s], 0), C.tokens) / C.page_tokens + 2 * s; }

__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const __grid_constant__ AppendArgs A) {
  __shared__ float2 angles[kAnglePairs];
  __shared__ uint32_t most[2];
  __shared__ int next, matches;
  pdl_wait();
  const KvView& C = A.kv;
  const int tid = threadIdx.x, x = blockIdx.x;
  const bool queries = blockIdx.y >= C.kv_heads;  // of the heads that share key head `head`, by CTAs of their own
  const int head = queries ? blockIdx.y - C.kv_heads : blockIdx.y;
  const int P = C.page_tokens, D = A.head_dim, log_units = __ffs(D) - 4, units = 1 << log_units, half = A.rotary / 2;
  const int chunk = half ? min(P, kAnglePairs / half) : P;
  // The sequence whose place this is; several only where the rows of sequences overlap, as they should not.
  for (int s = -1, left = 1; left > 0; --left) {
    if (A.splits > 0) {
      s = x / A.splits;
    } else {
      __syncthreads();
      if (tid == 0) next = INT_MAX, matches = 0;
      __syncthreads();
      for (int c = tid; c < C.sequences; c += kAppendThreads)
        if (c > s && places_before(C, c) <= x && x < places_before(C, c + 1)) atomicMin(&next, c), atomicAdd(&matches, 1);
      __syncthreads();
      s = next, left = matches;
      if (left == 0) break;
    }
    bool bad;
    const Span q = span_of(C, s, bad);
    if (bad || q.length < q.n || q.n == 0) continue;
    const int first = q.length - q.n, place = A.splits > 0 ? x % A.splits : x - places_before(C, s), stride = A.splits > 0 ? A.splits : INT_MAX / 2;
    for (int page = first / P + place; page <= (q.length - 1) / P; page += stride) {
      const int lo = max(first, page * P), kept = lo - page * P, n = min(q.length - lo, P - kept), row0 = q.row0 + lo - first;
      const int at = page_of(C, s, page);
      if (at < 0 && tid == 0 && blockIdx.y == 0) report_batch(C);
      if (tid < 2) most[tid] = 0;
      float now[2], inverse[2];
      for (int pass = 0; pass < (queries ? 1 : 2); ++pass) {
        uint32_t large[2] = {0, 0};
        for (int c0 = 0; c0 < n; c0 += chunk) {
          const int m = min(chunk, n - c0);
          __syncthreads();  // whoever still reads the angles, or `most`
          if (half && (pass == 0 || n > chunk))
            for (int i = tid; i < m * half; i += kAppendThreads) {
              const int t = i / half;
              const int position = A.positions ? A.positions[row0 + c0 + t] : lo + c0 + t;
              // in turns, less the whole ones, before anything is rounded to f32: a position of a million costs no digits
              double turns = static_cast<double>(position) * A.frequencies[i - t * half] * 0.15915494309189533577;
              turns -= rint(turns);
              float2 cs;
              sincospif(2.0f * static_cast<float>(turns), &cs.y, &cs.x);
              angles[i] = cs;
            }
          __syncthreads();
          const float2* cs = half ? angles : nullptr;
          for (int i = tid; !queries && i < m * units; i += kAppendThreads) {
            const int t = i >> log_units;
            const Piece u = piece_of(A, i & (units - 1));
            const int64_t k_at = (row0 + c0 + t) * A.ld_k + head * D, v_at = (row0 + c0 + t) * A.ld_v + head * D;
            float4 kx[2], vx[2];
            const int64_t from_k[2] = {k_at + u.lo, k_at + u.hi}, from_v[2] = {v_at + u.lo, v_at + u.hi};
            load_rows4(A.k, A.kv_dtype, from_k, A.k_vec, kx);
            load_rows4(A.v, A.kv_dtype, from_v, A.v_vec, vx);
            float x[8], y[8];
            turn(A, kx[0], kx[1], u, half ? cs + t * half : nullptr, x);
            turn(A, vx[0], vx[1], u, nullptr, y);
            if (pass == 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                large[0] = max(large[0], __float_as_uint(x[j]) & 0x7fffffffu);  // as integers: not-a-number is the largest
                large[1] = max(large[1], __float_as_uint(y[j]) & 0x7fffffffu);
              }
            } else if (at >= 0) {
              const int64_t dst = at * C.page_stride + (static_cast<int64_t>(head) * P + kept + c0 + t) * D;
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = now[0] == now[0] ? x[j] * inverse[0] : 0.0f, y[j] = now[1] == now[1] ? y[j] * inverse[1] : 0.0f;
              *reinterpret_cast<uint32_t*>(C.k + dst + u.lo) = codes4(x, A.int8);
              *reinterpret_cast<uint32_t*>(C.k + dst + u.hi) = codes4(x + 4, A.int8);
              *reinterpret_cast<uint32_t*>(C.v + dst + u.lo) = codes4(y, A.int8);
              *reinterpret_cast<uint32_t*>(C.v + dst + u.hi) = codes4(y + 4, A.int8);
            }
          }
          if (queries) {  // two pieces of a thread on their way at once
            const int all = m * A.group << log_units;
            for (int i0 = tid; i0 < all; i0 += 2 * kAppendThreads) {
              Piece u[2];
              int token[2];
              int64_t col[2], from[4];
              float4 x[4];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int i = min(i0 + e * kAppendThreads, all - 1), r = i >> log_units;
                token[e] = r / A.group;
                u[e] = piece_of(A, i & (units - 1));
                col[e] = static_cast<int64_t>(head * A.group + r - token[e] * A.group) * D;
                const int64_t at = (row0 + c0 + token[e]) * A.ld_q + col[e];
                from[2 * e] = at + u[e].lo, from[2 * e + 1] = at + u[e].hi;
              }
              load_rows4(A.q, A.q_dtype, from, A.q_vec, x);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (i0 + e * kAppendThreads >= all) break;
                float y[8];
                turn(A, x[2 * e], x[2 * e + 1], u[e], half ? cs + token[e] * half : nullptr, y);
                const int64_t at = (row0 + c0 + token[e]) * A.ld_q_out + col[e];
                store4(A.q_out, A.q_out_dtype, at + u[e].lo, y, A.q_out_vec);
                store4(A.q_out, A.q_out_dtype, at + u[e].hi, y + 4, A.q_out_vec);
              }
            }
          }
        }
        if (pass == 0 && !queries) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            large[w] = __reduce_max_sync(0xffffffffu, large[w]);
            if ((tid & 31) == 0) atomicMax(&most[w], large[w]);
          }
          __syncthreads();
          if (at < 0) break;
          const int64_t sc = static_cast<int64_t>(at) * C.kv_heads + head;
          float* const scales[2] = {C.k_scale + sc, C.v_scale + sc};
          uint8_t* const codes[2] = {C.k, C.v};
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const float want = scale_for(most[w], A.int8), was = kept ? *scales[w] : want;
            // not-a-number, of old or of new values, stays
            now[w] = was != was || want != want ? __uint_as_float(0x7fffffffu) : fmaxf(was, want);
            inverse[w] = 1.0f / now[w];
            if (kept && now[w] > was) {
              const float ratio = was / now[w];
              uint4* held = reinterpret_cast<uint4*>(codes[w] + at * C.page_stride + static_cast<int64_t>(head) * P * D);
              for (int i = tid; i < kept * D / 16; i += kAppendThreads) {
                const uint4 old = held[i];
                uint32_t word[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                  float x[4];
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    const uint32_t code = word[b] >> (8 * j) & 0xffu;
                    x[j] = (A.int8 ? static_cast<float>(static_cast<int8_t>(code)) : (code & 0x7fu) == 0x7fu ? __uint_as_float(0x7fffffffu) : e4m3_to_f32(code)) * ratio;
                  }
                  word[b] = codes4(x, A.int8);
                }
                held[i] = make_uint4(word[0], word[1], word[2], word[3]);
              }
            }
          }
          __syncthreads();  // every thread has read the old scales
          if (tid < 2) *scales[tid] = now[tid];
        }
      }
    }
  }
  if (x == 0 && blockIdx.y == 0)
    for (int c = tid; c < C.sequences; c += kAppendThreads) {
      bool bad;
      const Span q = span_of(C, c, bad);
      if (bad || q.length < q.n) report_batch(C);
    }
}

// Whether rows of heads begin and go on in pieces of four values.
bool fours(const void* p, int dtype, int64_t ld) { return aligned(p, dtype == LX_BF16 ? 8 : 16) && ld % 4 == 0; }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int lx_b200_kv_append(const lx_b200_kv_cache* cache, const lx_b200_kv_batch* batch, const void* k, int ld_k, const void* v, int ld_v,
                                 lx_dtype kv_dtype, const void* q, lx_dtype q_dtype, int ld_q, int q_heads, void* q_out, lx_dtype q_out_dtype,
                                 int ld_q_out, const int32_t* positions, const double* frequencies, int rotary_dim, int interleaved,
                                 void* stream) {
  if (int e = check_cache(cache)) return e;
  if (int e = check_batch(batch)) return e;
  const int64_t D = cache->head_dim, H = cache->kv_heads;
  if (!valid_dtype(kv_dtype) || !valid_dtype(q_dtype) || !valid_dtype(q_out_dtype) || q_heads < 0 || rotary_dim < 0 || rotary_dim > D) return kInvalid;
  if (rotary_dim % 8) return kNotSupported;
  if (rotary_dim && !frequencies) return kInvalid;
  if (batch->sequences == 0 || batch->tokens == 0) return kOk;
  if (!k || !v || ld_k < H * D || ld_v < H * D) return kInvalid;
  const int heads = q ? q_heads : 0;
  if (q && (q_heads < 1 || q_heads % H || !q_out || ld_q < q_heads * D || ld_q_out < q_heads * D)) return kInvalid;
  AppendArgs A;
  A.kv = view_of(*cache, *batch);
  A.k = k, A.v = v, A.q = q, A.q_out = q_out;
  A.ld_k = ld_k, A.ld_v = ld_v, A.ld_q = ld_q, A.ld_q_out = ld_q_out;
  A.kv_dtype = kv_dtype, A.q_dtype = q_dtype, A.q_out_dtype = q_out_dtype;
  A.group = heads / static_cast<int>(H), A.head_dim = static_cast<int>(D), A.rotary = rotary_dim, A.interleaved = interleaved;
  A.int8 = cache->type == LX_W_INT8;
  A.k_vec = fours(k, kv_dtype, ld_k), A.v_vec = fours(v, kv_dtype, ld_v), A.q_vec = fours(q, q_dtype, ld_q), A.q_out_vec = fours(q_out, q_out_dtype, ld_q_out);
  A.positions = positions, A.frequencies = frequencies;
  const int64_t places = batch->tokens / cache->page_tokens + 2 * static_cast<int64_t>(batch->sequences);
  if (places > INT_MAX) return kNotSupported;
  const int64_t splits = (std::min(std::max(batch->max_new, 1), batch->tokens) + cache->page_tokens - 2) / cache->page_tokens + 1;
  const bool even = splits * batch->sequences <= places;
  A.splits = even ? static_cast<int>(splits) : 0;
  return launch_kernel(kv_append_kernel, dim3(static_cast<unsigned>(even ? splits * batch->sequences : places), static_cast<unsigned>(H) * (heads ? 2 : 1)), dim3(kAppendThreads), 0,
                       static_cast<cudaStream_t>(stream), A);
}
