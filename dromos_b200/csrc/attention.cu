// lx_b200_attention: causal attention of new tokens' queries over a paged 8-bit cache.
//
//   out = sum_j w_j v_j / sum_j w_j,   w_j = exp2(c q . k_j),   k_j = kscale kcode_j,  v_j = vscale vcode_j
//
// One pass over the keys. The 8-bit codes are exact in f16 and go to the tensor cores as they are; the scales stay outside, in f32:
// t_j = c kscale (q . kcode_j) + log2 vscale, and with the running maximum m of these t the weights p_j = 2^(14 + t_j - m)
// are what multiplies vcode_j, rounded to f16 (2^-11; below 2^-14 the step is 2^-24, which is 2^-38 of the largest weight), so pages of
// very different loudness share one accumulator; the sum of the weights takes p_j 2^-14 / vscale, in f32.
#include <algorithm>

#include "attention.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kJoinThreads = 512;
constexpr int kTile = 16 * kWarps;  // slots of a tile: 16 for each warp

// Work of a sequence: units (blocks of ROWS query rows x key heads) of equally many tiles.
struct SeqWork {
  Span q;
  int blocks, tile0, tiles;
  int64_t all;
  bool bad;
};
template <int ROWS>
__device__ __forceinline__ SeqWork work_of(const AttentionArgs& A, int s) {
  SeqWork w;
  w.q = span_of(A.kv, s, w.bad);
  const int rows = w.q.n * A.group;
  w.blocks = rows <= A.most ? (rows + ROWS - 1) / ROWS : 0;
  const int first = w.q.length - w.q.n;
  w.tile0 = first_seen(first + 1, A.window) / kTile;
  w.tiles = max(1, tiles_before(w.q.length, kTile) - w.tile0);
  w.all = static_cast<int64_t>(w.blocks) * A.kv.kv_heads * w.tiles;
  return w;
}

// Every CTA has the same count of consecutive tiles of the whole batch, `per`; a unit that several CTAs share is joined by a second kernel.
// Called by all threads; `sums`: shared. The sequence that holds tile `at` and its first tile's number come back in shared memory.
struct Place {
  int64_t total, base;  // base: tiles of the sequences before `seq`
  int seq;              // -1: past the end
};
template <int ROWS>
__device__ Place find_tile(const AttentionArgs& A, int64_t piece, int pieces, int64_t& per, int64_t& at, Place* shared, int64_t* sums) {
  const int S = A.kv.sequences, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) shared->seq = -1;
  int64_t total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t base = 0;
    for (int s0 = 0; s0 < S; s0 += kThreads) {
      int64_t mine = 0;
      if (s0 + tid < S) {
        const SeqWork w = work_of<ROWS>(A, s0 + tid);
        mine = w.all;
        if (w.bad && piece == 0) report_batch(A.kv);
      }
      int64_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      __syncthreads();
      if (lane == 31) sums[warp] = incl;
      __syncthreads();
      int64_t all = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) incl += sums[w];
        all += sums[w];
      }
      const bool whole = S <= kThreads;  // one round: its sums serve both passes
      if (pass == 0) total += all;
      if (pass == 1 || whole) {
        if (whole) {
          per = max(static_cast<int64_t>(A.min_tiles), divide(total + pieces - 1, pieces));
          at = piece * per;
        }
        if (base + incl > at && base + incl - mine <= at) shared->seq = s0 + tid, shared->base = base + incl - mine;
        base += all;
        if (whole) pass = 1;
        else if (base > at) break;
      }
    }
    if (pass == 0) {
      per = max(static_cast<int64_t>(A.min_tiles), divide(total + pieces - 1, pieces));
      at = piece * per;
    }
  }
  __syncthreads();
  return {total, shared->base, shared->seq};
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Plain loads, not those of the read-only path: the kernel may be resident before the append that wrote the codes has ended.
template <int WORDS>
__device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 2) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "l"(p + 4 * i));
  }
}

// What a warp needs of a step's page beside its codes.
struct StepScale {
  float k, v;
};
__device__ __forceinline__ StepScale step_scale(const AttentionArgs& A, int page, int head) {
  if (page < 0) {
    const float nan = __uint_as_float(0x7fffffffu);
    return {nan, nan};
  }
  const int64_t at = static_cast<int64_t>(page) * A.kv.kv_heads + head;
  return {A.kv.k_scale[at], A.kv.v_scale[at]};
}

// CTAs of an SM: what the accumulators' registers leave room for. (256 values per head: three CTAs spill, 24 sequences 45 us for 43.)
template <int D, int NT>
constexpr int stream_ctas() {
  return D == 256 ? 2 : NT * D <= 128 ? 4 : NT * D <= 256 ? 3 : 2;
}

// NT groups of 8 query rows against the keys of one head. D: values of a head.
//
// A warp takes 16 slots at a time. Both products have the keys as the 16-row operand and the query rows as the 8 columns, so that a
// group of up to 8 queries wastes nothing: S^T = K Q^T, O^T += V^T P^T. The operands come straight from global memory into registers:
// lane (g, t) loads a quarter row of keys g and g + 8 (which of a head's values share an instruction does not matter to a dot
// product, the queries are laid out to match), and of values the dims g D/8 .. of slots 2t, 2t + 1, 2t + 8, 2t + 9, whose bytes are
// interleaved before they are widened. P^T turns from accumulator to operand by one movmatrix per 8 x 8.
template <bool kInt8, int D, int NT>
__global__ void __launch_bounds__(kThreads, stream_ctas<D, NT>()) attention_stream_kernel(const __grid_constant__ AttentionArgs A) {
  constexpr int ROWS = 8 * NT, KW = D / 16, VW = D / 32, MT = D / 16;
  constexpr int OS = D + 4;  // row stride of the accumulators in shared memory
  extern __shared__ __align__(16) uint8_t smem[];
  uint2* const qfrag = reinterpret_cast<uint2*>(smem);                     // [KW][NT][32]
  float* const osum = reinterpret_cast<float*>(smem + KW * NT * 32 * 8);   // [kWarps][ROWS][OS]
  float* const ms = osum + kWarps * ROWS * OS;                             // [kWarps][ROWS]
  float* const ls = ms + kWarps * ROWS;                                    // [kWarps][ROWS]
  float* const rowf = ls + kWarps * ROWS;                                  // [ROWS]
  __shared__ Place place;
  __shared__ int64_t sums[kWarps];
  pdl_wait();
  pdl_trigger();  // the join waits for the whole of this kernel; it may be brought up before
  const KvView& C = A.kv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  int64_t per, at;
  const Place start = find_tile<ROWS>(A, blockIdx.x, gridDim.x, per, at, &place, sums);
  if (tid == 0) A.join[blockIdx.x].rows = 0;  // so far
  if (start.seq < 0) return;
  const int64_t end = min(start.total, at + per);
  int s = start.seq;
  int64_t base = start.base;
  const int log_p = __ffs(C.page_tokens) - 1, page_mask = C.page_tokens - 1;
  while (at < end) {
    const SeqWork W = work_of<ROWS>(A, s);
    if (W.all == 0 || at >= base + W.all) {
      base += W.all;
      ++s;
      continue;
    }
    // this CTA's part of one unit
    const int unit = static_cast<int>(divide(at - base, W.tiles));
    const int64_t unit_at = base + static_cast<int64_t>(unit) * W.tiles;
    const int part0 = static_cast<int>(at - unit_at), part1 = static_cast<int>(min(static_cast<int64_t>(W.tiles), end - unit_at));
    const int head = unit % C.kv_heads, row_block = unit / C.kv_heads * ROWS, rows = min(ROWS, W.q.n * A.group - row_block);
    const int first = W.q.length - W.q.n;
    // what lane (g, t) knows of its rows 8 nt + 2 t and + 1: the first slot past what they see
    int past[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t4 + e;
        past[nt][e] = r < rows ? max(0, first + (row_block + r) / A.group + 1) : 0;
      }
    const int past_low = max(0, first + row_block / A.group + 1), past_high = max(0, first + (row_block + rows - 1) / A.group + 1);  // of the first and the last row
    const int see_low = first_seen(past_low, A.window);   // the first slot that any row sees
    const int see_all = first_seen(past_high, A.window);  // from here on all rows do
    float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    }
    // steps of 16 slots: this warp's every kWarps-th, those that some row sees
    int step = (W.tile0 + part0) * kWarps + warp;
    if (step < see_low / 16) step += (see_low / 16 - step + kWarps - 1) / kWarps * kWarps;
    const int step_end = min((W.tile0 + part1) * kWarps, tiles_before(past_high, 16));
    uint32_t kw[2][KW], vw[4][VW];
    auto page_at = [&](int st) {
      if (st >= step_end) return 0;
      const int p = page_of(C, s, st * 16 >> log_p);
      if (p < 0 && lane == 0) report_batch(C);
      return p;
    };
    auto slot_base = [&](int page, int st) {
      return max(page, 0) * C.page_stride + (static_cast<int64_t>(head) * C.page_tokens + (static_cast<uint32_t>(st) * 16 & page_mask)) * D;
    };
    auto load_k = [&](int64_t src) {
#pragma unroll
      for (int i = 0; i < 2; ++i) load_codes(C.k + src + (g + 8 * i) * D + t4 * (D / 4), kw[i]);
    };
    auto load_v = [&](int64_t src) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_codes(C.v + src + (2 * t4 + (i & 1) + 8 * (i >> 1)) * D + g * (D / 8), vw[i]);
    };
    const int page = page_at(step);
    int page_next = page_at(step + kWarps);
    // queries, while the table is read: each row times the power of two that brings it into f16's range
    {
      constexpr int PIECES = (D + 127) / 128, PER_WARP = ROWS / kWarps;
      float4 x[PER_WARP * PIECES];
      int64_t from[PER_WARP * PIECES];
#pragma unroll
      for (int i = 0; i < PER_WARP; ++i) {  // rows past the end: the last one, so that no load waits for a condition
        const int r = row_block + min(warp + kWarps * i, rows - 1);
        const int64_t src = (W.q.row0 + r / A.group) * A.ld_q + (static_cast<int64_t>(head) * A.group + r % A.group) * D;
#pragma unroll
        for (int b = 0; b < PIECES; ++b) from[i * PIECES + b] = src + (4 * lane + 128 * b) % D;
      }
      load_rows4(A.q, A.q_dtype, from, A.q_vec, x);
#pragma unroll
      for (int i = 0; i < PER_WARP; ++i) {
        const int r = warp + kWarps * i;
        float most = 0.0f;
#pragma unroll
        for (int b = 0; b < PIECES; ++b) most = fmaxf(fmaxf(fmaxf(most, fabsf(x[i * PIECES + b].x)), fabsf(x[i * PIECES + b].y)), fmaxf(fabsf(x[i * PIECES + b].z), fabsf(x[i * PIECES + b].w)));
        const float up = f16_scale(warp_max(most));
#pragma unroll
        for (int b = 0; b < PIECES; ++b) {
          const int d = 4 * lane + 128 * b;
          if (d >= D) continue;
          const float4 q = r < rows ? x[i * PIECES + b] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          const __half2 lo = __floats2half2_rn(q.x * up, q.y * up), hi = __floats2half2_rn(q.z * up, q.w * up);
          qfrag[(d % (D / 4) / 4 * NT + r / 8) * 32 + r % 8 * 4 + d / (D / 4)] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
        if (lane == 0) rowf[r] = A.scale_log2 / up;
      }
    }
    StepScale sc{};
    if (step < step_end) {
      const int64_t src = slot_base(page, step);
      load_k(src), load_v(src);
      sc = step_scale(A, page, head);
    }
    __syncthreads();
    float f[NT][2];  // the factors of the rows' scores
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) f[nt][0] = rowf[8 * nt + 2 * t4], f[nt][1] = rowf[8 * nt + 2 * t4 + 1];
    for (; step < step_end; step += kWarps) {
      const int slot = step * 16;
      // scores
      float x[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        uint32_t a[4];
        halves<kInt8>(kw[0][i], a[0], a[2]);
        halves<kInt8>(kw[1][i], a[1], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint2 b = qfrag[(i * NT + nt) * 32 + lane];
          mma16816<true>(x[nt], a, b.x, b.y);
        }
      }
      // the next step's keys, and what it needs of its page
      const bool more = step + kWarps < step_end;
      const int64_t src_next = slot_base(page_next, step + kWarps);
      const StepScale now = sc;
      if (more) {
        load_k(src_next);
        sc = step_scale(A, page_next, head);
      }
      page_next = page_at(step + 2 * kWarps);
      const float v_scale = now.v < 0x1p-100f ? 0x1p-100f : now.v, log_v = __log2f(v_scale), inv_v = 0x1p-14f / v_scale;
      const bool edge = slot + 16u > static_cast<uint32_t>(past_low) || slot < see_all;
      bool higher = false;
      float shrink[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[nt][e] = fmaf(x[nt][e], f[nt][e & 1] * now.k, log_v);
          if (edge) {
            const int j = slot + g + 8 * (e >> 1), p = past[nt][e & 1];
            if (j >= p || (A.window > 0 && j < p - A.window)) x[nt][e] = -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(x[nt][e], x[nt][e + 2]);
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
          const float old = m[nt][e];
          shrink[nt][e] = 1.0f;
          if (top > old) {
            m[nt][e] = top;
            shrink[nt][e] = exp2_fast(old - top);
            higher = true;
          }
        }
      }
      if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          l[nt][0] *= shrink[nt][0], l[nt][1] *= shrink[nt][1];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] *= shrink[nt][e & 1];
        }
      }
      uint32_t p0[NT], p1[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // a row that has seen nothing yet: 2^(-inf) and not 2^(-inf + inf)
          p[e] = exp2_fast(x[nt][e] - (m[nt][e & 1] == -INFINITY ? 0.0f : m[nt][e & 1] - 14.0f));
        }
        // a row that sees nothing of a page whose scale is not a number: nothing, and not 0 x NaN
        if (const float w = p[0] + p[2]; w != 0.0f) l[nt][0] = fmaf(w, inv_v, l[nt][0]);
        if (const float w = p[1] + p[3]; w != 0.0f) l[nt][1] = fmaf(w, inv_v, l[nt][1]);
        const __half2 a = __floats2half2_rn(p[0], p[1]), b = __floats2half2_rn(p[2], p[3]);
        p0[nt] = transpose8(*reinterpret_cast<const uint32_t*>(&a));
        p1[nt] = transpose8(*reinterpret_cast<const uint32_t*>(&b));
      }
      if (slot + 16u > static_cast<uint32_t>(past_high) || slot < see_low) {  // what no row sees may hold codes that are not numbers: 0 x NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = slot + 2 * t4 + (i & 1) + 8 * (i >> 1);
          if (j >= past_high || j < see_low)
#pragma unroll
            for (int w = 0; w < VW; ++w) vw[i][w] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t a[4];
          halves<kInt8>(__byte_perm(vw[0][w], vw[1][w], half ? 0x7362 : 0x5140), a[0], a[1]);
          halves<kInt8>(__byte_perm(vw[2][w], vw[3][w], half ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<true>(o[2 * w + half][nt], a, p0[nt], p1[nt]);
        }
      }
      if (more) load_v(src_next);
    }
    // the warps' parts meet in shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], sh);
        const int r = 8 * nt + 2 * t4 + e;
        if (g == 0) ms[warp * ROWS + r] = m[nt][e], ls[warp * ROWS + r] = l[nt][e];
#pragma unroll
        for (int w = 0; w < VW; ++w)
          *reinterpret_cast<float4*>(osum + (warp * ROWS + r) * OS + g * (D / 8) + 4 * w) =
              make_float4(o[2 * w][nt][e], o[2 * w][nt][e + 2], o[2 * w + 1][nt][e], o[2 * w + 1][nt][e + 2]);
      }
    __syncthreads();
    const bool complete = part0 == 0 && part1 == W.tiles;
    const int64_t slot_ws = 2 * static_cast<int64_t>(blockIdx.x) + (part0 == 0);
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float top = ms[r], sum = 0.0f;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ms[w * ROWS + r]);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = ms[w * ROWS + r], k = mw == -INFINITY ? 0.0f : exp2_fast(mw - top);
        // a warp whose scores were all not-a-number has no maximum, its sums say so
        const float lw = ls[w * ROWS + r];
        sum += mw == -INFINITY ? lw : lw * k;
        const float4 ow = *reinterpret_cast<const float4*>(osum + (w * ROWS + r) * OS + d);
        v.x = fmaf(ow.x, k, v.x), v.y = fmaf(ow.y, k, v.y), v.z = fmaf(ow.z, k, v.z), v.w = fmaf(ow.w, k, v.w);
      }
      if (complete) {
        const float inv = sum == 0.0f ? 0.0f : 0x1p-14f / sum;
        const int token = (row_block + r) / A.group, qh = head * A.group + (row_block + r) % A.group;
        store_out(A, (W.q.row0 + token) * A.ld_out + static_cast<int64_t>(qh) * D + d, v, inv);
      } else {
        float* dst = A.partial + slot_ws * (ROWS * (D + 2));
        if (d == 0) dst[r] = top, dst[ROWS + r] = sum;
        *reinterpret_cast<float4*>(dst + 2 * ROWS + r * D + d) = v;
      }
    }
    __syncthreads();  // before the next unit's queries and sums
    at = unit_at + part1;
    if (part0 == 0 && !complete && tid == 0) A.join[blockIdx.x] = {W.q.row0, row_block, rows, head, static_cast<int>((unit_at + W.tiles - 1) / per), {}};
  }
}

// Joins the units that several CTAs of the stream kernel shared: CTA i the one that began in share i and went on into the next. The
// parts' maxima and sums are looked at 32 parts at once, a lane for each; their accumulators are read by as many groups of threads as
// there are threads for (a part takes a thread 300 cycles, whatever is in flight beside it). As many CTAs as the stream kernel has are
// resident at once (one more wave of CTAs that find nothing costs 0.8 us). The rows of no sequence are zeroed here where that is asked for.
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads, stream_ctas<D, NT>()) attention_join_kernel(const __grid_constant__ AttentionArgs A) {
  constexpr int ROWS = 8 * NT, AT_ONCE = 32, CELLS = ROWS * (D / 4);  // four values each
  constexpr int GROUPS = CELLS >= kJoinThreads ? 1 : kJoinThreads / CELLS, ITEMS = CELLS > kJoinThreads ? CELLS / kJoinThreads : 1;
  __shared__ float ms[AT_ONCE][ROWS + 1], ls[AT_ONCE][ROWS + 1], shrink[ROWS], sums[ROWS], tops[ROWS];
  __shared__ float4 gathered[GROUPS > 1 ? GROUPS - 1 : 1][GROUPS > 1 ? CELLS : 1];
  pdl_wait();
  const JoinInfo u = A.join[blockIdx.x];
  const int behind = A.pad ? A.kv.starts[A.kv.sequences] : A.kv.tokens;  // on its way while the parts are joined
  if (u.rows == 0) {
    zero_rows_from(A, behind, D, blockIdx.x, gridDim.x);
    return;
  }
  const int tid = threadIdx.x, first = blockIdx.x, group = GROUPS > 1 ? tid / CELLS : 0, cell0 = GROUPS > 1 ? tid % CELLS : tid;
  const int64_t slot_floats = ROWS * (D + 2);
  auto slot = [&](int p) { return A.partial + (2 * static_cast<int64_t>(p) + (p == first)) * slot_floats; };
  if (tid < ROWS) sums[tid] = 0.0f, tops[tid] = -INFINITY;
  float4 v[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int p0 = first; p0 <= u.last; p0 += AT_ONCE) {
    const int n = min(AT_ONCE, u.last + 1 - p0);
    __syncthreads();
    for (int i = tid; i < n * ROWS; i += kJoinThreads) {
      const float* src = slot(p0 + i / ROWS) + i % ROWS;
      if (i % ROWS < u.rows) ms[i / ROWS][i % ROWS] = src[0], ls[i / ROWS][i % ROWS] = src[ROWS];
    }
    __syncthreads();
    for (int r = tid >> 5; r < u.rows; r += kJoinThreads / 32) {
      const int p = tid & 31;
      const float m = p < n ? ms[p][r] : -INFINITY, l = p < n ? ls[p][r] : 0.0f, before = tops[r], top = fmaxf(before, warp_max(m));
      // a part whose scores were all not-a-number has no maximum, its sums say so
      const float k = m == -INFINITY ? 0.0f : exp2_fast(m - top), gain = warp_sum(m == -INFINITY ? l : l * k);
      const float k0 = before == -INFINITY ? 0.0f : exp2_fast(before - top);
      if (p < n) ms[p][r] = k;
      __syncwarp();
      if (p == 0) shrink[r] = k0, tops[r] = top, sums[r] = (before == -INFINITY ? sums[r] : sums[r] * k0) + gain;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int cell = cell0 + i * kJoinThreads, r = cell / (D / 4);
      if (r >= u.rows) continue;
      const float k0 = shrink[r];
      v[i] = make_float4(v[i].x * k0, v[i].y * k0, v[i].z * k0, v[i].w * k0);
#pragma unroll 4
      for (int p = group; p < n; p += GROUPS) {
        const float4 o = *reinterpret_cast<const float4*>(slot(p0 + p) + 2 * ROWS + 4 * cell);
        const float k = ms[p][r];
        v[i].x = fmaf(o.x, k, v[i].x), v[i].y = fmaf(o.y, k, v[i].y), v[i].z = fmaf(o.z, k, v[i].z), v[i].w = fmaf(o.w, k, v[i].w);
      }
    }
  }
  zero_rows_from(A, behind, D, blockIdx.x, gridDim.x);
  if constexpr (GROUPS > 1) {
    if (group > 0) gathered[group - 1][cell0] = v[0];
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 0; g < GROUPS - 1; ++g) {
      const float4 o = gathered[g][cell0];
      v[0].x += o.x, v[0].y += o.y, v[0].z += o.z, v[0].w += o.w;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int cell = cell0 + i * kJoinThreads, r = cell / (D / 4);
    if (r >= u.rows) continue;
    const int token = (u.row_block + r) / A.group, qh = u.head * A.group + (u.row_block + r) % A.group;
    store_out(A, (u.row0 + token) * A.ld_out + static_cast<int64_t>(qh) * D + cell % (D / 4) * 4, v[i], sums[r] == 0.0f ? 0.0f : 0x1p-14f / sums[r]);
  }
}

template <int D, int NT>
constexpr size_t stream_smem() {
  return D / 16 * NT * 32 * 8 + sizeof(float) * (kWarps * 8 * NT * (D + 4) + 2 * kWarps * 8 * NT + 8 * NT);
}
template <int D, int NT>
int64_t stream_workspace() {
  return static_cast<int64_t>(sm_count()) * stream_ctas<D, NT>() * (2 * 8 * NT * (D + 2) * 4 + static_cast<int64_t>(sizeof(JoinInfo)));
}
template <bool kInt8, int D, int NT>
int launch_stream_attention(AttentionArgs A, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(sm_count()) * stream_ctas<D, NT>();
  if (grid == 0) return kNotSupported;
  A.join = reinterpret_cast<JoinInfo*>(A.partial + static_cast<int64_t>(grid) * 2 * 8 * NT * (D + 2));
  auto kernel = attention_stream_kernel<kInt8, D, NT>;
  if (int e = allow_dynamic_smem<(kInt8 * 4 + (D == 64 ? 0 : D == 128 ? 1 : 2)) * 8 + NT>(kernel)) return e;
  if (int e = launch_kernel(kernel, dim3(grid), dim3(kThreads), stream_smem<D, NT>(), stream, A)) return e;
  return launch_kernel(attention_join_kernel<D, NT>, dim3(grid), dim3(kJoinThreads), 0, stream, A);
}
// Groups of 8 rows that a CTA of the stream kernel takes at once: as few as hold a sequence's rows, 4 at most (2 with 256 values per
// head), whose accumulators fill the registers.
int row_groups(int head_dim, int64_t rows) { return rows <= 8 ? 1 : rows <= 16 || head_dim == 256 ? 2 : 4; }

template <bool kInt8, int D>
int stream_attention(const AttentionArgs& A, int64_t rows, cudaStream_t stream) {
  const int nt = row_groups(D, rows);
  if (nt == 1) return launch_stream_attention<kInt8, D, 1>(A, stream);
  if (nt == 2) return launch_stream_attention<kInt8, D, 2>(A, stream);
  if constexpr (D < 256) return launch_stream_attention<kInt8, D, 4>(A, stream);
  return kNotSupported;
}

}  // namespace
}  // namespace b200

using namespace b200;

// Query rows per key head up to which a sequence goes to the stream kernel; more go to tiles of 128 rows (attention_tile.cu).
static int stream_rows(int head_dim) { return head_dim == 256 ? 16 : 32; }

static int64_t stream_workspace(int head_dim, int64_t rows) {
  const int nt = row_groups(head_dim, rows);
  switch (head_dim) {
    case 64: return nt == 1 ? stream_workspace<64, 1>() : nt == 2 ? stream_workspace<64, 2>() : stream_workspace<64, 4>();
    case 128: return nt == 1 ? stream_workspace<128, 1>() : nt == 2 ? stream_workspace<128, 2>() : stream_workspace<128, 4>();
    default: return nt == 1 ? stream_workspace<256, 1>() : stream_workspace<256, 2>();
  }
}

// Which kernels a call launches, and where their workspaces are.
struct AttentionPlan {
  bool tiles, streams;
  int64_t rows;  // the most rows of a sequence that goes to the stream kernel
  int64_t tiles_at, total;
};
static AttentionPlan attention_plan(const lx_b200_kv_cache& c, const lx_b200_kv_batch& b, int group) {
  const int64_t rows = static_cast<int64_t>(std::max(1, b.max_new)) * group, limit = stream_rows(c.head_dim);
  AttentionPlan p;
  p.tiles = rows > limit, p.streams = !p.tiles || group <= limit;
  // beside sequences of many new tokens, those of one are what the stream kernel is cut for
  p.rows = p.tiles ? group : rows;
  p.tiles_at = p.streams ? (stream_workspace(c.head_dim, p.rows) + 255) / 256 * 256 : 0;
  p.total = p.tiles_at + (p.tiles ? tile_attention_workspace(c.head_dim, c.kv_heads, group, b.tokens, b.sequences) : 0);
  return p;
}

extern "C" int64_t lx_b200_attention_workspace_bytes(const lx_b200_kv_cache* cache, const lx_b200_kv_batch* batch, int q_heads) {
  if (check_cache(cache) || check_batch(batch) || q_heads < 1 || q_heads % cache->kv_heads) return -1;
  return attention_plan(*cache, *batch, q_heads / cache->kv_heads).total;
}

static int attention(const lx_b200_kv_cache* cache, const lx_b200_kv_batch* batch, const void* q, lx_dtype q_dtype, int ld_q, int q_heads, float scale, int window,
                     void* out, int ld_out, void* workspace, void* stream, bool pad) {
  if (int e = check_cache(cache)) return e;
  if (int e = check_batch(batch)) return e;
  const int64_t width = static_cast<int64_t>(q_heads) * cache->head_dim;
  if (!valid_dtype(q_dtype) || q_heads < 1 || q_heads % cache->kv_heads || window < 0 || width > INT_MAX) return kInvalid;
  if (batch->tokens == 0 || (batch->sequences == 0 && !pad)) return kOk;
  if (static_cast<int64_t>(batch->tokens) * (q_heads / cache->kv_heads) > INT_MAX / 2) return kNotSupported;
  if (!q || !out || ld_q < width || ld_out < width || !workspace || !aligned(workspace, 256)) return kInvalid;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (batch->sequences == 0) {
    const cudaError_t e = cudaMemset2DAsync(out, static_cast<size_t>(ld_out) * 2, 0, static_cast<size_t>(width) * 2, static_cast<size_t>(batch->tokens), st);
    if (e != cudaSuccess) cudaGetLastError();
    return static_cast<int>(e);
  }
  AttentionArgs A;
  A.kv = view_of(*cache, *batch);
  A.q = q, A.out = static_cast<uint16_t*>(out), A.ld_q = ld_q, A.ld_out = ld_out, A.partial = static_cast<float*>(workspace);
  A.q_dtype = q_dtype, A.q_heads = q_heads, A.group = q_heads / cache->kv_heads, A.window = window;
  A.out_vec = aligned(out, 8) && ld_out % 4 == 0, A.q_vec = aligned(q, q_dtype == LX_BF16 ? 8 : 16) && ld_q % 4 == 0;
  A.scale_log2 = scale * 1.4426950408889634f;
  A.min_tiles = 3;
  const bool int8 = cache->type == LX_W_INT8;
  const AttentionPlan plan = attention_plan(*cache, *batch, A.group);
  const int limit = stream_rows(cache->head_dim);
  A.pad = pad && !plan.streams;  // by the last join of the call
  if (plan.tiles)
    if (int e = tile_attention(A, cache->head_dim, int8, limit, static_cast<uint8_t*>(workspace) + plan.tiles_at, st)) return e;
  if (!plan.streams) return kOk;
  A.pad = pad;
  A.most = plan.tiles ? limit : INT_MAX;
  switch (cache->head_dim) {
    case 64: return int8 ? stream_attention<true, 64>(A, plan.rows, st) : stream_attention<false, 64>(A, plan.rows, st);
    case 128: return int8 ? stream_attention<true, 128>(A, plan.rows, st) : stream_attention<false, 128>(A, plan.rows, st);
    default: return int8 ? stream_attention<true, 256>(A, plan.rows, st) : stream_attention<false, 256>(A, plan.rows, st);
  }
}

extern "C" int lx_b200_attention(const lx_b200_kv_cache* cache, const lx_b200_kv_batch* batch, const void* q, lx_dtype q_dtype, int ld_q, int q_heads,
                                 float scale, int window, void* out, int ld_out, void* workspace, void* stream) {
  return attention(cache, batch, q, q_dtype, ld_q, q_heads, scale, window, out, ld_out, workspace, stream, false);
}

extern "C" int lx_b200_attention_padded(const lx_b200_kv_cache* cache, const lx_b200_kv_batch* batch, const void* q, lx_dtype q_dtype, int ld_q, int q_heads,
                                        float scale, int window, void* out, int ld_out, void* workspace, void* stream) {
  return attention(cache, batch, q, q_dtype, ld_q, q_heads, scale, window, out, ld_out, workspace, stream, true);
}
