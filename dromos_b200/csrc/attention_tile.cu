// Attention of many query rows per key head (prompts, pieces of prompts, groups of drafted tokens): both products on tcgen05.
//
// The mathematics is that of attention.cu: codes widened exactly to f16, scales outside in f32, t_j = c kscale (q . kcode_j) + log2 vscale,
// weights 2^(7 + t_j - m) that go to the second product in f16. m is a maximum the row had earlier: it moves when a larger one is more
// than 8 above it (2^15 is inside f16's range; a weight's smallest step, 2^-24, is 2^-31 of the largest weight or less), which spares
// the accumulator nearly every rescaling.
//
// A CTA takes 256 rows (128 where a head has 256 values) of one sequence and key head, a row being a new token and one of the heads that
// share the keys, in two tiles of 128: S = Q K^T of one tile runs while the other's softmax does. Roles: two groups of four warps each
// have a row per thread, read its scores from tensor memory and write the weights back over them, as the first operand of O += P V; one warp brings codes and scales in (bulk copies of 16 slots, so pages of any size); four warps widen keys and
// values (values transposed: both operands of both products lie along the summed dimension, in core matrices of 8 x 16 bytes); one
// thread issues the products. Values are stored with dim 4 l + j at n = 32 j + l, so that the four dims of a loaded word go to four
// conflict-free stores; results are put back in order as they are read.
//
// The (row block, key head, key tile) triples of the batch are dealt evenly over the SMs in order, with kBlockCost tiles' worth of time
// for beginning and ending a row block, so a CTA has part of at most two row blocks beside whole ones; parts are joined by a second
// kernel. The order is laid out by a kernel of one CTA.
#include <algorithm>

#include "attention.cuh"

namespace b200 {
namespace {

constexpr int kRowTile = 128;
constexpr int kSoftmaxWarps = 8, kWidenWarps = 4;
constexpr int kMmaWarp = kSoftmaxWarps + kWidenWarps, kLoadWarp = kMmaWarp + 1;
constexpr int kTileThreads = 32 * (kMmaWarp + 4);  // whole groups of four warps, each with its own share of the registers
// Registers a thread: 128 at launch (512 threads), 65,536 in all; 256 x kSoftmaxRegs + 128 x kWidenRegs + 128 x kMmaRegs are as many.
constexpr int kSoftmaxRegs = 176, kWidenRegs = 80, kMmaRegs = 80;
static_assert(256 * kSoftmaxRegs + 128 * kWidenRegs + 128 * kMmaRegs <= 512 * 128, "more registers than the launch has");
constexpr int kBlockCost = 6;
constexpr int kShift = 7;  // the largest weights are 2^7 .. 2^15
constexpr float kSlack = 8.0f, kUnshift = 0x1p-7f;

template <int D>
struct TileCfg {
  static constexpr int kRowTiles = D == 256 ? 1 : 2;
  static constexpr int kRows = kRowTiles * kRowTile;
  static constexpr int kKeys = D == 256 ? 64 : 128;  // keys of a tile
  static constexpr int kStages = 2, kRawStages = D == 64 ? 2 : 1, kScaleRing = 8;
  static constexpr int kQBytes = kRowTile * D * 2, kKvBytes = kKeys * D * 2, kRawBytes = kKeys * D;  // a tile: queries, keys or values, their codes
  static constexpr int kKOff = kRowTiles * kQBytes, kVOff = kKOff + kStages * kKvBytes, kRawOff = kVOff + kStages * kKvBytes;
  static constexpr int kScaleOff = kRawOff + 2 * kRawStages * kRawBytes, kScaleGroups = kKeys / 16;
  static constexpr int kBarOff = kScaleOff + kScaleRing * kScaleGroups * 16;
  static constexpr int kSmem = kBarOff + 512;
  static constexpr int kO = 256;  // first column of the sums in tensor memory; the scores (and the weights over them) begin at 0
  static_assert(kRowTiles * kKeys <= kO && kO + kRowTiles * D <= kTmemColumns, "tensor memory");
  static_assert(kSmem > 116 * 1024 && kSmem <= 226 * 1024, "one CTA per SM: it takes all of tensor memory");
  // A slot of the scales is written again kScaleRing tiles later: the copies are at most kRawStages + 1 tiles ahead of the widening,
  // which is at most kStages tiles ahead of the weights that use them.
  static_assert(kScaleRing >= kStages + kRawStages + 2, "scales");
};

struct BlockPlan {
  int s, row_block, tile0, tiles;
  int64_t before;  // the cost, in tiles, of the blocks before this one with all key heads
};
struct PlanHeader {
  int64_t total;
  int blocks;
  int pad;
};

struct TileArgs {
  AttentionArgs a;
  PlanHeader* header;
  BlockPlan* plan;
  float* partial;
  int capacity;  // blocks that `plan` has room for
  bool q_vec, out_whole;
};

// ---- the order of work -----------------------------------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(1024) attention_plan_kernel(const __grid_constant__ TileArgs T) {
  using C = TileCfg<D>;
  __shared__ int64_t sums[32];
  pdl_wait();
  const AttentionArgs& A = T.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto scan = [&](int64_t mine, int64_t& all) {  // the sum of the threads before
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int64_t x = sums[lane], below = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      const int64_t v = __shfl_sync(0xffffffffu, x, w);
      if (w < warp) below += v;
      all += v;
    }
    return below + incl - mine;
  };
  int64_t base = 0;
  for (int s0 = 0; s0 < A.kv.sequences; s0 += 1024) {
    int rows = 0;
    Span q{};
    if (s0 + tid < A.kv.sequences) {
      bool bad;
      q = span_of(A.kv, s0 + tid, bad);
      rows = q.n * A.group;
      if (bad) report_batch(A.kv);
    }
    const int blocks = rows > A.most ? (rows + C::kRows - 1) / C::kRows : 0;
    int64_t all;
    const int64_t at = base + scan(blocks, all);
    const int first = q.length - q.n;
    for (int b = 0; b < blocks; ++b) {
      if (at + b >= T.capacity) {  // sequences whose rows overlap: more blocks than there are rows
        report_batch(A.kv);
        break;
      }
      const int r0 = b * C::kRows, r1 = min(rows, r0 + C::kRows) - 1;
      const int low = first_seen(first + r0 / A.group + 1, A.window), past = first + r1 / A.group + 1;
      const int tile0 = low / C::kKeys;
      T.plan[at + b] = {s0 + tid, r0, tile0, max(1, tiles_before(past, C::kKeys) - tile0), 0};
    }
    base += all;
  }
  const int count = static_cast<int>(min(base, static_cast<int64_t>(T.capacity)));
  __syncthreads();
  int64_t before = 0;
  for (int b0 = 0; b0 < count; b0 += 1024) {
    const int64_t mine = b0 + tid < count ? static_cast<int64_t>(T.plan[b0 + tid].tiles + kBlockCost) * A.kv.kv_heads : 0;
    int64_t all;
    const int64_t at = before + scan(mine, all);
    if (b0 + tid < count) T.plan[b0 + tid].before = at;
    before += all;
  }
  if (tid == 0) *T.header = {before, count, 0};
}

// A CTA's way through its share.
struct Share {
  int64_t at, end, per;
  int block;
};
// The block that holds tile `at`; all threads of the CTA call it. found: shared.
__device__ __forceinline__ int find_block(const TileArgs& T, int count, int64_t total, int64_t at, int* found) {
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < count; b += blockDim.x) {
    const int64_t lo = T.plan[b].before, hi = b + 1 < count ? T.plan[b + 1].before : total;
    if (lo <= at && at < hi) *found = b;
  }
  __syncthreads();
  return *found;
}
struct Part {
  Span q;
  int s, head, row_block, rows, tile, tiles;  // tile: the first one, of the sequence's slots
  bool starts, whole;
  int past_high, see_low;
};
template <int ROWS>
__device__ __forceinline__ bool next_part(const TileArgs& T, Share& w, Part& p) {
  const AttentionArgs& A = T.a;
  const int heads = A.kv.kv_heads;
  for (;;) {
    if (w.at >= w.end) return false;
    BlockPlan b = T.plan[w.block];
    int cost = b.tiles + kBlockCost;
    while (w.at >= b.before + static_cast<int64_t>(cost) * heads) b = T.plan[++w.block], cost = b.tiles + kBlockCost;
    const int64_t in = w.at - b.before;
    p.s = b.s, p.row_block = b.row_block, p.head = static_cast<int>(divide(in, cost));
    const int64_t u0 = b.before + static_cast<int64_t>(p.head) * cost;
    const int c0 = static_cast<int>(w.at - u0), c1 = static_cast<int>(min(static_cast<int64_t>(cost), w.end - u0));
    w.at = u0 + c1;
    const int t0 = max(0, c0 - kBlockCost);
    p.tiles = max(0, c1 - kBlockCost) - t0;
    if (p.tiles == 0) continue;
    p.tile = b.tile0 + t0;
    p.starts = t0 == 0, p.whole = t0 == 0 && p.tiles == b.tiles;
    bool bad;
    p.q = span_of(A.kv, b.s, bad);
    p.rows = min(ROWS, p.q.n * A.group - b.row_block);
    const int first = p.q.length - p.q.n;
    p.past_high = max(0, first + (b.row_block + p.rows - 1) / A.group + 1);
    p.see_low = first_seen(first + b.row_block / A.group + 1, A.window);
    return true;
  }
}

// ---- tensor memory and products -----------------------------------------------------------------------------------------------
// Reads of tensor memory with their wait in one statement: the registers fill behind the compiler's back, and a copy that it made of
// them between the two would have what was there before.
__device__ __forceinline__ void tmem_ld_2x32(uint32_t taddr, uint32_t (&r)[2][32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0][0]), "=r"(r[0][1]), "=r"(r[0][2]), "=r"(r[0][3]), "=r"(r[0][4]), "=r"(r[0][5]), "=r"(r[0][6]), "=r"(r[0][7]), "=r"(r[0][8]), "=r"(r[0][9]), "=r"(r[0][10]), "=r"(r[0][11]), "=r"(r[0][12]), "=r"(r[0][13]), "=r"(r[0][14]), "=r"(r[0][15]), "=r"(r[0][16]), "=r"(r[0][17]), "=r"(r[0][18]), "=r"(r[0][19]), "=r"(r[0][20]), "=r"(r[0][21]), "=r"(r[0][22]), "=r"(r[0][23]), "=r"(r[0][24]), "=r"(r[0][25]), "=r"(r[0][26]), "=r"(r[0][27]), "=r"(r[0][28]), "=r"(r[0][29]), "=r"(r[0][30]), "=r"(r[0][31]),
        "=r"(r[1][0]), "=r"(r[1][1]), "=r"(r[1][2]), "=r"(r[1][3]), "=r"(r[1][4]), "=r"(r[1][5]), "=r"(r[1][6]), "=r"(r[1][7]), "=r"(r[1][8]), "=r"(r[1][9]), "=r"(r[1][10]), "=r"(r[1][11]), "=r"(r[1][12]), "=r"(r[1][13]), "=r"(r[1][14]), "=r"(r[1][15]), "=r"(r[1][16]), "=r"(r[1][17]), "=r"(r[1][18]), "=r"(r[1][19]), "=r"(r[1][20]), "=r"(r[1][21]), "=r"(r[1][22]), "=r"(r[1][23]), "=r"(r[1][24]), "=r"(r[1][25]), "=r"(r[1][26]), "=r"(r[1][27]), "=r"(r[1][28]), "=r"(r[1][29]), "=r"(r[1][30]), "=r"(r[1][31])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_4x16(uint32_t taddr, uint32_t step, uint32_t (&r)[4][16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%65];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47}, [%66];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%67];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0][0]), "=r"(r[0][1]), "=r"(r[0][2]), "=r"(r[0][3]), "=r"(r[0][4]), "=r"(r[0][5]), "=r"(r[0][6]), "=r"(r[0][7]), "=r"(r[0][8]), "=r"(r[0][9]), "=r"(r[0][10]), "=r"(r[0][11]), "=r"(r[0][12]), "=r"(r[0][13]), "=r"(r[0][14]), "=r"(r[0][15]),
        "=r"(r[1][0]), "=r"(r[1][1]), "=r"(r[1][2]), "=r"(r[1][3]), "=r"(r[1][4]), "=r"(r[1][5]), "=r"(r[1][6]), "=r"(r[1][7]), "=r"(r[1][8]), "=r"(r[1][9]), "=r"(r[1][10]), "=r"(r[1][11]), "=r"(r[1][12]), "=r"(r[1][13]), "=r"(r[1][14]), "=r"(r[1][15]),
        "=r"(r[2][0]), "=r"(r[2][1]), "=r"(r[2][2]), "=r"(r[2][3]), "=r"(r[2][4]), "=r"(r[2][5]), "=r"(r[2][6]), "=r"(r[2][7]), "=r"(r[2][8]), "=r"(r[2][9]), "=r"(r[2][10]), "=r"(r[2][11]), "=r"(r[2][12]), "=r"(r[2][13]), "=r"(r[2][14]), "=r"(r[2][15]),
        "=r"(r[3][0]), "=r"(r[3][1]), "=r"(r[3][2]), "=r"(r[3][3]), "=r"(r[3][4]), "=r"(r[3][5]), "=r"(r[3][6]), "=r"(r[3][7]), "=r"(r[3][8]), "=r"(r[3][9]), "=r"(r[3][10]), "=r"(r[3][11]), "=r"(r[3][12]), "=r"(r[3][13]), "=r"(r[3][14]), "=r"(r[3][15])
      : "r"(taddr), "r"(taddr + step), "r"(taddr + 2 * step), "r"(taddr + 3 * step)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem descriptor], f16 operands; the descriptor in halves, as umma_ss_halves has them.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 db; setp.ne.u32 p, %5, 0; mov.b64 db, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p; }" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One arrival for a warp, after all of its lanes: 128 arrivals of a role's threads take their turns at the barrier for as long as a
// tile's products take.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
// A wait of a whole warp: where one lane gives up all of them do.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* status) { return __all_sync(0xffffffffu, tc_wait(bar, parity, status)); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// A thread's query row into its row of the core matrices, times the power of two that brings it into f16's range (and the sign of the
// softmax's scale); returns the factor of its scores. Read twice: once for its largest magnitude. Rows past the end are zeros.
template <int D, int DTYPE, bool VEC>
__device__ __forceinline__ float load_query(const AttentionArgs& A, int64_t src, bool there, uint32_t to, float sign) {
  constexpr int RUN = DTYPE == LX_BF16 && D <= 128 ? D : 32;  // values at once
  constexpr int PIECES = RUN / 8;
  float most = 0.0f, up = 1.0f;
  uint4 raw[PIECES][DTYPE == LX_BF16 ? 1 : 2];
  auto load = [&](int d0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if constexpr (VEC) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(A.q) + (src + d0 + 8 * i) * (DTYPE == LX_BF16 ? 2 : 4));
        raw[i][0] = p[0];
        if constexpr (DTYPE == LX_F32) raw[i][1] = p[1];
      } else {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(load_f32(A.q, A.q_dtype, src + d0 + 8 * i + j));
        raw[i][0] = make_uint4(w[0], w[1], w[2], w[3]), raw[i][1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  };
  auto values = [&](int i, float (&v)[8]) {
    const uint32_t w[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
    if constexpr (DTYPE == LX_BF16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const uint32_t z[4] = {raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]), v[4 + j] = __uint_as_float(z[j]);
    }
  };
#pragma unroll 1
  for (int d0 = 0; d0 < D; d0 += RUN) {
    load(d0);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      float v[8];
      values(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[j]));
    }
  }
  up = f16_scale(most);
  const float by = there ? up * sign : 0.0f;
#pragma unroll 1
  for (int d0 = 0; d0 < D; d0 += RUN) {
    if constexpr (RUN < D) load(d0);
#pragma unroll
    for (int h = 0; h < RUN / 32; ++h) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[8];
        values(4 * h + i, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 x = __floats2half2_rn(there ? v[2 * j] * by : 0.0f, there ? v[2 * j + 1] * by : 0.0f);
          w[4 * i + j] = *reinterpret_cast<const uint32_t*>(&x);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sts128(to + (d0 / 8 + 4 * h + i) * (kRowTile * 16), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  return A.scale_log2 * sign / up;
}

// Sixteen results, or sums, of a row; whole: they lie on 32 bytes.
__device__ __forceinline__ void store8(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]),
               "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void store_out16(const AttentionArgs& A, int64_t at, const float (&v)[16], float factor, bool whole) {
  if (whole) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = f32_to_bf16_bits(v[2 * i] * factor) | f32_to_bf16_bits(v[2 * i + 1] * factor) << 16;
    store8(A.out + at, w);
  } else {
#pragma unroll
    for (int i = 0; i < 16; i += 4) store_out(A, at + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), factor);
  }
}

// ---- one row's softmax over a tile of scores -------------------------------------------------------------------------------------
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// Two f32 at once.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// EDGE: some row of the warps does not see all of a tile; this one sees its slots lo <= j < hi. The loops stay rolled and read the
// scores from tensor memory 64 at a time: 128 scores in registers and straight code for them ran at the rate of the instruction
// cache. (The next scores read while the last ones are worked on would hide more, but nothing may stand between a read and its wait.)
template <bool EDGE>
__device__ __forceinline__ void mask_scores(uint32_t (&u)[32], int at, int lo, int hi) {
  if constexpr (EDGE) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (at + j >= hi || at + j < lo) u[j] = 0xff800000u;
  }
}
// The largest t of a tile.
template <bool EDGE, int KT>
__device__ __forceinline__ float tile_top(uint32_t s_tmem, const float4* sc, float f, int lo, int hi) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c0 = 0; c0 < KT / 32; c0 += 2) {
    uint32_t u[2][32];
    tmem_ld_2x32(s_tmem + 32 * c0, u);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = c0 + e;
      mask_scores<EDGE>(u[e], 32 * c, lo, hi);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float a = __uint_as_float(u[e][16 * h]), b = __uint_as_float(u[e][16 * h + 1]);
#pragma unroll
        for (int j = 2; j < 14; j += 4) {
          a = max3(a, __uint_as_float(u[e][16 * h + j]), __uint_as_float(u[e][16 * h + j + 1]));
          b = max3(b, __uint_as_float(u[e][16 * h + j + 2]), __uint_as_float(u[e][16 * h + j + 3]));
        }
        const float most = fmaxf(max3(a, __uint_as_float(u[e][16 * h + 14]), __uint_as_float(u[e][16 * h + 15])), b);
        const float4 g = sc[2 * c + h];
        const float t = fmaf(most, f * g.x, g.y);
        top = fmaxf(top, EDGE && most == -INFINITY ? -INFINITY : t);
      }
    }
  }
  return top;
}
// The weights of a tile, in f16 over its scores; returns what the sum of weights gains.
template <bool EDGE, int KT>
__device__ __forceinline__ float tile_weights(uint32_t s_tmem, const float4* sc, float f, float from, int lo, int hi) {
  float l = 0.0f;
#pragma unroll 1
  for (int c0 = 0; c0 < KT / 32; c0 += 2) {
    uint32_t u[2][32];
    tmem_ld_2x32(s_tmem + 32 * c0, u);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = c0 + e;
      uint32_t w[16];
      mask_scores<EDGE>(u[e], 32 * c, lo, hi);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 g = sc[2 * c + h];
        const float by = f * g.x, add = g.y - from;
        const uint64_t by2 = pack2(by, by), add_2 = pack2(add, add);
        uint64_t sum2 = pack2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float u0 = __uint_as_float(u[e][16 * h + j]), u1 = __uint_as_float(u[e][16 * h + j + 1]);
          float x0, x1;
          unpack2(fma2(pack2(u0, u1), by2, add_2), x0, x1);
          if constexpr (EDGE) {  // what a row does not see stays -inf, whatever the scale
            x0 = u0 == -INFINITY ? u0 : x0;
            x1 = u1 == -INFINITY ? u1 : x1;
          }
          x0 = exp2_fast(x0), x1 = exp2_fast(x1);
          sum2 = add2(sum2, pack2(x0, x1));
          const __half2 x = __floats2half2_rn(x0, x1);
          w[8 * h + j / 2] = *reinterpret_cast<const uint32_t*>(&x);
        }
        float a, b;
        unpack2(sum2, a, b);
        // a row that sees nothing of a page whose scale is not a number: nothing, and not 0 x NaN
        l = EDGE && a + b == 0.0f ? l : fmaf(a + b, g.z, l);
      }
      tmem_st16(s_tmem + 16 * c, w);
    }
  }
  return l;
}

template <bool kInt8, int D>
__global__ void __launch_bounds__(kTileThreads, 1) attention_tile_kernel(const __grid_constant__ TileArgs T) {
  using C = TileCfg<D>;
  constexpr int RT = C::kRowTiles, KT = C::kKeys;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t tmem_slot;
  __shared__ int found;
  const AttentionArgs& A = T.a;
  const KvView& V = A.kv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NS = C::kStages, RS = C::kRawStages;
  const uint32_t q_base = smem_u32(smem), k_base = q_base + C::kKOff, v_base = q_base + C::kVOff, raw_base = q_base + C::kRawOff, bars = q_base + C::kBarOff;
  float4* const scales = reinterpret_cast<float4*>(smem + C::kScaleOff);  // [ring][group of 16 slots]: kscale, log2 vscale, 2^-shift / vscale, 1 with codes
  // per row tile: queries in, scores done, weights in, sums done; per stage: keys and values in and read; codes in and read (keys' two
  // stages, values' two)
  const uint32_t q_full = bars, s_full = bars + 16, p_full = bars + 32, o_full = bars + 48, raw_full = bars + 64, raw_empty = bars + 96, k_full = bars + 128,
                 k_empty = k_full + 8 * NS, v_full = k_empty + 8 * NS, v_empty = v_full + 8 * NS;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 4);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(o_full + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(raw_full + 8 * i, 1);
      mbar_init(raw_empty + 8 * i, kWidenWarps);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(k_full + 8 * i, kWidenWarps);
      mbar_init(k_empty + 8 * i, 1);
      mbar_init(v_full + 8 * i, kWidenWarps);
      mbar_init(v_empty + 8 * i, 1);
    }
    mbar_init_fence();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_slot), kTmemColumns);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  Share share;
  {
    const PlanHeader h = *T.header;
    share.per = max(static_cast<int64_t>(A.min_tiles), divide(h.total + gridDim.x - 1, gridDim.x));
    share.at = blockIdx.x * share.per;
    share.end = min(h.total, share.at + share.per);
    share.block = find_block(T, h.blocks, h.total, share.at, &found);
    if (share.block < 0) share.end = share.at;
  }
  Part p;
  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    // ================================ the products ================================
    if (warp == kMmaWarp) {
      // The whole warp goes through the loops, one lane issues: what the instructions take is then the same in all lanes and stays in
      // uniform registers. (One lane alone in the loops took 115 cycles for each product, whose own time is 66.)
      const uint32_t idesc_s = (1u << 4) | (static_cast<uint32_t>(KT >> 3) << 17) | (static_cast<uint32_t>(kRowTile >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(kRowTile >> 4) << 24);
      // descriptors of core matrices (smem_desc): address and the step along the summed dimension, both in 16 bytes, below; the step of
      // 128 bytes between groups of 8 rows above
      const uint32_t desc_hi = (128u >> 4) | (1u << 14);
      uint32_t kn = 0, vn = 0, qn[2] = {0, 0}, pn[2] = {0, 0};
      auto scores = [&](int rt) {
        const uint32_t qa = (q_base + rt * C::kQBytes) >> 4 | kRowTile << 16, kb = (k_base + kn % NS * C::kKvBytes) >> 4 | KT << 16;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            umma_ss_halves<kActF16>(tmem + rt * KT, qa + i * 2 * kRowTile, desc_hi, kb + i * 2 * KT, desc_hi, idesc_s, i > 0);
          umma_commit(s_full + 8 * rt);
        }
        __syncwarp();
      };
      bool more_parts = next_part<C::kRows>(T, share, p), ok = true;
      while (ok && more_parts) {
        const int tiles_of_rows = p.rows > kRowTile ? 2 : 1, tiles = p.tiles;
        if (!warp_wait(k_full + 8 * (kn % NS), kn / NS & 1, V.status)) break;
        for (int rt = 0; rt < tiles_of_rows && ok; ++rt) {
          ok = warp_wait(q_full + 8 * rt, qn[rt]++ & 1, V.status);
          if (!ok) break;
          tc_fence_after();
          scores(rt);
        }
        if (!ok) break;
        if (elect_one()) umma_commit(k_empty + 8 * (kn % NS));
        __syncwarp();
        ++kn;
        more_parts = next_part<C::kRows>(T, share, p);
        for (int i = 0; i < tiles && ok; ++i) {
          const bool more = i + 1 < tiles;
          for (int rt = 0; rt < tiles_of_rows; ++rt) {
            if ((rt == 0 && !warp_wait(v_full + 8 * (vn % NS), vn / NS & 1, V.status)) || !warp_wait(p_full + 8 * rt, pn[rt] & 1, V.status) ||
                (rt == 0 && more && !warp_wait(k_full + 8 * (kn % NS), kn / NS & 1, V.status))) {
              ok = false;
              break;
            }
            ++pn[rt];
            tc_fence_after();
            const uint32_t vb = (v_base + vn % NS * C::kKvBytes) >> 4 | D << 16;
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < KT / 16; ++j)
                umma_ts(tmem + C::kO + rt * D, tmem + rt * KT + 8 * j, vb + j * 2 * D, desc_hi, idesc_o, i > 0 || j > 0);
              if (!more) umma_commit(o_full + 8 * rt);
            }
            __syncwarp();
            if (more) scores(rt);
          }
          if (!ok) break;
          if (elect_one()) {
            umma_commit(v_empty + 8 * (vn % NS));
            if (more) umma_commit(k_empty + 8 * (kn % NS));
          }
          __syncwarp();
          ++vn;
          kn += more;
        }
      }
    }
    else if (warp == kLoadWarp) {
      // codes and scales: lane g has the slots 16 g .. 16 g + 15 of a tile
      const int log_p = __ffs(V.page_tokens) - 1, page_mask = V.page_tokens - 1;
      uint32_t n = 0, sent[2] = {0, 0};
      bool ok = true;
      while (ok && next_part<C::kRows>(T, share, p)) {
        for (int i = 0; i < p.tiles && ok; ++i, ++n) {
          const int slot = (p.tile + i) * KT + 16 * (lane & (C::kScaleGroups - 1));
          int page = -2;  // nothing that any row sees
          if (lane < C::kScaleGroups && slot < p.past_high && slot > p.see_low - 16) {
            page = page_of(V, p.s, slot >> log_p);
            if (page < 0) report_batch(V);
          }
          const int64_t src = max(page, 0) * V.page_stride + (static_cast<int64_t>(p.head) * V.page_tokens + (slot & page_mask)) * D;
          if (lane < C::kScaleGroups) {
            const float nan = __uint_as_float(0x7fffffffu);
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // the last one: whether there are codes
            if (page == -1) s = make_float4(nan, nan, nan, 0.0f);
            if (page >= 0) {
              const int64_t at = static_cast<int64_t>(page) * V.kv_heads + p.head;
              const float v = V.v_scale[at], vs = v < 0x1p-100f ? 0x1p-100f : v;
              s = make_float4(V.k_scale[at], __log2f(vs), kUnshift / vs, 1.0f);
            }
            scales[n % C::kScaleRing * C::kScaleGroups + lane] = s;
          }
          for (int kv = 0; kv < 2 && ok; ++kv) {
            const uint32_t at = RS * kv + n % RS;
            ok = warp_wait(raw_empty + 8 * at, (n / RS & 1) ^ 1, V.status);
            if (!ok) break;
            __syncwarp();
            const uint32_t copies = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) mbar_arrive_expect_tx(raw_full + 8 * at, __popc(copies) * 16 * D);
            __syncwarp();
            if (page >= 0) bulk_g2s(raw_base + at * C::kRawBytes + 16 * lane * D, (kv ? V.v : V.k) + src, 16 * D, raw_full + 8 * at);
            ++sent[kv];
          }
        }
      }
      // copies in flight end before the CTA does: the last ones of each kind
      for (int kv = 0; kv < 2; ++kv)
        for (uint32_t i = sent[kv] > RS ? sent[kv] - RS : 0; i < sent[kv]; ++i) tc_wait(raw_full + 8 * (RS * kv + i % RS), i / RS & 1, V.status);
    }
  } else if (warp < kSoftmaxWarps) {
    // ================================ softmax: a row per thread ================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int rt = warp >> 2, row = tid & (kRowTile - 1);
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_tmem = tmem + lanes + rt * KT, o_tmem = tmem + lanes + C::kO + rt * D;
    uint32_t sn = 0, on = 0, tiles_done = 0;
    bool ok = true;
    const float sign = A.scale_log2 < 0.0f ? -1.0f : 1.0f;
    Part next;
    bool more_parts = next_part<C::kRows>(T, share, next);
    float f = 0.0f;
    // the queries of a part, as soon as the scores of the part before are done
    auto queries = [&]() {
      const int r = next.row_block + rt * kRowTile + row;
      const bool there = r < next.row_block + next.rows;
      const int q = there ? r : next.row_block + next.rows - 1;  // a row that is there, for the loads
      const int64_t src = (next.q.row0 + q / A.group) * A.ld_q + (static_cast<int64_t>(next.head) * A.group + q % A.group) * D;
      const uint32_t to = q_base + rt * C::kQBytes + row * 16;
      if (T.q_vec && A.q_dtype == LX_BF16) f = load_query<D, LX_BF16, true>(A, src, there, to, sign);
      else if (T.q_vec) f = load_query<D, LX_F32, true>(A, src, there, to, sign);
      else f = load_query<D, -1, false>(A, src, there, to, sign);
      proxy_fence();
      warp_arrive(q_full + 8 * rt);
    };
    auto prefetch = [&]() {  // the same row into L2, a tile's time and more ahead
      const int q = min(next.row_block + rt * kRowTile + row, next.row_block + next.rows - 1), bytes = A.q_dtype == LX_BF16 ? 2 : 4;
      const uint8_t* src = static_cast<const uint8_t*>(A.q) +
                           ((next.q.row0 + q / A.group) * A.ld_q + (static_cast<int64_t>(next.head) * A.group + q % A.group) * D) * bytes;
      for (int b = 0; b < D * bytes; b += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + b));
    };
    auto takes = [&](const Part& x) { return rt < RT && (rt == 0 || x.rows > kRowTile); };
    if (more_parts && takes(next)) queries();
    while (ok && more_parts) {
      p = next;
      const int first = p.q.length - p.q.n, row0 = p.row_block + rt * kRowTile;
      if (!takes(p)) {
        tiles_done += p.tiles;
        more_parts = next_part<C::kRows>(T, share, next);
        if (more_parts && takes(next)) queries();
        continue;
      }
      const float f_now = f;
      const int r = row0 + row;
      const bool valid = r < p.row_block + p.rows;
      const int past = valid ? first + r / A.group + 1 : 0;
      const int past_low = first + row0 / A.group + 1, past_last = first + (min(row0 + kRowTile, p.row_block + p.rows) - 1) / A.group + 1;
      const int see_all = first_seen(past_last, A.window), low = first_seen(past, A.window);
      float m = -INFINITY, l = 0.0f;
      for (int i = 0; i < p.tiles; ++i) {
        const int key0 = (p.tile + i) * KT;
        const float4* sc = scales + (tiles_done + i) % C::kScaleRing * C::kScaleGroups;
        if (!warp_wait(s_full + 8 * rt, sn & 1, V.status)) {
          ok = false;
          break;
        }
        ++sn;
        tc_fence_after();
        const bool edge = key0 > past_low - KT || key0 < see_all;
        const int lo = low - key0, hi = past - key0;
        const float top = edge ? tile_top<true, KT>(s_tmem, sc, f_now, lo, hi) : tile_top<false, KT>(s_tmem, sc, f_now, lo, hi);
        const bool higher = top > m + kSlack;  // at first m is -inf
        if (__any_sync(0xffffffffu, higher)) {
          const float shrink = higher ? exp2_fast(m - top) : 1.0f;
          m = higher ? top : m;
          if (i > 0) {
            l *= shrink;
            // the scores of this tile came after the product of the tile before: nothing is at work on these sums
#pragma unroll 1
            for (int c = 0; c < D; c += 64) {
              uint32_t v[4][16];
              tmem_ld_4x16(o_tmem + c, 16, v);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[e][j] = __float_as_uint(__uint_as_float(v[e][j]) * shrink);
                tmem_st16(o_tmem + c + 16 * e, v[e]);
              }
            }
          }
        }
        const float from = (m == -INFINITY ? 0.0f : m) - kShift;
        l += edge ? tile_weights<true, KT>(s_tmem, sc, f_now, from, lo, hi) : tile_weights<false, KT>(s_tmem, sc, f_now, from, lo, hi);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(p_full + 8 * rt);
        if (i == 0) {
          more_parts = next_part<C::kRows>(T, share, next);
          if (more_parts && takes(next)) prefetch();
        }
      }
      tiles_done += p.tiles;
      if (!ok) break;
      if (more_parts && takes(next)) queries();
      if (!warp_wait(o_full + 8 * rt, on & 1, V.status)) {
        ok = false;
        break;
      }
      ++on;
      tc_fence_after();
      float* const part = T.partial + (2 * static_cast<int64_t>(blockIdx.x) + p.starts) * (C::kRows * (D + 2));
      const int pr = rt * kRowTile + row;
      const int64_t out_row = (p.q.row0 + r / A.group) * A.ld_out + (static_cast<int64_t>(p.head) * A.group + r % A.group) * D;
      const float factor = l == 0.0f ? 0.0f : kUnshift / l;
      if (!p.whole && valid) part[pr] = m, part[C::kRows + pr] = l;
      constexpr int W = D < 128 ? D / 4 : 32;  // dim 4 l + j of a run of 4 W lies at n = W j + l
#pragma unroll
      for (int h = 0; h < D / (4 * W); ++h)
#pragma unroll
        for (int k = 0; k < W / 16; ++k) {
          uint32_t u[4][16];
          tmem_ld_4x16(o_tmem + 4 * W * h + 16 * k, W, u);
          if (valid) {
#pragma unroll
            for (int q = 0; q < 16; q += 4) {
              const int d = 4 * (W * h + 16 * k + q);
              float v[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(u[e & 3][q + e / 4]);
              if (p.whole) {
                store_out16(A, out_row + d, v, factor, T.out_whole);
              } else {
                uint32_t w[8];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(v[8 * z + e]);
                  store8(part + 2 * C::kRows + pr * D + d + 8 * z, w);
                }
              }
            }
          }
          __syncwarp();
        }
      tc_fence_before();  // the next block's products come after this thread's next arrival
    }
  } else {
    // ================================ keys and values, widened ================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs));
    const int w4 = warp & 3;
    constexpr int WK = KT / 4;  // slots of a tile that one warp has
    uint32_t n = 0;
    bool ok = true;
    while (ok && next_part<C::kRows>(T, share, p)) {
      for (int i = 0; i < p.tiles && ok; ++i, ++n) {
        const int slot0 = (p.tile + i) * KT;
        const uint8_t* const raw_k = smem + C::kRawOff + n % RS * C::kRawBytes;
        const uint8_t* const raw_v = raw_k + RS * C::kRawBytes;
        // a word of slot j: all of it, or 0 where no row sees the slot (what it holds may be no numbers) or nothing was copied
        const float4* const sc = scales + n % C::kScaleRing * C::kScaleGroups;
        auto keep = [&](int j) {
          const bool there = slot0 + j < p.past_high && slot0 + j >= p.see_low && sc[j / 16].w != 0.0f;
          return there ? 0xffffffffu : 0u;
        };
        // keys. Lane i of eight takes key i of a run, and of its pieces of 16 bytes another one than its neighbours: neither the reads of
        // rows nor the writes of core matrices meet in a bank. The codes are taken into registers first, so that the next ones come
        // while these are widened.
        if (!warp_wait(raw_full + 8 * (n % RS), n / RS & 1, V.status)) {
          ok = false;
          break;
        }
        bool edge = slot0 < p.see_low || slot0 > p.past_high - KT;
#pragma unroll
        for (int g = 0; g < C::kScaleGroups; ++g) edge |= sc[g].w == 0.0f;
        {
          constexpr int PIECES = D / 16, RUNS = WK / 8;
          const int key8 = lane & 7;
          auto piece_at = [&](int b) { return ((D == 64 ? key8 >> 1 : key8) + 4 * b + (lane >> 3)) & (PIECES - 1); };
          uint4 x[RUNS][PIECES / 4];
#pragma unroll
          for (int a = 0; a < RUNS; ++a)
#pragma unroll
            for (int b = 0; b < PIECES / 4; ++b) x[a][b] = *reinterpret_cast<const uint4*>(raw_k + (w4 * WK + 8 * a + key8) * D + 16 * piece_at(b));
          if (edge) {
#pragma unroll
            for (int a = 0; a < RUNS; ++a) {
              const uint32_t k = keep(w4 * WK + 8 * a + key8);
#pragma unroll
              for (int b = 0; b < PIECES / 4; ++b) x[a][b] = make_uint4(x[a][b].x & k, x[a][b].y & k, x[a][b].z & k, x[a][b].w & k);
            }
          }
          proxy_fence();  // the codes have arrived in registers before a copy may write over them (without it some had not)
          warp_arrive(raw_empty + 8 * (n % RS));
          if (!warp_wait(k_empty + 8 * (n % NS), (n / NS & 1) ^ 1, V.status)) {
            ok = false;
            break;
          }
          const uint32_t dst = k_base + n % NS * C::kKvBytes;
#pragma unroll
          for (int a = 0; a < RUNS; ++a)
#pragma unroll
            for (int b = 0; b < PIECES / 4; ++b) {
              const uint32_t word[4] = {x[a][b].x, x[a][b].y, x[a][b].z, x[a][b].w};
              uint32_t o[8];
#pragma unroll
              for (int c = 0; c < 4; ++c) halves<kInt8>(word[c], o[2 * c], o[2 * c + 1]);
              const uint32_t to = dst + 2 * piece_at(b) * (KT * 16) + (w4 * WK + 8 * a + key8) * 16;
              sts128(to, o[0], o[1], o[2], o[3]);
              sts128(to + KT * 16, o[4], o[5], o[6], o[7]);
            }
        }
        proxy_fence();
        warp_arrive(k_full + 8 * (n % NS));
        // values: lane: four dims of eight keys; with 64 values per head the half warps have a run of eight keys each
        if (!warp_wait(raw_full + 8 * (RS + n % RS), n / RS & 1, V.status)) {
          ok = false;
          break;
        }
        {
          constexpr int LANES = D < 128 ? D / 4 : 32, AT_ONCE = 32 / LANES, RUNS = WK / (8 * AT_ONCE), HALVES = D > 128 ? 2 : 1;
          const int l = lane % LANES, sub = lane / LANES;
          uint32_t x[RUNS][HALVES][8];
#pragma unroll
          for (int a = 0; a < RUNS; ++a) {
            const int run = w4 * (WK / 8) + a * AT_ONCE + sub;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
              for (int j = 0; j < 8; ++j) x[a][h][j] = *reinterpret_cast<const uint32_t*>(raw_v + (8 * run + j) * D + 128 * h + 4 * l);
          }
          if (edge) {
#pragma unroll
            for (int a = 0; a < RUNS; ++a)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t k = keep(8 * (w4 * (WK / 8) + a * AT_ONCE + sub) + j);
#pragma unroll
                for (int h = 0; h < HALVES; ++h) x[a][h][j] &= k;
              }
          }
          proxy_fence();
          warp_arrive(raw_empty + 8 * (RS + n % RS));
          if (!warp_wait(v_empty + 8 * (n % NS), (n / NS & 1) ^ 1, V.status)) {
            ok = false;
            break;
          }
          const uint32_t dst = v_base + n % NS * C::kKvBytes;
#pragma unroll
          for (int a = 0; a < RUNS; ++a)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              uint32_t o[4][4];  // dim, pair of keys
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                halves<kInt8>(__byte_perm(x[a][h][2 * j], x[a][h][2 * j + 1], 0x5140), o[0][j], o[1][j]);
                halves<kInt8>(__byte_perm(x[a][h][2 * j], x[a][h][2 * j + 1], 0x7362), o[2][j], o[3][j]);
              }
              const uint32_t to = dst + (w4 * (WK / 8) + a * AT_ONCE + sub) * (D * 16) + (128 * h + l) * 16;
#pragma unroll
              for (int d = 0; d < 4; ++d) sts128(to + d * LANES * 16, o[d][0], o[d][1], o[d][2], o[d][3]);
            }
        }
        proxy_fence();
        warp_arrive(v_full + 8 * (n % NS));
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemColumns);
}

// Joins the row blocks that several CTAs shared: CTA (i, j) rows of the one that began in share i and went on into the next.
template <int D>
__global__ void __launch_bounds__(256) attention_tile_join_kernel(const __grid_constant__ TileArgs T, int shares) {
  using C = TileCfg<D>;
  __shared__ int found;
  pdl_wait();
  const AttentionArgs& A = T.a;
  const PlanHeader h = *T.header;
  if (A.pad) zero_rows_from(A, A.kv.starts[A.kv.sequences], D, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
  const int64_t per = max(static_cast<int64_t>(A.min_tiles), (h.total + shares - 1) / shares), at = (blockIdx.x + 1) * per;
  const int block = find_block(T, h.blocks, h.total, at, &found);
  if (block < 0) return;
  const BlockPlan b = T.plan[block];
  const int cost = b.tiles + kBlockCost, head = static_cast<int>((at - b.before) / cost);
  const int64_t u1 = b.before + static_cast<int64_t>(head + 1) * cost, first_tile = u1 - b.tiles;
  if (first_tile >= at || first_tile < at - per) return;  // nothing crosses this border, or it began earlier
  const int last = static_cast<int>((u1 - 1) / per);
  bool bad;
  const Span q = span_of(A.kv, b.s, bad);
  const int rows = min(C::kRows, q.n * A.group - b.row_block);
  for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * (D / 4); i += gridDim.y * 256) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    auto slot = [&](int p) { return T.partial + (2 * static_cast<int64_t>(p) + (p == static_cast<int>(blockIdx.x))) * (C::kRows * (D + 2)); };
    float top = -INFINITY, sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int p = blockIdx.x; p <= last; ++p) top = fmaxf(top, slot(p)[r]);
#pragma unroll 8
    for (int p = blockIdx.x; p <= last; ++p) {
      const float* src = slot(p);
      const float mp = src[r], lp = src[C::kRows + r];
      const float4 op = *reinterpret_cast<const float4*>(src + 2 * C::kRows + r * D + d);
      const float y = mp == -INFINITY ? 0.0f : exp2_fast(mp - top);
      sum += mp == -INFINITY ? lp : lp * y;
      v.x = fmaf(op.x, y, v.x), v.y = fmaf(op.y, y, v.y), v.z = fmaf(op.z, y, v.z), v.w = fmaf(op.w, y, v.w);
    }
    const int rr = b.row_block + r;
    store_out(A, (q.row0 + rr / A.group) * A.ld_out + (static_cast<int64_t>(head) * A.group + rr % A.group) * D + d, v, sum == 0.0f ? 0.0f : kUnshift / sum);
  }
}

struct TileLayout {
  int64_t plan, partial, total;
  int capacity;
};
TileLayout tile_layout(int head_dim, int kv_heads, int group, int tokens, int sequences) {
  const int rows = head_dim == 256 ? kRowTile : 2 * kRowTile;
  TileLayout L;
  // a block holds more than 0 rows: whole blocks of all rows, and a last one of each sequence
  L.capacity = static_cast<int>(static_cast<int64_t>(tokens) * group / rows + sequences);
  L.plan = 64;
  L.partial = (L.plan + static_cast<int64_t>(L.capacity) * static_cast<int64_t>(sizeof(BlockPlan)) + 255) / 256 * 256;
  L.total = L.partial + static_cast<int64_t>(sm_count()) * 2 * rows * (head_dim + 2) * 4;
  return L;
}

template <bool kInt8, int D>
int launch_tile(const TileArgs& T, cudaStream_t stream) {
  using C = TileCfg<D>;
  const unsigned grid = static_cast<unsigned>(sm_count());
  if (grid == 0) return kNotSupported;
  auto kernel = attention_tile_kernel<kInt8, D>;
  if (int e = allow_big_smem<kInt8 * 4 + (D == 64 ? 0 : D == 128 ? 1 : 2)>(kernel)) return e;
  if (int e = launch_kernel(attention_plan_kernel<D>, dim3(1), dim3(1024), 0, stream, T)) return e;
  if (int e = launch_kernel(kernel, dim3(grid), dim3(kTileThreads), C::kSmem, stream, T)) return e;
  return launch_kernel(attention_tile_join_kernel<D>, dim3(grid, 8), dim3(256), 0, stream, T, static_cast<int>(grid));
}

}  // namespace

int64_t tile_attention_workspace(int head_dim, int kv_heads, int group, int tokens, int sequences) {
  return tile_layout(head_dim, kv_heads, group, tokens, sequences).total;
}

int tile_attention(AttentionArgs A, int head_dim, bool int8, int limit, void* workspace, cudaStream_t stream) {
  const TileLayout L = tile_layout(head_dim, A.kv.kv_heads, A.group, A.kv.tokens, A.kv.sequences);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  TileArgs T;
  T.a = A;
  T.a.most = limit;
  T.a.min_tiles = 2 * kBlockCost + 2;
  T.header = reinterpret_cast<PlanHeader*>(ws), T.plan = reinterpret_cast<BlockPlan*>(ws + L.plan), T.partial = reinterpret_cast<float*>(ws + L.partial);
  T.capacity = L.capacity;
  T.out_whole = aligned(A.out, 32) && A.ld_out % 16 == 0;
  T.q_vec = aligned(A.q, 16) && A.ld_q % (A.q_dtype == LX_BF16 ? 8 : 4) == 0;
  switch (head_dim) {
    case 64: return int8 ? launch_tile<true, 64>(T, stream) : launch_tile<false, 64>(T, stream);
    case 128: return int8 ? launch_tile<true, 128>(T, stream) : launch_tile<false, 128>(T, stream);
    default: return int8 ? launch_tile<true, 256>(T, stream) : launch_tile<false, 256>(T, stream);
  }
}

}  // namespace b200
