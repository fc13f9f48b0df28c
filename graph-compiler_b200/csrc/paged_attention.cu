// Attention of one new token per sequence over a paged key-value cache:
//   out = sum_t p_t v_t / sum_t p_t,  p_t = 2^(x_t - m),  x_t = log2(e) scale q . k_t,  m a reference close to max_t x_t
// with the running reference and sum of an online softmax, so that keys and values are read once: for up to sixteen query heads to a
// KV head, eight with head_dim above 128.  More are several sets, each of which reads them again.
//
// Bound by HBM: 2 head_dim elements of cache per token and KV head, for 4 head_dim operations per query head, so everything is
// arranged for an even, unbroken stream of the cache:
//  * Work.  Sequences have any length, and the host does not know it (a captured step follows lengths in device memory).  Every
//    block adds up the lengths itself and takes an equal share of all tiles of tokens (paged_index.h).  Units (a sequence's KV
//    head) that a border cuts leave f32 parts in the workspace, which a second kernel, started behind the first by a dependent
//    launch, joins in the order of the blocks: the same bits every time, and no counter that a call leaves behind.
//  * A warp fetches its own tokens (16 or 32 of a tile) with asynchronous 16-byte copies, two or three tiles ahead, and waits for nobody:
//    page numbers come one tile further ahead, so that no copy waits for the table.  Rows behind the sequence's end are filled with
//    zeros by the copy.
//  * Products on the tensor cores with the TOKENS on the instruction's 16-row side and the query heads of the KV head on its
//    8-column side: S^T = K Q^T and O^T += V^T P^T.  Eight heads to a KV head fill it; fewer leave columns empty, which costs
//    nothing that the stream would notice.  P^T goes from the result layout of the first product to the operand layout of the
//    second by an 8 x 8 transposition in registers.
//  * The reference m only follows the maximum when that has grown by more than 2^8: one vote per tile instead of a reduction.
//  * P goes into the product with V as two 16-bit numbers, its upper bits and the rest: to 2^-15 of itself in bf16, 2^-20 in f16, where
//    one number leaves 2^-8 and 2^-11, and results 1.4 times as far off as their own rounding.  With one number and with two:
//    2 x 131071 tokens 168.3 and 169.3 us, 16 x 2048 of 32 heads 87.5 and 87.9, with sixteen query heads to each of them 94.5 and 96.4.
//    bf16 results over an 8-bit cache do with one f16 number, three bits more than they have themselves: two took 212 us instead of
//    203 at 128 x 1024..8192 tokens, at the power cap, for the same error.
//  * In f16 the reference lies 2^7 below the maximum: without that, tokens below 2^-25 of the largest would vanish, and a hundred
//    thousand of them may hold a third of a percent of the sum.
//  * 8-bit caches become f16 in registers (exact).  Queries are scaled to f16 by a power of two per head.
//
// Measured through Python with other calls around (two figures where GPUs differ), 128-wide heads, eight query heads to a KV head unless
// said otherwise: 2 x 131071 tokens 165 to 172 us (6.2 to 6.5 TB/s; a copy reaches 6.6), 64 x 512..4096 tokens with four heads to a KV
// head 101 to 104 (5.9), 16 x 2048 tokens of 32 heads of their own 88 to 91 (6.0), 128 x 1024..8192 tokens in 8 bits 195 to 206 (5.7 to
// 6.1, at the power cap: 620 instructions for 8 KB of cache against 360 in 16 bits).  Sixteen query heads to a KV head, whose registers
// leave two blocks to an SM: 2 x 131071 tokens 166 (6.5), 128 x 1024..8192 in 8 bits 235 (5.0), 64 x 512..4096 111 (5.5); 32 heads, 2 x
// 131071, 314.  256-wide heads, one sequence of 131071 tokens: 165 (6.5), sixteen to a KV head 315.  Few tokens: 1 x 1031 takes 8.5 us
// of the device, two launches; 37 windows of up to 700 tokens 12.5, a chain of latencies (lengths, page numbers, tokens, the warps'
// sums, the join).
#include "decode_ops.h"

#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "mma_ptx.cuh"
#include "runtime.h"

namespace gcb {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxBlocks = 592;   // the workspace has two parts for each
constexpr float kLazy = 8.f;

// The workspace: a Cut for every block, then two parts for every block.  Part of a cut unit: [cols][dim] f32 sums, then m and l of
// each column.
struct Cut {
  int seq, unit;
  int first, count;      // blocks with a part of the unit that the border before this block cuts; count 0: it cuts nothing
  int slot;              // of the first block's part (part_slot); the others' are their blocks' first
  int lead;              // the unit's first cut
  int pad[2];
};
struct PagedAttParams {
  PagedCache c;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_seq, q_head, o_seq, o_head;   // elements
  const int32_t *lengths;
  float *lse, *parts;
  Cut *cuts;
  float scale_log2e;
  int heads, group, sets, window, blocks;   // sets: of query heads per KV head, each the columns of one product
  bool q_aligned, same_strides;
};

// What a template instance keeps in shared memory.
template <bool F8, int DP, int NT> struct Shape {
  static constexpr int kRow = DP * (F8 ? 1 : 2);            // bytes of a token's row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kTokens = kRow <= 128 ? 32 : 16;     // of a warp in a tile
  static constexpr int kTile = kWarps * kTokens;
  static constexpr int kSlot = 2 * kTokens * kRow;          // a warp's keys and values of one tile
  static constexpr int kCols = 8 * NT;                      // query heads
  // Blocks to an SM: three where their registers allow it, else two, one with heads of 256.  Three stages where that many blocks then
  // find room in its 228 KB (each with its statically allocated 3 KB and 1 KB of the driver's), else two.
  static constexpr int kResident = NT == 1 && DP <= 128 ? 3 : DP <= 128 ? 2 : 1;
  static constexpr int kQRow = DP * 2 + 16;                 // bytes, padded against bank conflicts
  static constexpr int kQ = kCols * kQRow;
  static constexpr int bytes(int stages) { return stages * kWarps * kSlot + (stages + 1) * kQ; }
  static constexpr bool fits(int stages) { return kResident * (bytes(stages) + 4096) <= 228 * 1024; }
  static constexpr int kStages = fits(3) ? 3 : 2;
  static constexpr int kBytes = bytes(kStages);
  static_assert(fits(kStages), "as many blocks to an SM as the registers are shared out for");
  static_assert(kCols * DP * 4 <= kSlot, "a warp's results fit where its tokens were");
};
__host__ __device__ __forceinline__ int64_t part_floats(int cols, int dim) { return int64_t(cols) * (dim + 2); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }   // -inf - -inf would be NaN

// Two numbers of zero and more as the sums of two 16-bit ones each: the upper bits (returned) and what is left (`rest`).  With INF, where
// an infinity may meet them, both parts are above zero and not just the upper one, since zero times infinity is NaN: the upper bits
// are those of a little less.  In f16 the steps of a number below 2^-14 (2^-21 of the largest weight) are all 2^-24, and it is rounded to
// the nearest, whole or in halves: cutting it off, or a rest that is never zero, would add up over many.
template <bool BF16, bool INF> __device__ __forceinline__ uint32_t split_half2(float lo, float hi, uint32_t &rest) {
  constexpr float kLess = INF ? 1.f - 0x1p-10f : 1.f, kSmall = INF ? 0.5f : 1.f;
  if constexpr (BF16) {
    const float lo_up = __uint_as_float(__float_as_uint(lo) & 0xFFFF0000u), hi_up = __uint_as_float(__float_as_uint(hi) & 0xFFFF0000u);
    rest = pack_half2<true>(fmaf(lo_up, -(1.f - 0x1p-20f), lo), fmaf(hi_up, -(1.f - 0x1p-20f), hi));   // 2^-20 of the upper part on top
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
  } else {
    const float lo_up = lo < 0x1p-14f ? lo * kSmall : __uint_as_float(__float_as_uint(lo * kLess) & 0xFFFFE000u);
    const float hi_up = hi < 0x1p-14f ? hi * kSmall : __uint_as_float(__float_as_uint(hi * kLess) & 0xFFFFE000u);
    rest = pack_half2<false>(lo - lo_up, hi - hi_up);
    return pack_half2<false>(lo_up, hi_up);
  }
}

// Where a tile of the row of all tiles is.
struct Place {
  int seq;
  int64_t rest;     // tiles of the sequence before it
};
// The number of all tiles; pre (room for kThreads + 1) receives those before each thread's sequences, for one unit.  All threads of
// the block call it.
template <int TILE> __device__ __forceinline__ int64_t count_tiles(const PagedAttParams &p, int units, int64_t *pre) {
  const int n = p.c.table.sequences, each = (n + kThreads - 1) / kThreads, s0 = threadIdx.x * each, s1 = min(n, s0 + each);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += tiles_of(seen_of(p.c.table, p.lengths[s], p.window), TILE);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t sum = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const int64_t other = __shfl_up_sync(0xFFFFFFFFu, sum, i);
    if (lane >= i) sum += other;
  }
  __shared__ int64_t warp_sum[kWarps];
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  pre[threadIdx.x] = before + sum - mine;
  if (threadIdx.x == 0) pre[kThreads] = all;
  return all * units;
}
// The place of tile number `want` < total, behind count_tiles; all threads call it, `found` is shared.
template <int TILE> __device__ __forceinline__ Place locate(const PagedAttParams &p, int units, const int64_t *pre, int64_t want, Place *found) {
  if (threadIdx.x == 0) *found = Place{};
  __syncthreads();
  const int n = p.c.table.sequences, each = (n + kThreads - 1) / kThreads;
  int64_t at = pre[threadIdx.x] * units;
  if (at <= want && want < pre[threadIdx.x + 1] * units) {
    int s = threadIdx.x * each;
    for (; s < n - 1; ++s) {
      const int64_t here = int64_t(tiles_of(seen_of(p.c.table, p.lengths[s], p.window), TILE)) * units;
      if (want < at + here) break;
      at += here;
    }
    found->seq = s;
    found->rest = want - at;
  }
  __syncthreads();
  return *found;
}

// Walks the row of tiles.
struct Cursor {
  int seq, unit, tile, tiles, first, end;
};
template <int TILE> __device__ __forceinline__ void open_sequence(const PagedAttParams &p, Cursor &c) {
  const Seen s = seen_of(p.c.table, p.lengths[c.seq], p.window);
  c.first = s.first;
  c.end = s.end;
  c.tiles = tiles_of(s, TILE);
}
// To the next tile, which must exist.
template <int TILE> __device__ __forceinline__ void advance(const PagedAttParams &p, int units, Cursor &c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.unit < units) return;
  c.unit = 0;
  do {
    if (c.seq + 1 >= p.c.table.sequences) return;   // only if somebody changes the lengths meanwhile
    ++c.seq;
    open_sequence<TILE>(p, c);
  } while (c.tiles == 0);
}

// 16-byte chunk `ch` of row `r`: chunks of eight neighbouring rows lie in different banks.
template <int CHUNKS> __device__ __forceinline__ uint32_t chunk_at(int r, int ch) {
  if constexpr (CHUNKS >= 8) return uint32_t(r * CHUNKS + (ch ^ (r & 7))) * 16u;
  else return uint32_t(r * CHUNKS + (ch ^ ((r >> 1) & 3))) * 16u;
}

// FULL: head_dim is DP, and nothing has to ask where it ends.
template <bool BF16, bool F8, int DP, int NT, bool FULL>
__global__ void __launch_bounds__(kThreads, Shape<F8, DP, NT>::kResident) paged_attention_kernel(const __grid_constant__ PagedAttParams p) {
  using S = Shape<F8, DP, NT>;
  constexpr bool kMmaBf16 = BF16 && !F8;
  constexpr bool kSplit = !(F8 && BF16);   // P as two numbers: where one alone has no more bits than the result
  constexpr int kStages = S::kStages, kSteps = DP / 16, kSubs = S::kTokens / 16;
  constexpr float kBelow = kMmaBf16 ? 0.f : 7.f;   // the reference under the maximum: P reaches 2^(kBelow + kLazy), below f16's 2^16
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t pre[kThreads + 1];
  __shared__ Place found;
  __shared__ float stat_m[kWarps][S::kCols], stat_l[kWarps][S::kCols];
  __shared__ __align__(16) float share[kWarps][kWarps][S::kCols];   // each warp's own copy: what part of the sum the warps' results are

  const PagedCache &c = p.c;
  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x >> 5), 0);   // known to be the same in all lanes
  const int lane = threadIdx.x & 31, row8 = lane >> 2, col4 = lane & 3;
  const int units = c.kv_heads * p.sets, dim = FULL ? DP : c.dim;
  pdl_wait();
  pdl_launch_dependents();   // behind the wait: what starts now finds everything before this kernel done

  const int64_t total = count_tiles<S::kTile>(p, units, pre), per = share_of(total, p.blocks, 1);
  const int64_t begin = int64_t(blockIdx.x) * per, stop = min(total, begin + per);
  Cut cut{};

  if (begin < stop) {
    Place at = locate<S::kTile>(p, units, pre, begin, &found);
    Cursor comp;   // of the tile being computed
    comp.seq = at.seq;
    open_sequence<S::kTile>(p, comp);
    comp.unit = min(units - 1, int(at.rest / max(1, comp.tiles)));
    comp.tile = int(at.rest - int64_t(comp.unit) * comp.tiles);
    Cursor ahead = comp;   // of the tile whose page numbers are being fetched
    const int count = int(stop - begin);
    const int first_tile = comp.tile;
    const int64_t unit_begin = begin - first_tile;
    if (first_tile > 0) {
      cut.seq = comp.seq;
      cut.unit = comp.unit;
      cut.lead = first_cut(blockIdx.x, per, unit_begin, unit_begin + comp.tiles);
      cut.first = int(unit_begin / per);
      cut.count = int((unit_begin + comp.tiles - 1) / per) - cut.first + 1;
      cut.slot = int(part_slot(cut.first, per, unit_begin));
    }

    uint8_t *mine = smem + warp * kStages * S::kSlot;
    uint8_t *qring = smem + kWarps * kStages * S::kSlot;
    // ---- what the next tile to fetch needs: this lane's token's entry of the page table, and its place in the page
    int next_page = -1, next_slot = 0, fetched = 0, segments = 0;
    int entry = 0, slot = 0;              // of this lane's token of tile `ahead`
    int ahead_kv = 0, ahead_set = 0, next_kv = 0, next_set = 0, next_seq = 0;
    bool next_new = true, opened = true;
    const int step_entry = S::kTile / c.table.page_size, step_slot = S::kTile % c.table.page_size;
    auto look_up = [&]() {
      if (fetched >= count) return;
      const int pos = ahead.first + ahead.tile * S::kTile + warp * S::kTokens + lane;
      if (opened) {   // divisions once per unit; from tile to tile the place moves by the same step
        entry = pos / c.table.page_size;
        slot = pos - entry * c.table.page_size;
        ahead_kv = ahead.unit / p.sets;
        ahead_set = ahead.unit - ahead_kv * p.sets;
      }
      next_new = opened;
      next_seq = ahead.seq;
      next_kv = ahead_kv;
      next_set = ahead_set;
      next_slot = slot;
      next_page = -1;
      if (lane < S::kTokens && pos < ahead.end) {
        next_page = page_at(c.table, ahead.seq, entry);
        if (next_page < 0) report_bad_page(c.error);
      }
      entry += step_entry;
      slot += step_slot;
      if (slot >= c.table.page_size) {
        slot -= c.table.page_size;
        ++entry;
      }
      opened = false;
      if (++fetched < count) {
        advance<S::kTile>(p, units, ahead);
        opened = ahead.tile == 0;
      }
    };
    // Copies: eight lanes (four for rows of 64 bytes) take one row's chunks, and go on every 128 bytes and every kRows rows.
    constexpr int kLanes = S::kChunks < 8 ? S::kChunks : 8, kRows = 32 / kLanes, kPieces = S::kChunks / kLanes;
    const int lane_row = lane / kLanes, lane_chunk = lane % kLanes;
    const uint32_t copy_even = chunk_at<S::kChunks>(lane_row, lane_chunk), copy_odd = chunk_at<S::kChunks>(lane_row + kRows, lane_chunk) - kRows * S::kRow;
    const uint32_t mine_s = smem_u32(mine);
    auto issue = [&](int stage) {
      if (next_new) {
        uint8_t *dst = qring + (segments % (kStages + 1)) * S::kQ;
        ++segments;
        for (int i = threadIdx.x; i < S::kCols * (DP / 8); i += kThreads) {
          const int col = i / (DP / 8), d = (i - col * (DP / 8)) * 8, in_group = next_set * S::kCols + col;
          const bool there = in_group < p.group && d < dim;
          const uint16_t *src = p.q + (there ? next_seq * p.q_seq + (next_kv * p.group + in_group) * p.q_head + d : 0);
          uint8_t *to = dst + col * S::kQRow + d * 2;
          if (p.q_aligned) {
            cp_async_16(smem_u32(to), src, there ? 16u : 0u);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) reinterpret_cast<uint16_t *>(to)[e] = there ? src[e] : uint16_t(0);
          }
        }
      }
      const int64_t koff = next_page < 0 ? -1 : next_page * c.key_page + next_slot * c.key_token;
      const int64_t voff = p.same_strides || next_page < 0 ? koff : next_page * c.value_page + next_slot * c.value_token;
      const uint8_t *kbase = c.keys + next_kv * c.key_head + lane_chunk * 16, *vbase = c.values + next_kv * c.value_head + lane_chunk * 16;
      const uint32_t even = mine_s + stage * S::kSlot + copy_even, odd = mine_s + stage * S::kSlot + copy_odd;
#pragma unroll
      for (int i = 0; i < S::kTokens / kRows; ++i) {
        const int64_t ko = __shfl_sync(0xFFFFFFFFu, koff, i * kRows + lane_row);
        int64_t vo = ko;
        if (!p.same_strides) vo = __shfl_sync(0xFFFFFFFFu, voff, i * kRows + lane_row);
        const uint32_t bytes = ko < 0 ? 0u : 16u, to = (i & 1 ? odd : even) + i * kRows * S::kRow;
        const uint8_t *kp = ko < 0 ? kbase : kbase + ko, *vp = ko < 0 ? vbase : vbase + vo;
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
          if (FULL || (lane_chunk + e * kLanes) * 16 < dim * (F8 ? 1 : 2)) {
            cp_async_16(to + e * 128, kp + e * 128, bytes);
            cp_async_16(to + e * 128 + S::kTokens * S::kRow, vp + e * 128, bytes);
          }
        }
      }
      look_up();
    };

    look_up();
    for (int i = 0; i < kStages; ++i) {
      if (i < count) issue(i);
      cp_async_commit();
    }

    // Where this lane points the matrix loads of step j: four places, the rest is a constant distance (two with rows of 64 bytes).
    const int k_row = lane & 15, k_chunk = lane >> 4, v_row = (lane & 7) + 8 * (lane >> 4), v_chunk = (lane >> 3) & 1;
    uint32_t k_at[4], v_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k_at[i] = chunk_at<S::kChunks>(k_row, (2 * i + k_chunk) % S::kChunks);
      v_at[i] = chunk_at<S::kChunks>(v_row, (2 * i + v_chunk) % S::kChunks);
    }
    // chunk pair `pair` (two chunks) of sixteen rows from row 16 u
    auto pair_at = [](const uint32_t (&at)[4], int u, int pair) {
      return at[pair & 3] + uint32_t((pair >> 2) * 128 + u * 16 * S::kRow);
    };
    uint32_t qf[kSteps][NT][2];
    float acc[kSteps][NT][4], m[NT][2], ref[NT][2], l[NT][2], factor[NT][2];
    int stage = 0, segment = 0;
    bool fresh = true;   // the tile is the first one of its unit here
    for (int x = 0; x < count; ++x) {
      cp_async_wait<kStages - 1>();
      __syncwarp();
      if (fresh) {
        __syncthreads();   // the queries were fetched by all warps
        const uint8_t *qs = qring + (segment % (kStages + 1)) * S::kQ + row8 * S::kQRow;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint8_t *qrow = qs + n * 8 * S::kQRow;
          float mul = p.scale_log2e;
          if constexpr (F8) {
            // a power of two brings the row's largest magnitude to [2^7, 2^8); what f16 then drops is below 2^-31 of it
            float big = 0.f;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              const uint2 u = *reinterpret_cast<const uint2 *>(qrow + j * 32 + col4 * 8);
              big = fmaxf(big, fmaxf(fmaxf(fabsf(half_to_f32<BF16>(u.x & 0xFFFFu)), fabsf(half_to_f32<BF16>(u.x >> 16))),
                                     fmaxf(fabsf(half_to_f32<BF16>(u.y & 0xFFFFu)), fabsf(half_to_f32<BF16>(u.y >> 16)))));
            }
            big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
            int e = int(__float_as_uint(big) >> 23) - 127 - 7;   // big in [2^(e + 7), 2^(e + 8))
            if (!(big < INFINITY) || big < 1e-30f) e = 0;
            const float down = __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              const uint2 u = *reinterpret_cast<const uint2 *>(qrow + j * 32 + col4 * 8);
              qf[j][n][0] = pack_half2<false>(half_to_f32<BF16>(u.x & 0xFFFFu) * down, half_to_f32<BF16>(u.x >> 16) * down);
              qf[j][n][1] = pack_half2<false>(half_to_f32<BF16>(u.y & 0xFFFFu) * down, half_to_f32<BF16>(u.y >> 16) * down);
            }
            mul *= __uint_as_float(uint32_t(127 + e) << 23);
            if (c.key_scale) mul *= c.key_scale[comp.unit / p.sets];
          } else {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              qf[j][n][0] = *reinterpret_cast<const uint32_t *>(qrow + j * 32 + col4 * 4);
              qf[j][n][1] = *reinterpret_cast<const uint32_t *>(qrow + j * 32 + col4 * 4 + 16);
            }
          }
          // this thread's results belong to columns 2 col4 and 2 col4 + 1
          factor[n][0] = __shfl_sync(0xFFFFFFFFu, mul, col4 * 8);
          factor[n][1] = __shfl_sync(0xFFFFFFFFu, mul, col4 * 8 + 4);
          m[n][0] = m[n][1] = -INFINITY;
          ref[n][0] = ref[n][1] = 0.f;
          l[n][0] = l[n][1] = 0.f;
#pragma unroll
          for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][n][i] = 0.f;
        }
        fresh = false;
      }

      const uint32_t ks = mine_s + stage * S::kSlot, vs = ks + S::kTokens * S::kRow;
      // ---- S^T = K Q^T
      float sc[kSubs][NT][4], sd[kSubs][NT][4];   // even and odd steps: one chain of dependent products half as long
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[u][n][i] = sd[u][n][i] = 0.f;
#pragma unroll
      for (int u = 0; u < kSubs; ++u) {
        if constexpr (F8) {
#pragma unroll
          for (int j = 0; j < kSteps; j += 2) {
            if (FULL || j * 16 < dim) {
              uint32_t r[4];   // tokens 0-7 and 8-15 of chunk j, then of chunk j + 1
              ldmatrix_x4(r, ks + pair_at(k_at, u, j / 2));
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (!FULL && (j + h) * 16 >= dim) break;   // an odd number of chunks: nobody has filled the last one
                uint32_t a[4];
                e4m3x4_to_f16x2(r[2 * h], a[0], a[2]);
                e4m3x4_to_f16x2(r[2 * h + 1], a[1], a[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816<kMmaBf16>(h ? sd[u][n] : sc[u][n], a, qf[j + h][n][0], qf[j + h][n][1]);
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            if (FULL || j * 16 < dim) {
              uint32_t a[4];
              ldmatrix_x4(a, ks + pair_at(k_at, u, j));
              if (!FULL && j * 16 + 8 >= dim) a[2] = a[3] = 0u;   // half a step: nobody has filled the other half
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_16816<kMmaBf16>(j & 1 ? sd[u][n] : sc[u][n], a, qf[j][n][0], qf[j][n][1]);
            }
          }
        }
      }
      // ---- softmax
      const int pos0 = comp.first + comp.tile * S::kTile + warp * S::kTokens;
      bool grow = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[u][n][i] = (sc[u][n][i] + sd[u][n][i]) * factor[n][i & 1];
      if (pos0 + S::kTokens > comp.end) {
#pragma unroll
        for (int u = 0; u < kSubs; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (pos0 + u * 16 + row8 + 8 * (i >> 1) >= comp.end) sc[u][n][i] = -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) top[n][i & 1] = fmaxf(top[n][i & 1], sc[u][n][i]);
#pragma unroll
      for (int n = 0; n < NT; ++n) grow = grow || top[n][0] > m[n][0] + (kLazy + kBelow) || top[n][1] > m[n][1] + (kLazy + kBelow);
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float t = top[n][h];
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, i));
            t = fmaxf(t - kBelow, m[n][h]);
            ref[n][h] = finite_ref(t);
            const float alpha = ex2(m[n][h] - ref[n][h]);
            m[n][h] = t;
            l[n][h] *= alpha;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              acc[j][n][h] *= alpha;
              acc[j][n][2 + h] *= alpha;
            }
          }
      }
      // ---- P, its sum, and O^T += V^T P^T
#pragma unroll
      for (int u = 0; u < kSubs; ++u) {
        uint32_t pt[NT][2], rt[NT][2];   // the weights' upper bits and the rest
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float w[4] = {ex2(sc[u][n][0] - ref[n][0]), ex2(sc[u][n][1] - ref[n][1]), ex2(sc[u][n][2] - ref[n][0]), ex2(sc[u][n][3] - ref[n][1])};
          l[n][0] += w[0] + w[2];
          l[n][1] += w[1] + w[3];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (kSplit) {
              uint32_t rest;
              pt[n][h] = movmatrix_trans(split_half2<kMmaBf16, !F8>(w[2 * h], w[2 * h + 1], rest));
              rt[n][h] = movmatrix_trans(rest);
            } else {
              pt[n][h] = movmatrix_trans(pack_half2<kMmaBf16>(w[2 * h], w[2 * h + 1]));
            }
          }
        }
        if constexpr (F8) {
          // chunk j holds head_dim 16 j ..: rows 2 i and 2 i + 1 of the result come from the low and the high byte of its pair i
#pragma unroll
          for (int j = 0; j < kSteps; j += 2) {
            if (FULL || j * 16 < dim) {
              uint32_t r[4];   // chunk j, tokens 0-7; chunk j + 1, tokens 0-7; chunk j, tokens 8-15; chunk j + 1, tokens 8-15
              ldmatrix_x4_trans(r, vs + pair_at(v_at, u, j / 2));
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (!FULL && (j + h) * 16 >= dim) break;
                const uint32_t t0 = __byte_perm(r[h], 0, 0x3120), t1 = __byte_perm(r[h + 2], 0, 0x3120);
                uint32_t a[4];
                e4m3x4_to_f16x2(t0, a[0], a[1]);
                e4m3x4_to_f16x2(t1, a[2], a[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma_16816<kMmaBf16>(acc[j + h][n], a, pt[n][0], pt[n][1]);
                  if constexpr (kSplit) mma_16816<kMmaBf16>(acc[j + h][n], a, rt[n][0], rt[n][1]);
                }
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            if (FULL || j * 16 < dim) {
              uint32_t a[4];
              ldmatrix_x4_trans(a, vs + pair_at(v_at, u, j));
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma_16816<kMmaBf16>(acc[j][n], a, pt[n][0], pt[n][1]);
                if constexpr (kSplit) mma_16816<kMmaBf16>(acc[j][n], a, rt[n][0], rt[n][1]);
              }
            }
          }
        }
      }

      const bool unit_ends = comp.tile + 1 == comp.tiles;
      if (unit_ends || x + 1 == count) {
        // ---- the four warps' parts meet in shared memory, each in the slot whose tokens it has just used
        __syncwarp();
        float *own = reinterpret_cast<float *>(mine + stage * S::kSlot);   // [DP][cols]
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            const int d0 = F8 ? j * 16 + 2 * row8 : j * 16 + row8, d1 = F8 ? d0 + 1 : d0 + 8;
            *reinterpret_cast<float2 *>(own + d0 * S::kCols + n * 8 + 2 * col4) = make_float2(acc[j][n][0], acc[j][n][1]);
            *reinterpret_cast<float2 *>(own + d1 * S::kCols + n * 8 + 2 * col4) = make_float2(acc[j][n][2], acc[j][n][3]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) l[n][h] += __shfl_xor_sync(0xFFFFFFFFu, l[n][h], i);
            if (lane < 4) {
              stat_m[warp][n * 8 + 2 * col4 + h] = m[n][h];
              stat_l[warp][n * 8 + 2 * col4 + h] = l[n][h];
            }
          }
        }
        __syncthreads();
        const int kv = comp.unit / p.sets, set = comp.unit - kv * p.sets;
        const int cols = min(S::kCols, p.group - set * S::kCols);
        const bool begins = segment > 0 || first_tile == 0;   // not the unit that the block before began
        const bool whole = begins && unit_ends;
        float *out_part = p.parts + (2 * int64_t(blockIdx.x) + (begins ? 1 : 0)) * part_floats(S::kCols, dim);
        const float vscale = F8 && c.value_scale ? c.value_scale[kv] : 1.f;
        // lane (w, h) of each warp: what warp w's result of column h counts
        float top_m[NT], sum_l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float mine_m = stat_m[lane >> 3][n * 8 + (lane & 7)];
          float t = fmaxf(mine_m, __shfl_xor_sync(0xFFFFFFFFu, mine_m, 8));
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 16));
          const float part = ex2(mine_m - finite_ref(t));
          float sum = stat_l[lane >> 3][n * 8 + (lane & 7)] * part;
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
          top_m[n] = t;
          sum_l[n] = sum;
          share[warp][lane >> 3][n * 8 + (lane & 7)] = whole ? part / sum * vscale : part;
        }
        __syncwarp();
        for (int i = threadIdx.x; i < NT * dim; i += kThreads) {
          const int n = NT == 1 ? 0 : i / dim, d = i - n * dim;
          float sum[8] = {};
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 *src = reinterpret_cast<const float4 *>(smem + (w * kStages + stage) * S::kSlot) + (d * S::kCols + n * 8) / 4;
            const float4 *by = reinterpret_cast<const float4 *>(&share[warp][w][n * 8]);
            const float4 a = src[0], b = src[1], x0 = by[0], x1 = by[1];
            sum[0] = fmaf(a.x, x0.x, sum[0]); sum[1] = fmaf(a.y, x0.y, sum[1]); sum[2] = fmaf(a.z, x0.z, sum[2]); sum[3] = fmaf(a.w, x0.w, sum[3]);
            sum[4] = fmaf(b.x, x1.x, sum[4]); sum[5] = fmaf(b.y, x1.y, sum[5]); sum[6] = fmaf(b.z, x1.z, sum[6]); sum[7] = fmaf(b.w, x1.w, sum[7]);
          }
          const int head = kv * p.group + set * S::kCols + n * 8;
#pragma unroll
          for (int h = 0; h < 8; ++h) {
            if (n * 8 + h >= cols) break;
            if (whole) p.out[comp.seq * p.o_seq + (head + h) * p.o_head + d] = f32_to_half<BF16>(sum[h]);
            else out_part[int64_t(n * 8 + h) * dim + d] = sum[h];
          }
        }
        if (warp == 0 && lane < 8) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int col = n * 8 + lane, head = kv * p.group + set * S::kCols + col;
            if (col >= cols) break;
            if (!whole) {
              out_part[int64_t(S::kCols) * dim + 2 * col] = top_m[n];
              out_part[int64_t(S::kCols) * dim + 2 * col + 1] = sum_l[n];
            } else if (p.lse) {
              p.lse[int64_t(comp.seq) * p.heads + head] = (finite_ref(top_m[n]) + log2f(sum_l[n])) * 0.6931471805599453f;
            }
          }
        }
        __syncthreads();   // before the slots are filled again
        fresh = true;
        ++segment;
      }
      __syncwarp();
      if (x + kStages < count) issue(stage);
      cp_async_commit();
      if (++stage == kStages) stage = 0;
      if (x + 1 < count) advance<S::kTile>(p, units, comp);
    }
    cp_async_wait<0>();
  }

  if (threadIdx.x == 0) p.cuts[blockIdx.x] = cut;
  // ---- sequences of which nothing is seen
  for (int s = blockIdx.x; s < c.table.sequences; s += gridDim.x) {
    const Seen see = seen_of(c.table, p.lengths[s], p.window);
    if (see.cut && threadIdx.x == 0) report_bad_page(c.error);
    if (see.end > see.first) continue;
    for (int i = threadIdx.x; i < p.heads * dim; i += kThreads) {
      const int h = i / dim;
      p.out[s * p.o_seq + h * p.o_head + (i - h * dim)] = 0;
    }
    if (p.lse)
      for (int h = threadIdx.x; h < p.heads; h += kThreads) p.lse[int64_t(s) * p.heads + h] = -INFINITY;
  }
}

// Block (i - 1, y): the unit that border i cuts.  Up to sixteen parts: the blocks of its first cut join them, a warp to a column.  More:
// the blocks of all its cuts take a column each, the four warps every fourth part (156 parts behind one warp took 15 us).  The lanes
// weigh 32 parts at a time by their maxima, then add the parts up, four elements to a lane.
template <bool BF16, bool F8, int NT, int HALVES>   // HALVES: of head_dim, 128 elements to the lanes at a time
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const __grid_constant__ PagedAttParams p) {
  constexpr int kCols = 8 * NT;
  const PagedCache &c = p.c;
  __shared__ __align__(16) float warp_m[kWarps], warp_l[kWarps], warp_sum[kWarps][HALVES * 128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = c.dim;
  pdl_wait();
  pdl_launch_dependents();
  const Cut cut = p.cuts[blockIdx.x + 1];
  constexpr int kAhead = 16;   // parts asked for at once (one by one behind their weights, eight under way, 17 parts took 2.3 us longer)
  const bool together = cut.count > kAhead;
  if (cut.count == 0 || (!together && !cut.lead)) return;
  const int kv = cut.unit / p.sets, set = cut.unit - kv * p.sets;
  const int col = together ? (int(blockIdx.x) - cut.first) * int(gridDim.y) + int(blockIdx.y) : int(blockIdx.y) * kWarps + warp;
  if (col >= min(kCols, p.group - set * kCols)) return;
  const int step = together ? kWarps : 1, start = together ? warp : 0, count = (cut.count - start + step - 1) / step;   // this warp's parts
  const int64_t floats = part_floats(kCols, dim);
  // part i of the unit: every block but the first one continues the unit and has its part in its first slot
  const float *rest = p.parts + 2 * int64_t(cut.first) * floats, *first = p.parts + cut.slot * floats;
  auto part = [&](int i) {
    const int at = start + i * step;
    return at == 0 ? first : rest + 2 * int64_t(at) * floats;
  };
  auto of_lane = [&](int i, int h) {   // this lane's four elements of part i
    return i < count && h * 128 + lane * 4 < dim ? *reinterpret_cast<const float4 *>(part(i) + int64_t(col) * dim + h * 128 + lane * 4)
                                                 : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float4 ahead[kAhead][HALVES];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (i == kAhead / 2 && count <= kAhead / 2) break;
#pragma unroll
    for (int h = 0; h < HALVES; ++h) ahead[i][h] = of_lane(i, h);
  }
  float m = -INFINITY;
  for (int i = lane; i < count; i += 32) m = fmaxf(m, part(i)[int64_t(kCols) * dim + 2 * col]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, i));
  const float ref = finite_ref(m);
  float l = 0.f;
  float4 sum[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) sum[h] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4 &v, float by, int h) {
    sum[h].x = fmaf(v.x, by, sum[h].x);
    sum[h].y = fmaf(v.y, by, sum[h].y);
    sum[h].z = fmaf(v.z, by, sum[h].z);
    sum[h].w = fmaf(v.w, by, sum[h].w);
  };
  for (int i0 = 0; i0 < count; i0 += 32) {
    float w = 0.f;
    if (i0 + lane < count) {
      const float2 ml = *reinterpret_cast<const float2 *>(part(i0 + lane) + int64_t(kCols) * dim + 2 * col);
      w = ex2(ml.x - ref);
      l = fmaf(ml.y, w, l);
    }
    const int n = min(32, count - i0);
    int i = 0;
    if (i0 == 0) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (a == kAhead / 2 && n <= kAhead / 2) break;
        const float by = __shfl_sync(0xFFFFFFFFu, w, a);
        if (a < n)
#pragma unroll
          for (int h = 0; h < HALVES; ++h) add(ahead[a][h], by, h);
      }
      i = kAhead;
    }
#pragma unroll 8
    for (; i < n; ++i) {
      const float by = __shfl_sync(0xFFFFFFFFu, w, i);
#pragma unroll
      for (int h = 0; h < HALVES; ++h) add(of_lane(i0 + i, h), by, h);
    }
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, i);
  if (together) {
    if (lane == 0) {
      warp_m[warp] = m;
      warp_l[warp] = l;
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h) *reinterpret_cast<float4 *>(&warp_sum[warp][h * 128 + lane * 4]) = sum[h];
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, warp_m[w]);
    l = 0.f;
#pragma unroll
    for (int h = 0; h < HALVES; ++h) sum[h] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float by = ex2(warp_m[w] - finite_ref(m));
      l = fmaf(warp_l[w], by, l);
#pragma unroll
      for (int h = 0; h < HALVES; ++h) add(*reinterpret_cast<const float4 *>(&warp_sum[w][h * 128 + lane * 4]), by, h);
    }
  }
  const float scale = (F8 && c.value_scale ? c.value_scale[kv] : 1.f) / l;
  const int head = kv * p.group + set * kCols + col;
  uint16_t *out = p.out + cut.seq * p.o_seq + head * p.o_head;
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
    if (h * 128 + lane * 4 < dim) {
      const float v[4] = {sum[h].x, sum[h].y, sum[h].z, sum[h].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) out[h * 128 + lane * 4 + e] = f32_to_half<BF16>(v[e] * scale);
    }
  if (lane == 0 && p.lse) p.lse[int64_t(cut.seq) * p.heads + head] = (finite_ref(m) + log2f(l)) * 0.6931471805599453f;
}

void require(bool ok, const char *what) {
  if (!ok) throw std::invalid_argument(what);
}

// Columns of a product: 16 for more than eight heads to a KV head, where the registers allow it.
int columns(int64_t group, int64_t dim) { return group > 8 && dim <= 128 ? 16 : 8; }

template <typename... KArgs, typename... Args>
void launch_dependent(void (*kernel)(KArgs...), dim3 grid, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  GCB_CUDA(cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...));
  count_launch();
}

template <bool BF16, bool F8, int DP, int NT, bool FULL> void launch(PagedAttParams p, DeviceState &dev, cudaStream_t stream) {
  using S = Shape<F8, DP, NT>;
  auto kernel = paged_attention_kernel<BF16, F8, DP, NT, FULL>;
  static int resident[64] = {};   // blocks of an SM
  int &r = resident[dev.device & 63];
  if (!r) {
    int n = 0;
    GCB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    GCB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, S::kBytes));
    r = std::max(1, n);
  }
  p.blocks = std::min(kMaxBlocks, dev.sm_count * r);
  launch_dependent(kernel, dim3(unsigned(p.blocks)), S::kBytes, stream, p);
  if (p.blocks > 1) launch_dependent(paged_join_kernel<BF16, F8, NT, (DP + 127) / 128>, dim3(unsigned(p.blocks - 1), 2 * NT), 0, stream, p);
}

template <bool BF16, bool F8> void launch(const PagedAttParams &p, int cols, DeviceState &dev, cudaStream_t stream) {
  const int dim = p.c.dim;
  if (dim == 64) cols == 16 ? launch<BF16, F8, 64, 2, true>(p, dev, stream) : launch<BF16, F8, 64, 1, true>(p, dev, stream);
  else if (dim < 64) cols == 16 ? launch<BF16, F8, 64, 2, false>(p, dev, stream) : launch<BF16, F8, 64, 1, false>(p, dev, stream);
  else if (dim == 128) cols == 16 ? launch<BF16, F8, 128, 2, true>(p, dev, stream) : launch<BF16, F8, 128, 1, true>(p, dev, stream);
  else if (dim < 128) cols == 16 ? launch<BF16, F8, 128, 2, false>(p, dev, stream) : launch<BF16, F8, 128, 1, false>(p, dev, stream);
  else if (dim == 256) launch<BF16, F8, 256, 1, true>(p, dev, stream);
  else launch<BF16, F8, 256, 1, false>(p, dev, stream);
}

} // namespace

size_t paged_attention_workspace(int64_t heads, int64_t kv_heads, int64_t head_dim) {
  require(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads < 65536, "paged attention: heads must be a multiple of kv_heads");
  require(head_dim > 0 && head_dim <= 256, "paged attention: head_dim must be at most 256");
  return kMaxBlocks * (sizeof(Cut) + 2 * size_t(part_floats(columns(heads / kv_heads, head_dim), int(head_dim))) * sizeof(float));
}

void paged_attention(const gcb200_paged_cache &cache, const PagedAttentionArgs &a, cudaStream_t stream) {
  PagedAttParams p{};
  p.c = checked_cache(cache, false);
  require(cache.sequences == 0 || (a.q && a.out && a.lengths && a.workspace), "paged attention: null pointer");
  require((reinterpret_cast<uintptr_t>(a.workspace) & 15) == 0, "paged attention: the workspace must be 16-byte aligned");
  require(a.workspace_bytes >= paged_attention_workspace(a.heads, cache.kv_heads, cache.head_dim), "paged attention: the workspace is too small");
  require(a.window >= 0, "paged attention: negative window");
  require(!rows_overlap(cache.sequences, a.out_stride[0], a.heads, a.out_stride[1], cache.head_dim), "paged attention: rows of the result overlap");
  require(aligned(a.q, 2) && aligned(a.out, 2) && aligned(a.lengths, 4) && aligned(a.lse, 4), "paged attention: misaligned pointer");
  if (cache.sequences == 0) return;
  DeviceState &dev = device_state();
  p.c.error = dev.d_page_error;
  p.q = static_cast<const uint16_t *>(a.q);
  p.out = static_cast<uint16_t *>(a.out);
  p.q_seq = cache.sequences > 1 ? a.q_stride[0] : 0;
  p.q_head = a.heads > 1 ? a.q_stride[1] : 0;
  p.o_seq = cache.sequences > 1 ? a.out_stride[0] : 0;
  p.o_head = a.heads > 1 ? a.out_stride[1] : 0;
  p.q_aligned = ((reinterpret_cast<uintptr_t>(a.q) | uintptr_t(2 * p.q_seq) | uintptr_t(2 * p.q_head)) & 15) == 0;
  p.same_strides = p.c.key_page == p.c.value_page && p.c.key_token == p.c.value_token;
  p.lengths = a.lengths;
  p.lse = a.lse;
  static_assert(kMaxBlocks * sizeof(Cut) % 16 == 0, "the parts are read in fours");
  p.cuts = static_cast<Cut *>(a.workspace);
  p.parts = reinterpret_cast<float *>(p.cuts + kMaxBlocks);
  p.scale_log2e = a.scale * 1.4426950408889634f;
  p.heads = int(a.heads);
  p.group = int(a.heads / cache.kv_heads);
  const int cols = columns(p.group, cache.head_dim);
  p.sets = (p.group + cols - 1) / cols;
  p.window = int(std::min<int64_t>(a.window, INT32_MAX));
  const bool bf16 = cache.dtype == GCB200_BF16, f8 = cache.cache_dtype == GCB200_F8_E4M3;
  (bf16 ? (f8 ? launch<true, true> : launch<true, false>) : (f8 ? launch<false, true> : launch<false, false>))(p, cols, dev, stream);
}

} // namespace gcb
