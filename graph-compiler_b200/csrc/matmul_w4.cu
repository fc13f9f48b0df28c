// Linear layers of a few rows with 4-bit weights:  Y = act(X . W^T + bias),  W[n][k] = (code - zero) * scale of n's group.
//
// Layout.  The weights are packed once into blocks of 16 outputs x 128 k, in the order in which a warp's matrix instruction
// takes them: 1024 bytes of codes (lane l reads 16 bytes at 16 l of each half), the scales of the 16 outputs for each of the
// block's groups, and their zeros.  The k range of an output tile is one contiguous stream.
//
// Codes become f16 numbers by a mask alone: four bits in the mantissa of a number with exponent zero are code * 2^-22 or
// code * 2^-18 (a subnormal, exact).  A word of eight codes takes one byte permutation and four masks; one that went through
// 16 + code took eight operations, and the integer units were what the kernel waited for.  With the sum of x over a group,
// sum x (code - zero) = sum x code - zero sum x:  the zero costs one multiply-add per group and result.
// X is f16 as it is; bf16 is scaled by a power of two per row and 128 k, which puts the largest magnitude at 2^14 and drops
// nothing above 2^-38 of it.  Products are exact in f32, sums are f32, a group's scale multiplies its f32 sum.
//
// Bound by HBM: half a byte per weight.  One block of sixteen warps to an SM stays there and works off its share of the output
// tiles; every warp streams blocks of its own through a ring of asynchronous copies that runs on across the tiles.  X lies in shared
// memory for the whole call.  Where it does not fit, or where there are fewer tiles than SMs, a cluster of 2 to 8 blocks shares
// the k of its tiles and exchanges f32 sums through distributed shared memory, one tile late, so that nobody waits for them.
// Measured: 1 x 28672 x 8192 28 us (4.3 TB/s), 8 rows 36, 16 rows 46, 32 rows 94, 64 rows 185 (a reading of the weights for every 16);
// 1 x 4096 x 4096 6, of which 4 are launch, first loads and the last sums; 5 x 11001 x 4095 with groups of 32 and zeros 14.  With one
// row what is left is that fixed time, with sixteen the multiplying warps' instructions: the kernel takes 41 of 47 us with no loads
// in its loop.  640 threads leave 96 registers: 21 of the 48 variants spill, at most 96 bytes (two tiles, 16 rows, groups of 32: 16 x
// 28672 x 8192 66 us, groups of 64 61).
// (1 KB bulk copies instead of the warps' 16-byte ones kept an SM at 12 to 20 bytes a cycle, half of what HBM gives it.)
#include "decode_ops.h"

#include <algorithm>
#include <mutex>
#include <stdexcept>
#include <type_traits>

#include "mma_ptx.cuh"
#include "runtime.h"
#include "w4_plan.h"

namespace gcb {

namespace {

void require(bool ok, const char *what) {
  if (!ok) throw std::invalid_argument(what);
}

struct W4PackParams {
  const uint8_t *codes, *zeros;
  const uint16_t *scales;
  int64_t codes_stride, scales_stride, zeros_stride, N, K, group;
  uint8_t *packed;
  int64_t kblocks;
  int gpb, bytes;
};

// 64 threads pack one 16 x 128 block, a thread 16 bytes: the four words of a lane in one half.  Word w of a lane in half h covers
// k = 64 h + 32 (w >> 1) + 8 c + 4 (w & 1) + {0, 1, 2, 3} of outputs r and r + 8 (r = lane / 4, c = lane % 4): the registers
// s = 0..3 of the instruction's A operand, each a pair of k in the word's halves.  Within a half, code s lies where a mask finds
// it: at bit 2, at bit 6, and, with the half's bytes exchanged, at bit 2 and bit 6 again.
constexpr int kPackBlocks = 4;   // k blocks of a thread block: 256 contiguous bytes of each row of codes
__global__ void __launch_bounds__(kPackBlocks * 64) w4_pack_kernel(const __grid_constant__ W4PackParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t kb = int64_t(blockIdx.x) * kPackBlocks + (threadIdx.x >> 6), nt = blockIdx.y + int64_t(blockIdx.z) * gridDim.y;
  if (nt * kRows >= p.N || kb >= p.kblocks) return;
  uint8_t *block = p.packed + (nt * p.kblocks + kb) * p.bytes;
  const int t = threadIdx.x & 63, h = t >> 5, lane = t & 31, r = lane >> 2, c = lane & 3;
  // eight codes of output n from k (a multiple of 8): k + i at bits 4 i
  auto codes8 = [&](int64_t n, int64_t k) -> uint32_t {
    if (n >= p.N || k >= p.K) return 0u;   // meets a scale or an x of zero
    const uint8_t *from = p.codes + n * p.codes_stride + (k >> 1);
    if (k + 8 <= p.K && (reinterpret_cast<uintptr_t>(from) & 3) == 0) return *reinterpret_cast<const uint32_t *>(from);
    uint32_t v = 0;
    for (int i = 0; i < 4; ++i)
      if (k + 2 * i < p.K) v |= uint32_t(from[i]) << (8 * i);
    return v;
  };
  uint32_t word[4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t k = kb * kBlockK + 64 * h + 32 * u + 8 * c, n = nt * kRows + r;
    const uint32_t row[2] = {codes8(n, k), codes8(n + 8, k)};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t out = 0;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t two = row[s & 1] >> (16 * w + 8 * (s >> 1)), pair = (two & 15u) | (two & 0xF0u) << 12;
        out |= s < 3 ? pair << (4 * s + 2) : (pair & 0x00030003u) << 14 | (pair >> 2 & 0x00030003u);
      }
      word[2 * u + w] = out;
    }
  }
  reinterpret_cast<uint4 *>(block)[h * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
  if (t < p.gpb * kRows) {   // [output][group]
    const int64_t n = nt * kRows + t / p.gpb, g = (kb * kBlockK + int64_t(t % p.gpb) * (kBlockK / p.gpb)) / p.group;
    const bool in = n < p.N && g * p.group < p.K;
    reinterpret_cast<uint16_t *>(block + kCodes)[t] = in ? p.scales[n * p.scales_stride + g] : uint16_t(0);
    if (p.zeros) block[kCodes + p.gpb * kRows * 2 + t] = in ? uint8_t(p.zeros[n * p.zeros_stride + g] & 15u) : uint8_t(0);
  }
}

struct W4Params {
  const uint16_t *x, *bias;
  const uint8_t *packed;
  uint16_t *y;
  int64_t ldx, ldy, N, K;
  int M, pass, relu, kblocks, tiles;   // pass: rows of x that a block takes; tiles: of 16 outputs
  int cluster, share, wk, stages;      // blocks that share k; k blocks of each; warps of a block that share them; depth of a ring
  int x_at, table_at, meet_at, part_at;
  int *error;
};

// Eight elements of x at `from`, of which the first `count` exist; [lo, hi): the bytes of all of x.  Rows on any two bytes: the two
// aligned pieces around, where both lie inside x.
__device__ __forceinline__ uint4 load_piece(const uint16_t *from, int64_t count, uintptr_t lo, uintptr_t hi) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(from), base = at & ~uintptr_t(15);
  if (count >= 8 && at == base) return *reinterpret_cast<const uint4 *>(from);
  if (count >= 8 && base >= lo && base + 32 <= hi) {
    const uint4 u = *reinterpret_cast<const uint4 *>(base), v = *reinterpret_cast<const uint4 *>(base + 16);
    uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    const uint32_t off = uint32_t(at - base);
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
    const uint32_t bits = (off & 2) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < count) w[e >> 1] |= uint32_t(from[e]) << (16 * (e & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct W4Bars {
  uint64_t meet_full, meet_empty;      // the warps' sums of an item are there / have been read
  uint64_t parts_in[2], parts_out[2];  // the cluster's sums of an item are there / have been read by everyone
};
__device__ __forceinline__ float4 ld_shared_cluster_v4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
// Bounded waits of the adding warps, which wait most of the time: asleep, off the issue slots of the warps that multiply.
template <bool CLUSTER> __device__ __forceinline__ bool wait_asleep(uint32_t bar, uint32_t parity) {
  auto there = [&] { return CLUSTER ? mbar_test_cluster(bar, parity) : mbar_test(bar, parity); };
  const long long t0 = clock64();
  while (!__all_sync(0xFFFFFFFFu, there())) {
    if (__any_sync(0xFFFFFFFFu, clock64() - t0 > WAIT_LIMIT_CYCLES)) return false;
    __nanosleep(100);
  }
  return true;
}
__device__ __forceinline__ void complain(int *error, bool ok, int code) {
  if (!ok && lane_id() == 0) atomicExch(error, code);
}

// RT tiles of 16 outputs to a warp, NT sets of 8 rows of x.  Warps 0-15 multiply, each with a stream of weights of its own; warps
// 16-19 add up and store.  Nobody waits for all the others.
template <bool BF16, int NT, int RT, int GPB, bool ZEROS>
__global__ void __launch_bounds__(kW4Threads, 1) matmul_w4_kernel(const __grid_constant__ W4Params p) {
  constexpr int kBlock = kCodes + GPB * kRows * (ZEROS ? 3 : 2), kStage = RT * kBlock;
  constexpr int kGroup = kBlockK / GPB, kMulThreads = kW4Warps * 32;
  constexpr float kUnit = 1.f / 4194304.f;   // of the codes of outputs r; of outputs r + 8 it is 16 times that
  constexpr int kOuts = 16 * RT, kMeetRow = kOuts + 4, kMeet = 8 * NT * kMeetRow;   // floats; the pad keeps the columns' banks apart
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ W4Bars bars;
  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x >> 5), 0);   // known to be the same in all lanes
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int wn = kW4Warps / p.wk;
  const int m0 = blockIdx.y * p.pass, rows = min(p.M - m0, p.pass);
  const int cluster = int(blockIdx.x) / p.cluster, clusters = int(gridDim.x) / p.cluster, rank = int(blockIdx.x) - cluster * p.cluster;
  const int kb0 = rank * p.share, here = max(0, min(p.share, p.kblocks - kb0));   // this block's k blocks
  const int pitch = p.share * kBlockK * 2 + kXPad, outs = kOuts * wn;             // outs: outputs of an item
  uint8_t *x = smem + p.x_at;   // [rows + 1][pitch] f16, the last row zeros
  // [group][rows + 1]: factor of the scaled x, and -2^-22 sum of the scaled x (times 8 where that is the zero of all)
  float2 *table = reinterpret_cast<float2 *>(smem + p.table_at);
  float *meet = reinterpret_cast<float *>(smem + p.meet_at), *part = reinterpret_cast<float *>(smem + p.part_at);
  const uint32_t meet_full = smem_u32(&bars.meet_full), meet_empty = smem_u32(&bars.meet_empty);
  if (threadIdx.x == 0) {
    mbar_init(meet_full, kW4Warps);
    mbar_init(meet_empty, kSumWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.parts_in[i]), uint32_t(p.cluster * kSumWarps));
      mbar_init(smem_u32(&bars.parts_out[i]), uint32_t(p.cluster * kSumWarps));
    }
    mbar_fence_init();
  }
  __syncthreads();
  if (p.cluster > 1) cluster_sync_all();   // every block's barriers are there before another one signals them
  pdl_wait();
  pdl_launch_dependents();
  // A cluster's tiles, an equal share of all, in items of wn RT; warp w multiplies k blocks kb0 + w % wk, + wk, ... of RT of them.
  const int first = int(int64_t(p.tiles) * cluster / clusters), last = int(int64_t(p.tiles) * (cluster + 1) / clusters);
  const int items = (last - first + wn * RT - 1) / (wn * RT);
  auto tile_of = [&](int w, int item) { return first + (item * wn + w / p.wk) * RT; };

  if (warp >= kW4Warps) {
    // ------------------------------------------------------------------ sums of the warps and of the cluster, results
    const int thread = threadIdx.x - kW4Warps * 32;
    const int64_t n_end = min(p.N, int64_t(last) * kRows);
    auto store = [&](int item, int m, int o, const float (&v)[4], int count) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t n = int64_t(first) * kRows + int64_t(item) * outs + o + i;
        if (i >= count || n >= n_end) break;
        float y = v[i];
        if (p.bias) y += half_to_f32<BF16>(p.bias[n]);
        if (p.relu) y = y != y ? y : fmaxf(y, 0.f);
        p.y[(m0 + m) * p.ldy + n] = f32_to_half<BF16>(y);
      }
    };
    const int mine = outs / p.cluster;                         // outputs of an item that this block finishes
    auto signal = [&](uint64_t *bar) {                         // to every block of the cluster, by one lane each
      __syncwarp();
      if (lane < p.cluster) mbar_arrive_cluster(mapa_shared(smem_u32(bar), uint32_t(lane)));
    };
    bool ok = true;
    auto finish = [&](int item, int use) {   // use: which item of this block, in order
      const int buffer = use & 1;
      ok = wait_asleep<true>(smem_u32(&bars.parts_in[buffer]), uint32_t(use >> 1) & 1u) && ok;
      const uint32_t base = smem_u32(part + buffer * 8 * NT * outs);
      const int per = (mine + 3) / 4;   // fours of a row; `mine` may be 2
      for (int i = thread; i < rows * per; i += kSumWarps * 32) {
        const int m = i / per, o = rank * mine + (i - m * per) * 4;
        const uint32_t at = base + uint32_t(m * outs + (o & ~3)) * 4u;
        float4 f[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < p.cluster) f[q] = ld_shared_cluster_v4(mapa_shared(at, uint32_t(q)));
        float v[4] = {};
#pragma unroll
        for (int q = 0; q < 8; ++q)   // in k order
          if (q < p.cluster) {
            v[0] += f[q].x; v[1] += f[q].y; v[2] += f[q].z; v[3] += f[q].w;
          }
        if (o & 3) {   // two outputs to a block, the second pair of a four
          v[0] = v[2];
          v[1] = v[3];
        }
        store(item, m, o, v, mine);
      }
      signal(&bars.parts_out[buffer]);
    };
    int use = 0, before = -1;
    for (int item = 0; item < items; ++item, ++use) {
      ok = wait_asleep<false>(meet_full, uint32_t(use) & 1u) && ok;
      const int buffer = use & 1;
      if (p.cluster > 1 && use >= 2) ok = wait_asleep<true>(smem_u32(&bars.parts_out[buffer]), uint32_t((use >> 1) - 1) & 1u) && ok;
      for (int i = thread; i < rows * (outs / 4); i += kSumWarps * 32) {
        const int m = i / (outs / 4), o = (i - m * (outs / 4)) * 4;
        const float *at = meet + o / kOuts * p.wk * kMeet + m * kMeetRow + o % kOuts;
        float v[4] = {};
#pragma unroll 4
        for (int w = 0; w < p.wk; ++w) {
          const float4 f = *reinterpret_cast<const float4 *>(at + w * kMeet);
          v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        }
        if (p.cluster > 1) *reinterpret_cast<float4 *>(part + (buffer * 8 * NT + m) * outs + o) = make_float4(v[0], v[1], v[2], v[3]);
        else store(item, m, o, v, 4);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(meet_empty);
      if (p.cluster > 1) {
        signal(&bars.parts_in[buffer]);
        if (before >= 0) finish(before, use - 1);   // one item late: everybody's part has come meanwhile
        before = item;
      }
    }
    if (before >= 0) finish(before, use - 1);
    complain(p.error, ok, ERR_WAIT_PARTS);
  } else {
    // ------------------------------------------------------------------ this warp's stream of weights
    const int warp_k = warp % p.wk, turns = max(0, (here - warp_k + p.wk - 1) / p.wk);
    const int64_t tile_bytes = int64_t(p.kblocks) * kBlock, turn_bytes = int64_t(p.wk) * kBlock;
    uint8_t *ring = smem + warp * p.stages * kStage;
    const uint32_t ring_s = smem_u32(ring) + lane * 16;
    int ask_item = 0, ask_turn = 0, ask_tiles = 0;
    const uint8_t *ask = nullptr;
    auto ask_next = [&]() {
      const int tile = tile_of(warp, ask_item);
      ask_turn = turns;
      ask_tiles = turns > 0 && ask_item < items ? max(0, min(RT, last - tile)) : 0;
      ask = p.packed + tile * tile_bytes + int64_t(kb0 + warp_k) * kBlock + lane * 16;
      ++ask_item;
    };
    auto issue = [&](int st) {   // the next block, if there is one
      if (ask_tiles > 0) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if (t < ask_tiles) {
            const uint32_t dst = ring_s + st * kStage + t * kBlock;
            const uint8_t *from = ask + t * tile_bytes;
            cp_async_16(dst, from, 16);
            cp_async_16(dst + 512, from + 512, 16);
            if (lane * 16 < kBlock - kCodes) cp_async_16(dst + 1024, from + 1024, 16);
          }
        }
        ask += turn_bytes;
        if (--ask_turn == 0) ask_next();
      }
      cp_async_commit();
    };
    auto arrived = [&]() {   // the oldest block asked for
      if (p.stages == 4) cp_async_wait<3>();
      else if (p.stages == 3) cp_async_wait<2>();
      else cp_async_wait<1>();
      __syncwarp();
    };
    ask_next();
    for (int i = 0; i < p.stages; ++i) issue(i);
    // ------------------------------------------------------------------ x into shared memory, a warp to two k blocks of a row
    {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(p.x), hi = reinterpret_cast<uintptr_t>(p.x + (p.M - 1) * p.ldx + p.K);
      const int row_pairs = (p.share + 1) / 2, pieces = p.share * (kBlockK / 8);
      constexpr int kBatch = 4;   // loads under way at a time
      int m = 0, pair = warp;
      while (m < rows) {
        uint4 held[kBatch];
        int row[kBatch], piece[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          while (m < rows && pair >= row_pairs) {
            pair -= row_pairs;
            ++m;
          }
          row[b] = m;
          piece[b] = pair * 32 + lane;
          const int64_t k = int64_t(kb0) * kBlockK + piece[b] * 8;
          held[b] = make_uint4(0, 0, 0, 0);
          if (m < rows && piece[b] < pieces && k < p.K) held[b] = load_piece(p.x + (m0 + m) * p.ldx + k, p.K - k, lo, hi);
          pair += kW4Warps;
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (row[b] >= rows) break;
          uint4 u = held[b];
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
          float lift = 1.f, down = 1.f, factor = 1.f;
          if constexpr (BF16) {
            // magnitudes compare like their bits; the largest of the k block lies in [2^(e + 14), 2^(e + 15))
            uint32_t big2 = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) big2 = __vmaxu2(big2, __shfl_xor_sync(0xFFFFFFFFu, big2, d));
            const int field = int(max(big2 & 0xFFFFu, big2 >> 16) >> 7), e = field == 255 ? 0 : max(field, 1) - 127 - 14;
            const int first = e < -100 ? 60 : 0;   // a scale beyond f32's range in two steps
            lift = __uint_as_float(uint32_t(127 + first) << 23);
            down = __uint_as_float(uint32_t(127 - e - first) << 23);
            factor = __uint_as_float(e >= -126 ? uint32_t(127 + e) << 23 : 1u << (149 + e));
          }
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = half_to_f32<BF16>((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
            if (BF16) v[e] = v[e] * lift * down;
          }
          float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
          if constexpr (BF16) u = make_uint4(pack_half2<false>(v[0], v[1]), pack_half2<false>(v[2], v[3]), pack_half2<false>(v[4], v[5]), pack_half2<false>(v[6], v[7]));
#pragma unroll
          for (int d = 1; d < kGroup / 8; d <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
          if (piece[b] < pieces) {
            *reinterpret_cast<uint4 *>(x + row[b] * pitch + piece[b] * 16) = u;
            if (lane % (kGroup / 8) == 0) table[piece[b] / (kGroup / 8) * (rows + 1) + row[b]] = make_float2(factor, sum * (ZEROS ? -kUnit : -8.f * kUnit));
          }
        }
      }
      for (int i = threadIdx.x; i < pitch / 16; i += kMulThreads) *reinterpret_cast<uint4 *>(x + rows * pitch + i * 16) = make_uint4(0, 0, 0, 0);
      for (int i = threadIdx.x; i < p.share * GPB; i += kMulThreads) table[i * (rows + 1) + rows] = make_float2(0.f, 0.f);
      asm volatile("bar.sync 1, %0;" ::"n"(kMulThreads) : "memory");
    }
    // ------------------------------------------------------------------ products
    const uint8_t *xrow[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xrow[n] = x + min(n * 8 + r, rows) * pitch + warp_k * kBlockK * 2 + c * 16;
    const int col0 = min(2 * c, rows), col1 = min(2 * c + 1, rows), col2 = min(2 * c + 8, rows), col3 = min(2 * c + 9, rows);
    const int x_turn = p.wk * kBlockK * 2, table_turn = (p.wk - 1) * GPB * (rows + 1);
    float *own = meet + warp * kMeet + 2 * c * kMeetRow + r;
    int st = 0;
    uint32_t meet_parity = 1;   // the first item finds the place free
    bool ok = true;
    for (int item = 0; item < items; ++item) {
      float acc[RT][NT][4] = {};
      const int todo = tile_of(warp, item) < last ? turns : 0;
      const uint8_t *xt[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) xt[n] = xrow[n];
      const float2 *tab = table + warp_k * GPB * (rows + 1);
#pragma unroll 1
      for (int turn = 0; turn < todo; ++turn) {
        arrived();
        const uint8_t *block = ring + st * kStage;
        uint4 w4[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) w4[t][h] = *reinterpret_cast<const uint4 *>(block + t * kBlock + h * 512 + lane * 16);
        // scales of outputs r and r + 8, all groups of the block
        uint32_t scale[RT][2][(GPB + 1) / 2], zero[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t *from = block + t * kBlock + kCodes + (r + 8 * h) * GPB * 2, *zfrom = block + t * kBlock + kCodes + GPB * kRows * 2 + (r + 8 * h) * GPB;
            if constexpr (GPB == 1) {
              scale[t][h][0] = *reinterpret_cast<const uint16_t *>(from);
              zero[t][h] = ZEROS ? *zfrom : 0u;
            } else if constexpr (GPB == 2) {
              scale[t][h][0] = *reinterpret_cast<const uint32_t *>(from);
              zero[t][h] = ZEROS ? *reinterpret_cast<const uint16_t *>(zfrom) : 0u;
            } else {
              const uint2 u = *reinterpret_cast<const uint2 *>(from);
              scale[t][h][0] = u.x;
              scale[t][h][1] = u.y;
              zero[t][h] = ZEROS ? *reinterpret_cast<const uint32_t *>(zfrom) : 0u;
            }
          }
        __syncwarp();
        issue(st);   // all of the stage is in registers
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
          float sum[RT][NT][4];
          // acc += scale factor (sum x code - zero sum x);  the second term is what the products start from
          float2 xs[NT][2];   // columns 2 c and 2 c + 1
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            xs[n][0] = tab[n ? col2 : col0];
            xs[n][1] = tab[n ? col3 : col1];
          }
          tab += rows + 1;
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float z = ZEROS ? (__uint_as_float(0x4B000000u | ((zero[t][h] >> (8 * g)) & 0xFFu)) - 8388608.f) * (h ? 16.f : 1.f) : (h ? 16.f : 1.f);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) sum[t][n][2 * h + i] = xs[n][i].y * z;
            }
#pragma unroll
          for (int q = g * 4 / GPB; q < (g + 1) * 4 / GPB; ++q) {   // 32 k
            uint32_t b[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 u = *reinterpret_cast<const uint4 *>(xt[n] + q * 64);
              b[n][0] = u.x; b[n][1] = u.y; b[n][2] = u.z; b[n][3] = u.w;
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              const uint4 &u = w4[t][q >> 1];
              const uint32_t w[2] = {q & 1 ? u.z : u.x, q & 1 ? u.w : u.y};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t v = __byte_perm(w[h], 0, 0x2301);
                const uint32_t a[4] = {w[h] & 0x003C003Cu, w[h] & 0x03C003C0u, v & 0x003C003Cu, v & 0x03C003C0u};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816<false>(sum[t][n], a, b[n][2 * h], b[n][2 * h + 1]);
              }
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float s = half_to_f32<BF16>((scale[t][h][g / 2] >> (16 * (g & 1))) & 0xFFFFu) * (h ? 0.0625f / kUnit : 1.f / kUnit);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[t][n][2 * h + i] = BF16 ? fmaf(sum[t][n][2 * h + i] * s, xs[n][i].x, acc[t][n][2 * h + i]) : fmaf(sum[t][n][2 * h + i], s, acc[t][n][2 * h + i]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) xt[n] += x_turn;
        tab += table_turn;
        if (++st == p.stages) st = 0;
      }
      // ---- [warp][rows of x][outputs]
      if (!mbar_wait(meet_empty, meet_parity)) ok = false;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) own[(n * 8 + (i & 1)) * kMeetRow + t * 16 + 8 * (i >> 1)] = acc[t][n][i];
      __syncwarp();
      if (lane == 0) mbar_arrive(meet_full);
      meet_parity ^= 1u;
    }
    complain(p.error, ok, ERR_WAIT_EMPTY);
  }
  if (p.cluster > 1) {
    __syncwarp();
    cluster_sync_all();   // nobody leaves while others read its sums
  }
}

void checked_w4(int64_t N, int64_t K, int64_t group) {
  require(N > 0 && K > 0 && N < (int64_t(1) << 31) && K < (int64_t(1) << 31), "4-bit weights: sizes must be positive");
  require(group == 32 || group == 64 || (group > 0 && group % kBlockK == 0), "4-bit weights: group must be 32, 64 or a multiple of 128");
}

template <bool BF16, int NT, int RT, int GPB, bool ZEROS> struct W4Kernel {
  static void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute (&at)[2], int grid_x, int grid_y, int cluster, size_t smem, cudaStream_t stream) {
    cfg = {};
    cfg.gridDim = dim3(unsigned(grid_x), unsigned(grid_y), 1u);
    cfg.blockDim = dim3(kW4Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = unsigned(cluster);
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
  }
  static void run(const W4Params &p, const W4Plan &plan, int grid_y, int device, cudaStream_t stream) {
    static bool ready[64] = {};
    auto kernel = matmul_w4_kernel<BF16, NT, RT, GPB, ZEROS>;
    if (!ready[device & 63]) {
      GCB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
      ready[device & 63] = true;
    }
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute at[2];
    configure(cfg, at, plan.cluster * plan.clusters, grid_y, plan.cluster, size_t(plan.smem), stream);
    GCB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    count_launch();
  }
};

template <bool BF16, int NT, int RT> void launch(const W4Params &p, const W4Plan &plan, int gpb, bool zeros, int grid_y, int device, cudaStream_t stream) {
  if (zeros) gpb == 1 ? W4Kernel<BF16, NT, RT, 1, true>::run(p, plan, grid_y, device, stream) : gpb == 2 ? W4Kernel<BF16, NT, RT, 2, true>::run(p, plan, grid_y, device, stream)
                                                                                                         : W4Kernel<BF16, NT, RT, 4, true>::run(p, plan, grid_y, device, stream);
  else gpb == 1 ? W4Kernel<BF16, NT, RT, 1, false>::run(p, plan, grid_y, device, stream) : gpb == 2 ? W4Kernel<BF16, NT, RT, 2, false>::run(p, plan, grid_y, device, stream)
                                                                                                    : W4Kernel<BF16, NT, RT, 4, false>::run(p, plan, grid_y, device, stream);
}

// Clusters of each size that a device runs at the same time, one block to an SM.
const int *clusters_at_once(const DeviceState &dev) {
  struct State {
    std::once_flag once;
    int at_once[9] = {};
  };
  static State states[64];
  State &s = states[dev.device & 63];
  std::call_once(s.once, [&] {
    using Kernel = W4Kernel<true, 1, 2, 1, false>;
    auto kernel = matmul_w4_kernel<true, 1, 2, 1, false>;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
    s.at_once[1] = dev.sm_count;
    for (int n = 2; n <= 8; n *= 2) {
      cudaLaunchConfig_t cfg;
      cudaLaunchAttribute at[2];
      Kernel::configure(cfg, at, n, 1, n, kMostSmem, nullptr);
      int k = 0;
      if (cudaOccupancyMaxActiveClusters(&k, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        k = 0;
      }
      s.at_once[n] = k;
    }
  });
  return s.at_once;
}

} // namespace

size_t w4_packed_bytes(int64_t N, int64_t K, int64_t group, int has_zeros) {
  checked_w4(N, K, group);
  return size_t((N + kRows - 1) / kRows) * size_t((K + kBlockK - 1) / kBlockK) * size_t(block_bytes(group, has_zeros != 0));
}

void w4_pack(const uint8_t *codes, int64_t codes_stride, const void *scales, int64_t scales_stride, const uint8_t *zeros,
             int64_t zeros_stride, int64_t N, int64_t K, int64_t group, void *packed, cudaStream_t stream) {
  checked_w4(N, K, group);
  require(codes && scales && packed, "4-bit weights: null pointer");
  require((reinterpret_cast<uintptr_t>(packed) & 15) == 0, "4-bit weights: the packed buffer must be 16-byte aligned");
  require((reinterpret_cast<uintptr_t>(scales) & 1) == 0, "4-bit weights: misaligned scales");
  device_state();
  W4PackParams p{};
  p.codes = codes;
  p.zeros = zeros;
  p.scales = static_cast<const uint16_t *>(scales);
  p.codes_stride = codes_stride;
  p.scales_stride = scales_stride;
  p.zeros_stride = zeros_stride;
  p.N = N;
  p.K = K;
  p.group = group;
  p.packed = static_cast<uint8_t *>(packed);
  p.kblocks = (K + kBlockK - 1) / kBlockK;
  p.gpb = groups_per_block(group);
  p.bytes = block_bytes(group, zeros != nullptr);
  const int64_t tiles = (N + kRows - 1) / kRows, y = std::min<int64_t>(tiles, 32768);
  const dim3 grid{unsigned((p.kblocks + kPackBlocks - 1) / kPackBlocks), unsigned(y), unsigned((tiles + y - 1) / y)};
  w4_pack_kernel<<<grid, kPackBlocks * 64, 0, stream>>>(p);
  GCB_CUDA(cudaGetLastError());
  count_launch();
}

void matmul_w4(int dtype, const void *X, int64_t ldx, const void *packed, const void *bias, void *Y, int64_t ldy, int64_t M,
               int64_t N, int64_t K, int64_t group, int has_zeros, int relu, cudaStream_t stream) {
  checked_w4(N, K, group);
  require(dtype == GCB200_BF16 || dtype == GCB200_F16, "4-bit weights: x must be bf16 or f16");
  require(M >= 0 && M < (int64_t(1) << 31), "4-bit weights: number of rows out of range");
  if (M == 0) return;
  require(X && packed && Y, "4-bit weights: null pointer");
  require((reinterpret_cast<uintptr_t>(packed) & 15) == 0, "4-bit weights: the packed buffer must be 16-byte aligned");
  require(aligned(X, 2) && aligned(bias, 2) && aligned(Y, 2), "4-bit weights: misaligned pointer");
  require(M == 1 || (ldx >= K && ldy >= N), "4-bit weights: rows overlap");
  DeviceState &dev = device_state();
  const int kblocks = int((K + kBlockK - 1) / kBlockK), tiles = int((N + kRows - 1) / kRows);
  const int gpb = groups_per_block(group), bytes = block_bytes(group, has_zeros != 0);
  W4Plan plan{};
  if (!plan_w4(int(M), tiles, kblocks, gpb, bytes, clusters_at_once(dev), &plan)) throw std::logic_error("4-bit weights: a row of x does not fit into the shared memory of a cluster");
  W4Params p{};
  p.bias = static_cast<const uint16_t *>(bias);
  p.packed = static_cast<const uint8_t *>(packed);
  p.ldx = M > 1 ? ldx : 0;
  p.ldy = M > 1 ? ldy : 0;
  p.N = N;
  p.K = K;
  p.pass = plan.pass;
  p.relu = relu;
  p.kblocks = kblocks;
  p.tiles = tiles;
  p.cluster = plan.cluster;
  p.share = plan.share;
  p.wk = plan.wk;
  p.stages = plan.stages;
  p.x_at = plan.x_at;
  p.table_at = plan.table_at;
  p.meet_at = plan.meet_at;
  p.part_at = plan.part_at;
  p.error = dev.d_error;
  const int64_t most = int64_t(65535) * plan.pass;   // rows of a launch: a grid has that many passes
  for (int64_t m = 0; m < M; m += most) {
    p.x = static_cast<const uint16_t *>(X) + m * p.ldx;
    p.y = static_cast<uint16_t *>(Y) + m * p.ldy;
    p.M = int(std::min(most, M - m));
    const int grid_y = (p.M + plan.pass - 1) / plan.pass;
    auto go = [&](auto bf16) {
      constexpr bool B = decltype(bf16)::value;
      if (plan.nt == 1) plan.rt == 2 ? launch<B, 1, 2>(p, plan, gpb, has_zeros != 0, grid_y, dev.device, stream) : launch<B, 1, 1>(p, plan, gpb, has_zeros != 0, grid_y, dev.device, stream);
      else plan.rt == 2 ? launch<B, 2, 2>(p, plan, gpb, has_zeros != 0, grid_y, dev.device, stream) : launch<B, 2, 1>(p, plan, gpb, has_zeros != 0, grid_y, dev.device, stream);
    };
    dtype == GCB200_BF16 ? go(std::true_type{}) : go(std::false_type{});
  }
}

} // namespace gcb
