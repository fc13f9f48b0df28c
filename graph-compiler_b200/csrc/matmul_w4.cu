// Linear layers of a few rows with 4-bit weights:  Y = act(X . W^T + bias),  W[n][k] = (code - zero) * scale of n's group.
//
// Layout.  The weights are packed once into blocks of 16 outputs x 128 k, in the order in which a warp's matrix instruction
// takes them: 1024 bytes of codes (lane l reads 16 bytes at 16 l of each half), the scales of the 16 outputs for each of the
// block's groups, and their zeros.  The k range of an output tile is one contiguous stream.
//
// Codes become 16-bit floats without a conversion: four bits or-ed into the mantissa of 128 (bf16) or 1024 (f16) are that
// number plus the code, and subtracting (128 or 1024) + zero is exact.  Products with X then are exact in f32, sums are f32, and
// a group's scale multiplies the f32 sum of its products.
//
// Bound by HBM: half a byte per weight.
#include "decode_ops.h"

#include <algorithm>
#include <stdexcept>

#include "mma_ptx.cuh"
#include "runtime.h"

namespace gcb {

namespace {

constexpr int kRows = 16;      // outputs of a tile: M of the matrix instruction
constexpr int kBlockK = 128;
constexpr int kCodes = kRows * kBlockK / 2;
constexpr int kW4Warps = 8;

void require(bool ok, const char *what) {
  if (!ok) throw std::invalid_argument(what);
}
int groups_per_block(int64_t group) { return group >= kBlockK ? 1 : int(kBlockK / group); }
int block_bytes(int64_t group, bool zeros) { return kCodes + groups_per_block(group) * kRows * (zeros ? 3 : 2); }

struct W4PackParams {
  const uint8_t *codes, *zeros;
  const uint16_t *scales;
  int64_t codes_stride, scales_stride, zeros_stride, N, K, group;
  uint8_t *packed;
  int64_t kblocks;
  int gpb, bytes;
};

// One block of 256 threads packs one 16 x 128 block; a thread one 32-bit word.  Word w of a lane in half h covers
// k = 64 h + 32 (w >> 1) + 8 c + 4 (w & 1) + {0, 1, 2, 3} of outputs r and r + 8 (r = lane / 4, c = lane % 4).
__global__ void __launch_bounds__(256) w4_pack_kernel(const __grid_constant__ W4PackParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t kb = blockIdx.x, nt = blockIdx.y + int64_t(blockIdx.z) * gridDim.y;
  if (nt * kRows >= p.N) return;
  uint8_t *block = p.packed + (nt * p.kblocks + kb) * p.bytes;
  const int t = threadIdx.x, h = t >> 7, lane = (t >> 2) & 31, w = t & 3, r = lane >> 2, c = lane & 3;
  const int64_t k0 = kb * kBlockK + 64 * h + 32 * (w >> 1) + 8 * c + 4 * (w & 1);
  auto code = [&](int64_t n, int64_t k) -> uint32_t {
    if (n >= p.N) return 8u;
    if (k >= p.K) return p.zeros ? 0u : 8u;   // meets an x of zero
    const uint32_t b = p.codes[n * p.codes_stride + (k >> 1)];
    return (k & 1) ? b >> 4 : b & 15u;
  };
  uint32_t word = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) {   // nibbles s and s + 4: one register of the instruction's A operand
    const int64_t n = nt * kRows + r + 8 * (s & 1), k = k0 + 2 * (s >> 1);
    word |= code(n, k) << (4 * s) | code(n, k + 1) << (4 * s + 16);
  }
  reinterpret_cast<uint32_t *>(block)[h * 128 + lane * 4 + w] = word;
  if (t < p.gpb * kRows) {
    const int64_t n = nt * kRows + (t & 15), g = (kb * kBlockK + int64_t(t >> 4) * (kBlockK / p.gpb)) / p.group;
    const bool in = n < p.N && g * p.group < p.K;
    reinterpret_cast<uint16_t *>(block + kCodes)[t] = in ? p.scales[n * p.scales_stride + g] : uint16_t(0);
    if (p.zeros) block[kCodes + p.gpb * kRows * 2 + t] = in ? uint8_t(p.zeros[n * p.zeros_stride + g] & 15u) : uint8_t(8);
  }
}

struct W4Params {
  const uint16_t *x, *bias;
  const uint8_t *packed;
  uint16_t *y;
  int64_t ldx, ldy, N, K, kblocks;
  int M, relu, bytes;
};

template <bool BF16> __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A block of eight warps per 16 outputs and 8 rows of x; the warps take every eighth k block and their sums meet in shared memory.
template <bool BF16, int GPB, bool ZEROS>
__global__ void __launch_bounds__(kW4Warps * 32) matmul_w4_kernel(const __grid_constant__ W4Params p) {
  __shared__ float sums[kW4Warps][kRows][9];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int64_t nt = blockIdx.x;
  const int m = blockIdx.y * 8 + r;
  const uint32_t magic = BF16 ? 0x43004300u : 0x64006400u;
  float acc[4] = {};
  for (int64_t kb = warp; kb < p.kblocks; kb += kW4Warps) {
    const uint8_t *block = p.packed + (nt * p.kblocks + kb) * p.bytes;
    const uint16_t *scales = reinterpret_cast<const uint16_t *>(block + kCodes);
    const uint8_t *zeros = block + kCodes + GPB * kRows * 2;
#pragma unroll
    for (int g = 0; g < GPB; ++g) {
      float part[4] = {};
      const uint32_t z0 = magic + (ZEROS ? zeros[g * 16 + r] : 8u) * 0x10001u, z1 = magic + (ZEROS ? zeros[g * 16 + r + 8] : 8u) * 0x10001u;
#pragma unroll
      for (int s = g * 8 / GPB; s < (g + 1) * 8 / GPB; ++s) {   // sixteen k to a step
        const uint32_t w = reinterpret_cast<const uint32_t *>(block)[(s >> 2) * 128 + lane * 4 + (s & 3)];
        const int64_t k = kb * kBlockK + (s >> 1) * 32 + 8 * c + 4 * (s & 1);
        uint32_t b[2] = {0u, 0u};
        if (m < p.M) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k + i < p.K) b[i >> 1] |= uint32_t(p.x[m * p.ldx + k + i]) << (16 * (i & 1));
        }
        const uint32_t a[4] = {sub2<BF16>((w & 0x000F000Fu) | magic, z0), sub2<BF16>(((w >> 4) & 0x000F000Fu) | magic, z1),
                               sub2<BF16>(((w >> 8) & 0x000F000Fu) | magic, z0), sub2<BF16>(((w >> 12) & 0x000F000Fu) | magic, z1)};
        mma_16816<BF16>(part, a, b[0], b[1]);
      }
      const float s0 = half_to_f32<BF16>(scales[g * 16 + r]), s1 = half_to_f32<BF16>(scales[g * 16 + r + 8]);
      acc[0] = fmaf(part[0], s0, acc[0]);
      acc[1] = fmaf(part[1], s0, acc[1]);
      acc[2] = fmaf(part[2], s1, acc[2]);
      acc[3] = fmaf(part[3], s1, acc[3]);
    }
  }
  sums[warp][r][2 * c] = acc[0];
  sums[warp][r][2 * c + 1] = acc[1];
  sums[warp][r + 8][2 * c] = acc[2];
  sums[warp][r + 8][2 * c + 1] = acc[3];
  __syncthreads();
  if (threadIdx.x < 128) {
    const int row = threadIdx.x & 15, col = threadIdx.x >> 4, out_m = blockIdx.y * 8 + col;
    const int64_t n = nt * kRows + row;
    if (n < p.N && out_m < p.M) {
      float y = 0.f;
      for (int w = 0; w < kW4Warps; ++w) y += sums[w][row][col];
      if (p.bias) y += half_to_f32<BF16>(p.bias[n]);
      if (p.relu) y = y != y ? y : fmaxf(y, 0.f);
      p.y[out_m * p.ldy + n] = f32_to_half<BF16>(y);
    }
  }
}

void checked_w4(int64_t N, int64_t K, int64_t group) {
  require(N > 0 && K > 0 && N < (int64_t(1) << 31) && K < (int64_t(1) << 31), "4-bit weights: sizes must be positive");
  require(group == 32 || group == 64 || (group > 0 && group % kBlockK == 0), "4-bit weights: group must be 32, 64 or a multiple of 128");
}

template <bool BF16> void launch(const W4Params &p, int gpb, bool zeros, dim3 grid, cudaStream_t stream) {
  auto go = [&](auto kernel) { kernel<<<grid, kW4Warps * 32, 0, stream>>>(p); };
  if (zeros) gpb == 1 ? go(matmul_w4_kernel<BF16, 1, true>) : gpb == 2 ? go(matmul_w4_kernel<BF16, 2, true>) : go(matmul_w4_kernel<BF16, 4, true>);
  else gpb == 1 ? go(matmul_w4_kernel<BF16, 1, false>) : gpb == 2 ? go(matmul_w4_kernel<BF16, 2, false>) : go(matmul_w4_kernel<BF16, 4, false>);
  GCB_CUDA(cudaGetLastError());
  count_launch();
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
  w4_pack_kernel<<<dim3(unsigned(p.kblocks), unsigned(y), unsigned((tiles + y - 1) / y)), 256, 0, stream>>>(p);
  GCB_CUDA(cudaGetLastError());
  count_launch();
}

void matmul_w4(int dtype, const void *X, int64_t ldx, const void *packed, const void *bias, void *Y, int64_t ldy, int64_t M,
               int64_t N, int64_t K, int64_t group, int has_zeros, int relu, cudaStream_t stream) {
  checked_w4(N, K, group);
  require(dtype == GCB200_BF16 || dtype == GCB200_F16, "4-bit weights: x must be bf16 or f16");
  require(M >= 0 && M <= 8 * 65535, "4-bit weights: number of rows out of range");
  if (M == 0) return;
  require(X && packed && Y, "4-bit weights: null pointer");
  require((reinterpret_cast<uintptr_t>(packed) & 15) == 0, "4-bit weights: the packed buffer must be 16-byte aligned");
  require(M == 1 || (ldx >= K && ldy >= N), "4-bit weights: rows overlap");
  device_state();
  W4Params p{};
  p.x = static_cast<const uint16_t *>(X);
  p.bias = static_cast<const uint16_t *>(bias);
  p.packed = static_cast<const uint8_t *>(packed);
  p.y = static_cast<uint16_t *>(Y);
  p.ldx = ldx;
  p.ldy = ldy;
  p.N = N;
  p.K = K;
  p.kblocks = (K + kBlockK - 1) / kBlockK;
  p.M = int(M);
  p.relu = relu;
  p.bytes = block_bytes(group, has_zeros != 0);
  const dim3 grid(unsigned((N + kRows - 1) / kRows), unsigned((M + 7) / 8));
  if (dtype == GCB200_BF16) launch<true>(p, groups_per_block(group), has_zeros != 0, grid, stream);
  else launch<false>(p, groups_per_block(group), has_zeros != 0, grid, stream);
}

} // namespace gcb
