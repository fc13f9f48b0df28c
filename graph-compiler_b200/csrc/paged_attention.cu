// Attention of one new token per sequence over a paged key-value cache:
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - m),  m = max_t scale q . k_t
// with the running maximum and sum of an online softmax, so that keys and values are read once.
//
// Bound by HBM: 2 head_dim elements of cache per token and KV head for 4 head_dim operations per query head.
#include "decode_ops.h"

#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "mma_ptx.cuh"
#include "runtime.h"

namespace gcb {

namespace {

constexpr int kWarps = 4;

struct PagedAttParams {
  PagedCache c;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_seq, q_head, o_seq, o_head;   // elements
  const int32_t *lengths;
  float *lse;
  float scale;
  int heads, group, window;
};

template <bool BF16, bool F8> __device__ __forceinline__ void load8(const uint8_t *p, float (&x)[8]) {
  if constexpr (F8) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t h = e4m3x2_to_f16x2((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
      x[2 * i] = half_to_f32<false>(h & 0xFFFFu);
      x[2 * i + 1] = half_to_f32<false>(h >> 16);
    }
  } else {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = half_to_f32<BF16>(w[i] & 0xFFFFu);
      x[2 * i + 1] = half_to_f32<BF16>(w[i] >> 16);
    }
  }
}

// One block per sequence and query head; a warp per token, eight elements of head_dim to a lane.
template <bool BF16, bool F8>
__global__ void __launch_bounds__(kWarps * 32) paged_attention_kernel(const __grid_constant__ PagedAttParams p) {
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][256];
  const PagedCache &c = p.c;
  const int s = blockIdx.y, h = blockIdx.x, kvh = h / p.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Seen see = seen_of(c.table, p.lengths[s], p.window);
  const int first = see.first, len = see.end;
  if (see.cut && threadIdx.x == 0) atomicExch(c.error, int(ERR_BAD_PAGE));
  const float ks = F8 && c.key_scale ? c.key_scale[kvh] : 1.f, vs = F8 && c.value_scale ? c.value_scale[kvh] : 1.f;
  const int d0 = lane * 8;
  const bool mine = d0 < c.dim;
  const int size = F8 ? 1 : 2;
  float q[8], o[8] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = mine ? half_to_f32<BF16>(p.q[s * p.q_seq + h * p.q_head + d0 + i]) * p.scale * ks : 0.f;
  for (int t = first + warp; t < len; t += kWarps) {
    const int page = page_of(c.table, s, t), slot = t % c.table.page_size;
    const bool held = page >= 0;
    if (!held && lane == 0) atomicExch(c.error, int(ERR_BAD_PAGE));
    float k[8] = {}, v[8] = {};
    if (held && mine) {
      load8<BF16, F8>(c.keys + page * c.key_page + kvh * c.key_head + slot * c.key_token + d0 * size, k);
      load8<BF16, F8>(c.values + page * c.value_page + kvh * c.value_head + slot * c.value_token + d0 * size, v);
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = fmaf(q[i], k[i], dot);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, i);
    const float mn = fmaxf(m, dot), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = __expf(m - base), w = __expf(dot - base);
    m = mn;
    l = l * alpha + w;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf(w, v[i], o[i] * alpha);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][d0 + i] = o[i];
  __syncthreads();
  float mx = -INFINITY, total = 0.f;
  for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[w]);
  const float base = mx == -INFINITY ? 0.f : mx;
  for (int w = 0; w < kWarps; ++w) total += sl[w] * __expf(sm[w] - base);
  for (int d = threadIdx.x; d < c.dim; d += kWarps * 32) {
    float sum = 0.f;
    for (int w = 0; w < kWarps; ++w) sum += so[w][d] * __expf(sm[w] - base);
    p.out[s * p.o_seq + h * p.o_head + d] = f32_to_half<BF16>(len > first ? sum / total * vs : 0.f);
  }
  if (p.lse && threadIdx.x == 0) p.lse[int64_t(s) * p.heads + h] = base + logf(total);
}

void require(bool ok, const char *what) {
  if (!ok) throw std::invalid_argument(what);
}

} // namespace

size_t paged_attention_workspace(int64_t heads, int64_t kv_heads, int64_t head_dim) {
  require(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads < 65536, "paged attention: heads must be a multiple of kv_heads");
  require(head_dim > 0 && head_dim <= 256, "paged attention: head_dim must be at most 256");
  return 16;
}

void paged_attention(const gcb200_paged_cache &cache, const PagedAttentionArgs &a, cudaStream_t stream) {
  PagedAttParams p{};
  p.c = checked_cache(cache, false);
  require(cache.sequences == 0 || (a.q && a.out && a.lengths && a.workspace), "paged attention: null pointer");
  require((reinterpret_cast<uintptr_t>(a.workspace) & 15) == 0, "paged attention: the workspace must be 16-byte aligned");
  require(a.workspace_bytes >= paged_attention_workspace(a.heads, cache.kv_heads, cache.head_dim), "paged attention: the workspace is too small");
  require(a.window >= 0, "paged attention: negative window");
  require(cache.sequences < 65536, "paged attention: more than 65535 sequences");
  if (cache.sequences == 0) return;
  DeviceState &dev = device_state();
  p.c.error = dev.d_error;
  p.q = static_cast<const uint16_t *>(a.q);
  p.out = static_cast<uint16_t *>(a.out);
  p.q_seq = a.q_stride[0];
  p.q_head = a.q_stride[1];
  p.o_seq = a.out_stride[0];
  p.o_head = a.out_stride[1];
  p.lengths = a.lengths;
  p.lse = a.lse;
  p.scale = a.scale;
  p.heads = int(a.heads);
  p.group = int(a.heads / cache.kv_heads);
  p.window = int(std::min<int64_t>(a.window, INT32_MAX));
  const dim3 grid(unsigned(a.heads), unsigned(cache.sequences));
  const bool bf16 = cache.dtype == GCB200_BF16, f8 = cache.cache_dtype == GCB200_F8_E4M3;
  (bf16 ? (f8 ? paged_attention_kernel<true, true> : paged_attention_kernel<true, false>)
        : (f8 ? paged_attention_kernel<false, true> : paged_attention_kernel<false, false>))<<<grid, kWarps * 32, 0, stream>>>(p);
  GCB_CUDA(cudaGetLastError());
  count_launch();
}

} // namespace gcb
