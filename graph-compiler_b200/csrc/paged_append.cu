// Appending to a paged key-value cache: k (rotated) and v of new tokens into their pages, q rotated beside them.
//
// A rotation turns pair (a, b) of a query or key by angle = position * inv_freq[i]:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// The angle of a far position has no bits of its fraction left in f32 (position 10^6: the spacing is 0.06), so it is formed in
// f64 in whole turns, reduced by the whole turns there, and only the remaining fraction becomes f32 for sincospi.  All heads of
// a token share its angles: a block computes them once, into shared memory.
//
// Bound by HBM: q read and written, k and v read, the cache's rows written.  Small blocks and few rows under way in a thread leave
// registers for many threads: 8192 tokens of 32 + 2 x 8 heads of 128 (201 MB) 38 us, 5.3 TB/s, with 64 threads and two rows; four
// rows 42, 128 threads and two rows 41, 128 and four 45.  Into 8 bits, 3001 tokens of 28 + 2 x 4 heads of 80 (33 MB): 10.8 us, 59 % of the
// issue slots.
#include "decode_ops.h"

#include <algorithm>
#include <stdexcept>
#include <string>

#include "mma_ptx.cuh"
#include "runtime.h"

namespace gcb {

namespace {

// Threads of a block: at least the pieces of a row (at most 128 of single elements, 64 of two).
template <int VEC> constexpr int kAppendThreads = VEC == 1 ? 128 : 64;
constexpr int kMaxDim = 256;

struct AppendParams {
  PagedCache c;
  const uint16_t *q, *k, *v;
  uint16_t *q_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;   // elements
  const int32_t *sequences, *positions;
  const double *inv_freq;
  int heads, rotary, interleaved, units;   // units: pieces of a row, two chunks each
};

// VEC consecutive 16-bit elements as they lie in memory; ALIGNED: moved in one access.  VEC 1 fills the low half of a word.
template <int VEC> struct Chunk {
  uint32_t w[(VEC + 1) / 2];
};
template <int VEC, bool ALIGNED> __device__ __forceinline__ Chunk<VEC> load(const uint16_t *p) {
  Chunk<VEC> x;
  if constexpr (ALIGNED && VEC == 8) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    x.w[0] = u.x; x.w[1] = u.y; x.w[2] = u.z; x.w[3] = u.w;
  } else if constexpr (ALIGNED && VEC == 4) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    x.w[0] = u.x; x.w[1] = u.y;
  } else if constexpr (VEC == 1) {
    x.w[0] = p[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) x.w[i] = p[2 * i] | (uint32_t(p[2 * i + 1]) << 16);
  }
  return x;
}
template <int VEC, bool ALIGNED> __device__ __forceinline__ void store(uint16_t *p, const Chunk<VEC> &x) {
  if constexpr (ALIGNED && VEC == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
  else if constexpr (ALIGNED && VEC == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(x.w[0], x.w[1]);
  else if constexpr (VEC == 1) p[0] = uint16_t(x.w[0]);
  else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      p[2 * i] = uint16_t(x.w[i]);
      p[2 * i + 1] = uint16_t(x.w[i] >> 16);
    }
  }
}
template <bool BF16, int VEC> __device__ __forceinline__ void unpack(const Chunk<VEC> &c, float (&x)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = half_to_f32<BF16>((c.w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
}
template <bool BF16, int VEC> __device__ __forceinline__ Chunk<VEC> pack(const float (&x)[VEC]) {
  Chunk<VEC> c;
#pragma unroll
  for (int i = 0; i < (VEC + 1) / 2; ++i) c.w[i] = pack_half2<BF16>(x[2 * i], VEC > 1 ? x[VEC > 1 ? 2 * i + 1 : 0] : 0.f);
  return c;
}
// x / scale as a division gives it, from by = 1 / scale: x by is off by a few units in the last place; one step of Newton's method on
// the remainder, which the fused multiply-add keeps whole, rounds it right (Markstein, IBM J. Res. Dev. 34, 1990).  A division takes
// four times the instructions of all the rest.  Without the step, quotients on the border between two codes went to either.  Infinities
// and NaN stay what x by is.
__device__ __forceinline__ float divided(float x, float scale, float by) {
  const float y = x * by, z = fmaf(fmaf(-y, scale, x), by, y);
  return fabsf(y) < 1024.f ? z : y;   // beyond: limited to 448 all the same
}
template <int VEC, bool ALIGNED> __device__ __forceinline__ void store_e4m3(uint8_t *p, float (&x)[VEC], float scale, float by) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = divided(x[i], scale, by);
  if constexpr (ALIGNED) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) w[i] = f32x2_to_e4m3x2(x[4 * i], x[4 * i + 1]) | (f32x2_to_e4m3x2(x[4 * i + 2], x[4 * i + 3]) << 16);
    if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t *>(p) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = uint8_t(f32x2_to_e4m3x2(x[i], 0.f));
  }
}

// One block per token.  A thread has the same piece of every row it takes - two chunks of VEC elements, the partners of a rotation by
// halves or neighbours - so that it loads its cosines and sines once; it asks for kBatch rows at a time, the first ones before
// the angles are there.
template <bool BF16, bool F8, int VEC, bool ALIGNED>
__global__ void __launch_bounds__(kAppendThreads<VEC>) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kThreads = kAppendThreads<VEC>;
  __shared__ float2 turn[kMaxDim / 2];   // (cos, sin) of each pair
  pdl_wait();
  pdl_launch_dependents();
  const PagedCache &c = p.c;
  const int64_t t = blockIdx.x;
  const int seq = p.sequences ? p.sequences[t] : int(t), pos = p.positions[t];
  if (seq < 0 || pos < 0) return;   // padding

  const int half = p.rotary >> 1, q_rows = p.q ? p.heads : 0, rows = q_rows + 2 * c.kv_heads;
  const int row_step = kThreads / p.units, row0 = int(threadIdx.x) / p.units, piece = int(threadIdx.x) - row0 * p.units;
  // Where the piece lies in a rotated row and in a row that is only copied.
  const bool halves = p.rotary > 0 && !p.interleaved, partners = halves && piece * VEC < half;
  const int rot0 = partners ? piece * VEC : halves ? p.rotary + 2 * (piece - half / VEC) * VEC : 2 * piece * VEC, rot1 = rot0 + (partners ? half : VEC);
  const int copy0 = 2 * piece * VEC, copy1 = copy0 + VEC;

  constexpr int kBatch = 2;
  Chunk<VEC> a[kBatch], b[kBatch];
  auto fetch = [&](int first) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int row = first + i * row_step;
      if (row0 < row_step && row < rows) {
        const bool copied = row >= q_rows + c.kv_heads;
        const uint16_t *src = row < q_rows ? p.q + t * p.q_token + row * p.q_head
                              : copied     ? p.v + t * p.v_token + (row - q_rows - c.kv_heads) * p.v_head
                                           : p.k + t * p.k_token + (row - q_rows) * p.k_head;
        const int d0 = copied ? copy0 : rot0, d1 = copied ? copy1 : rot1;
        if (d0 < c.dim) a[i] = load<VEC, ALIGNED>(src + d0);
        if (d1 < c.dim) b[i] = load<VEC, ALIGNED>(src + d1);
      }
    }
  };
  fetch(row0);
  for (int i = threadIdx.x; i < half; i += kThreads) {
    const double turns = double(pos) * p.inv_freq[i] * 0.15915494309189533577;   // 1 / (2 pi)
    float s, co;
    sincospif(2.f * float(turns - rint(turns)), &s, &co);
    turn[i] = make_float2(co, s);
  }
  const int slot = pos % c.table.page_size, page = page_of(c.table, seq, pos);
  if (page < 0 && threadIdx.x == 0) report_bad_page(c.error);
  __syncthreads();
  // this piece's pairs: element i of one chunk and of the other, or neighbours within a chunk
  float cs[VEC], sn[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int at = partners ? rot0 + i : ((i < VEC / 2 ? rot0 : rot1) >> 1) + (VEC > 1 ? i % ((VEC + 1) / 2) : 0);
    const float2 w = turn[partners || (p.interleaved && at < half) ? at : 0];   // unused where the piece does not turn
    cs[i] = w.x;
    sn[i] = w.y;
  }
  const bool turns = partners || (p.rotary > 0 && p.interleaved);

  for (int first = row0; first < rows; first += kBatch * row_step) {
    if (first != row0) fetch(first);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int row = first + i * row_step;
      if (row0 >= row_step || row >= rows) continue;
      const bool cached = row >= q_rows, copied = row >= q_rows + c.kv_heads;
      if (cached && page < 0) continue;
      const int d0 = copied ? copy0 : rot0, d1 = copied ? copy1 : rot1, head = copied ? row - q_rows - c.kv_heads : row - q_rows;
      uint8_t *dst = !cached ? reinterpret_cast<uint8_t *>(p.q_out + t * p.o_token + row * p.o_head)
                     : copied ? c.values + page * c.value_page + head * c.value_head + slot * c.value_token
                              : c.keys + page * c.key_page + head * c.key_head + slot * c.key_token;
      Chunk<VEC> ca = a[i], cb = b[i];
      if ((turns && !copied) || (F8 && cached)) {
        float x[VEC], y[VEC];
        unpack<BF16, VEC>(ca, x);
        unpack<BF16, VEC>(cb, y);
        if (!copied) {
          if (partners) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float f = x[e], g = y[e];
              x[e] = f * cs[e] - g * sn[e];
              y[e] = g * cs[e] + f * sn[e];
            }
          } else if (p.interleaved) {
            if constexpr (VEC >= 2) {
#pragma unroll
              for (int e = 0; e < VEC / 2; ++e) {
                const float f = x[2 * e], g = x[2 * e + 1], u = y[2 * e], w = y[2 * e + 1];
                if (rot0 + 2 * e < p.rotary) {
                  x[2 * e] = f * cs[e] - g * sn[e];
                  x[2 * e + 1] = g * cs[e] + f * sn[e];
                }
                if (rot1 + 2 * e < p.rotary) {
                  y[2 * e] = u * cs[VEC / 2 + e] - w * sn[VEC / 2 + e];
                  y[2 * e + 1] = w * cs[VEC / 2 + e] + u * sn[VEC / 2 + e];
                }
              }
            }
          }
        }
        if (F8 && cached) {
          const float *scales = copied ? c.value_scale : c.key_scale;
          const float scale = scales ? scales[head] : 1.f, by = 1.f / scale;
          if (d0 < c.dim) store_e4m3<VEC, ALIGNED>(dst + d0, x, scale, by);
          if (d1 < c.dim) store_e4m3<VEC, ALIGNED>(dst + d1, y, scale, by);
          continue;
        }
        ca = pack<BF16, VEC>(x);
        cb = pack<BF16, VEC>(y);
      }
      if (d0 < c.dim) store<VEC, ALIGNED>(reinterpret_cast<uint16_t *>(dst) + d0, ca);
      if (d1 < c.dim) store<VEC, ALIGNED>(reinterpret_cast<uint16_t *>(dst) + d1, cb);
    }
  }
}

template <bool BF16, bool F8>
void launch(const AppendParams &p, int vec, unsigned blocks, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(unsigned(vec == 1 ? kAppendThreads<1> : kAppendThreads<8>));
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  GCB_CUDA(cudaLaunchKernelEx(&cfg, vec == 8   ? append_kernel<BF16, F8, 8, true>
                                    : vec == 4 ? append_kernel<BF16, F8, 4, true>
                                    : vec == 2 ? append_kernel<BF16, F8, 2, false>
                                               : append_kernel<BF16, F8, 1, false>, p));
  count_launch();
}

void require(bool ok, const char *what) {
  if (!ok) throw std::invalid_argument(what);
}

} // namespace

PagedCache checked_cache(const gcb200_paged_cache &c, bool writes) {
  require(c.dtype == GCB200_BF16 || c.dtype == GCB200_F16, "paged cache: dtype must be bf16 or f16");
  require(c.cache_dtype == c.dtype || c.cache_dtype == GCB200_F8_E4M3, "paged cache: the cache must have the operands' type, or e4m3");
  require(c.keys && c.values && (c.page_table || c.sequences == 0 || c.max_pages == 0), "paged cache: null pointer");
  require(c.pages > 0 && c.page_size > 0 && c.kv_heads > 0 && c.sequences >= 0 && c.max_pages >= 0, "paged cache: sizes must be positive");
  require(c.pages < (int64_t(1) << 31) && c.sequences < (int64_t(1) << 31) && c.kv_heads < 65536 && c.page_size <= (int64_t(1) << 30) &&
              c.max_pages < (int64_t(1) << 31) && c.page_size * c.max_pages <= (int64_t(1) << 31) - 65536,
          "paged cache: positions and page numbers are 32-bit");
  const int size = c.cache_dtype == GCB200_F8_E4M3 ? 1 : 2;
  require(c.head_dim >= 8 && c.head_dim <= kMaxDim && c.head_dim * size % 16 == 0,
          "paged cache: head_dim must be at most 256 and a multiple of 8 (of 16 for an 8-bit cache)");
  require(size == 1 || (!c.key_scale && !c.value_scale), "paged cache: scales are for 8-bit caches");
  require(c.sequences <= 1 || c.page_table_stride >= c.max_pages, "paged cache: rows of the page table overlap");
  const int64_t extent[3] = {c.pages, c.kv_heads, c.page_size};
  int64_t ks[3], vs[3];
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of one is never used, whatever it says
    ks[i] = extent[i] > 1 ? c.key_stride[i] * size : 0;
    vs[i] = extent[i] > 1 ? c.value_stride[i] * size : 0;
    require(ks[i] >= 0 && vs[i] >= 0 && ks[i] % 16 == 0 && vs[i] % 16 == 0, "paged cache: strides must be multiples of 16 bytes");
    if (writes && extent[i] > 1) require(ks[i] >= c.head_dim * size && vs[i] >= c.head_dim * size, "paged cache: rows of the cache overlap");
  }
  require(((reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values)) & 15) == 0, "paged cache: keys and values must be 16-byte aligned");
  require(aligned(c.page_table, 4) && aligned(c.key_scale, 4) && aligned(c.value_scale, 4), "paged cache: misaligned page table or scales");
  PagedCache d{};
  d.keys = static_cast<uint8_t *>(c.keys);
  d.values = static_cast<uint8_t *>(c.values);
  d.key_page = ks[0]; d.key_head = ks[1]; d.key_token = ks[2];
  d.value_page = vs[0]; d.value_head = vs[1]; d.value_token = vs[2];
  d.key_scale = c.key_scale;
  d.value_scale = c.value_scale;
  d.table = PageTable{c.page_table, c.page_table_stride, int(c.sequences), int(c.max_pages), int(c.page_size), int(c.pages)};
  d.kv_heads = int(c.kv_heads);
  d.dim = int(c.head_dim);
  return d;
}

void paged_kv_append(const gcb200_paged_cache &cache, const AppendArgs &a, cudaStream_t stream) {
  AppendParams p{};
  p.c = checked_cache(cache, true);
  require(a.tokens == 0 || (a.k && a.v && a.positions), "paged append: null pointer");
  require(!a.q || a.q_out, "paged append: queries without a place to go");
  require(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "paged append: number of tokens out of range");
  require(!a.q || (a.heads > 0 && a.heads < 65536), "paged append: number of heads out of range");
  require(!a.q || !rows_overlap(a.tokens, a.q_out_stride[0], a.heads, a.q_out_stride[1], cache.head_dim), "paged append: rows of the rotated queries overlap");
  require(a.sequences || a.tokens <= cache.sequences, "paged append: more tokens than sequences, and no sequence numbers");
  require(a.inv_freq ? a.rotary_dim >= 2 && a.rotary_dim % 2 == 0 && a.rotary_dim <= cache.head_dim : a.rotary_dim == 0,
          "paged append: rotary_dim must be even and at most head_dim (0 without inv_freq)");
  require(aligned(a.q, 2) && aligned(a.k, 2) && aligned(a.v, 2) && aligned(a.q_out, 2) && aligned(a.sequences, 4) && aligned(a.positions, 4) && aligned(a.inv_freq, 8),
          "paged append: misaligned pointer");
  if (a.tokens == 0) return;
  DeviceState &dev = device_state();
  p.c.error = dev.d_page_error;
  p.q = static_cast<const uint16_t *>(a.q);
  p.k = static_cast<const uint16_t *>(a.k);
  p.v = static_cast<const uint16_t *>(a.v);
  p.q_out = static_cast<uint16_t *>(a.q_out);
  auto of = [](const int64_t s[2], int64_t tokens, int64_t heads, int64_t &token, int64_t &head) {
    token = tokens > 1 ? s[0] : 0;
    head = heads > 1 ? s[1] : 0;
  };
  if (a.q) {
    of(a.q_stride, a.tokens, a.heads, p.q_token, p.q_head);
    of(a.q_out_stride, a.tokens, a.heads, p.o_token, p.o_head);
  }
  of(a.k_stride, a.tokens, cache.kv_heads, p.k_token, p.k_head);
  of(a.v_stride, a.tokens, cache.kv_heads, p.v_token, p.v_head);
  p.sequences = a.sequences;
  p.positions = a.positions;
  p.inv_freq = a.inv_freq;
  p.heads = int(a.heads);
  p.rotary = int(a.rotary_dim);
  p.interleaved = a.interleaved;
  // the widest chunk that every address and both halves of a rotation are multiples of
  const int64_t rest = cache.head_dim - a.rotary_dim, half = a.rotary_dim / 2;
  int64_t all = int64_t(reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) | 2 * (p.k_token | p.k_head | p.v_token | p.v_head);
  if (a.q) all |= int64_t(reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out)) | 2 * (p.q_token | p.q_head | p.o_token | p.o_head);
  const int64_t pieces = a.interleaved ? 0 : (half | rest);
  const int vec = all % 16 == 0 && pieces % 8 == 0 ? 8 : all % 8 == 0 && pieces % 4 == 0 ? 4 : pieces % 2 == 0 ? 2 : 1;
  const int64_t chunks = cache.head_dim / vec;
  const int64_t rotated_units = a.interleaved || !a.rotary_dim ? 0 : half / vec + (rest / vec + 1) / 2;
  p.units = int(std::max((chunks + 1) / 2, rotated_units));
  const bool bf16 = cache.dtype == GCB200_BF16, f8 = cache.cache_dtype == GCB200_F8_E4M3;
  (bf16 ? (f8 ? launch<true, true> : launch<true, false>) : (f8 ? launch<false, true> : launch<false, false>))(p, vec, unsigned(a.tokens), stream);
}

} // namespace gcb
