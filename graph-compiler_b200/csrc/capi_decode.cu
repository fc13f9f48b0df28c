// extern "C" launchers of the decode operators declared in include/gc_b200.h.
#include <exception>
#include <stdexcept>

#include "../../include/gc_b200.h"
#include "decode_ops.h"
#include "runtime.h"

#define GCB_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcb {
int guard_status(const std::exception_ptr &ep);   // capi_kernels.cu
}

using namespace gcb;

template <class F> static int guarded(F &&f) {
  try {
    f();
    return GCB200_OK;
  } catch (...) {
    return guard_status(std::current_exception());
  }
}
static void require(bool ok, const char *msg) {
  if (!ok) throw std::invalid_argument(msg);
}

GCB_EXPORT int gcb200_paged_kv_append(const gcb200_paged_cache *cache, const void *q, const int64_t q_stride[2], int64_t heads,
                                      const void *k, const int64_t k_stride[2], const void *v, const int64_t v_stride[2], void *q_out,
                                      const int64_t q_out_stride[2], const int32_t *sequences, const int32_t *positions, int64_t tokens,
                                      const double *inv_freq, int64_t rotary_dim, int interleaved, void *stream) {
  return guarded([&] {
    require(cache && k_stride && v_stride && (!q || (q_stride && q_out_stride)), "paged append: null pointer");
    AppendArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    for (int i = 0; i < 2; ++i) {
      a.q_stride[i] = q ? q_stride[i] : 0;
      a.q_out_stride[i] = q ? q_out_stride[i] : 0;
      a.k_stride[i] = k_stride[i];
      a.v_stride[i] = v_stride[i];
    }
    a.heads = heads;
    a.tokens = tokens;
    a.rotary_dim = rotary_dim;
    a.sequences = sequences;
    a.positions = positions;
    a.inv_freq = inv_freq;
    a.interleaved = interleaved != 0;
    paged_kv_append(*cache, a, static_cast<cudaStream_t>(stream));
  });
}

GCB_EXPORT int gcb200_paged_attention_workspace(int64_t heads, int64_t kv_heads, int64_t head_dim, size_t *bytes) {
  return guarded([&] {
    require(bytes != nullptr, "paged attention: null pointer");
    *bytes = paged_attention_workspace(heads, kv_heads, head_dim);
  });
}

GCB_EXPORT int gcb200_paged_attention(const gcb200_paged_cache *cache, const void *q, const int64_t q_stride[2], int64_t heads,
                                      const int32_t *lengths, float scale, int64_t window, void *out, const int64_t out_stride[2],
                                      float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  return guarded([&] {
    require(cache && q_stride && out_stride, "paged attention: null pointer");
    PagedAttentionArgs a{};
    a.q = q;
    a.out = out;
    for (int i = 0; i < 2; ++i) {
      a.q_stride[i] = q_stride[i];
      a.out_stride[i] = out_stride[i];
    }
    a.heads = heads;
    a.window = window;
    a.lengths = lengths;
    a.scale = scale;
    a.lse = lse;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    paged_attention(*cache, a, static_cast<cudaStream_t>(stream));
  });
}

GCB_EXPORT int gcb200_w4_packed_bytes(int64_t N, int64_t K, int64_t group, int has_zeros, size_t *bytes) {
  return guarded([&] {
    require(bytes != nullptr, "4-bit weights: null pointer");
    *bytes = w4_packed_bytes(N, K, group, has_zeros);
  });
}

GCB_EXPORT int gcb200_w4_pack(const uint8_t *codes, int64_t codes_stride, const void *scales, int64_t scales_stride, const uint8_t *zeros,
                              int64_t zeros_stride, int64_t N, int64_t K, int64_t group, void *packed, void *stream) {
  return guarded([&] {
    w4_pack(codes, codes_stride, scales, scales_stride, zeros, zeros_stride, N, K, group, packed, static_cast<cudaStream_t>(stream));
  });
}

GCB_EXPORT int gcb200_matmul_w4(int dtype, const void *X, int64_t ldx, const void *packed, const void *bias, void *Y, int64_t ldy, int64_t M,
                                int64_t N, int64_t K, int64_t group, int has_zeros, int relu, void *stream) {
  return guarded([&] {
    matmul_w4(dtype, X, ldx, packed, bias, Y, ldy, M, N, K, group, has_zeros, relu, static_cast<cudaStream_t>(stream));
  });
}
