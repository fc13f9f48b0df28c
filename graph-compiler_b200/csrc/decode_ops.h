// Operators of a decode step: the paged key-value cache (paged_append.cu, paged_attention.cu) and linear layers with 4-bit
// weights (matmul_w4.cu).  Arguments as in include/gc_b200.h; the launchers check them and throw.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/gc_b200.h"
#include "gemm_sm100.cuh"
#include "paged_index.h"

namespace gcb {

// Whether an address (or none) is a multiple of `bytes`: the kernels would stop at any other with a fault.
inline bool aligned(const void *p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// What the kernels of the cache see.  Strides in bytes.
struct PagedCache {
  uint8_t *keys, *values;
  int64_t key_page, key_head, key_token, value_page, value_head, value_token;
  const float *key_scale, *value_scale;
  PageTable table;
  int kv_heads, dim;
  int *error;
};
#ifdef __CUDACC__
// The word lies in host memory and never holds another code than this: a plain store by one of the threads that are here.  (An
// atomic exchange by each waits for the host every time: 2 x 16384 tokens of 8 KV heads on bad pages took 218 ms, now 41 us.)
__device__ __forceinline__ void report_bad_page(int *word) {
  if (int(threadIdx.x & 31) == __ffs(int(__activemask())) - 1) *static_cast<volatile int *>(word) = ERR_BAD_PAGE;
}
#endif
// Checks a descriptor; `writes`: the call stores into the cache.
PagedCache checked_cache(const gcb200_paged_cache &c, bool writes);

struct AppendArgs {
  const void *q, *k, *v;
  void *q_out;
  int64_t q_stride[2], k_stride[2], v_stride[2], q_out_stride[2], heads, tokens, rotary_dim;
  const int32_t *sequences, *positions;
  const double *inv_freq;
  int interleaved;
};
void paged_kv_append(const gcb200_paged_cache &cache, const AppendArgs &a, cudaStream_t stream);

struct PagedAttentionArgs {
  const void *q;
  void *out;
  int64_t q_stride[2], out_stride[2], heads, window;
  const int32_t *lengths;
  float scale;
  float *lse;
  void *workspace;
  size_t workspace_bytes;
};
size_t paged_attention_workspace(int64_t heads, int64_t kv_heads, int64_t head_dim);
void paged_attention(const gcb200_paged_cache &cache, const PagedAttentionArgs &a, cudaStream_t stream);

size_t w4_packed_bytes(int64_t N, int64_t K, int64_t group, int has_zeros);
void w4_pack(const uint8_t *codes, int64_t codes_stride, const void *scales, int64_t scales_stride, const uint8_t *zeros,
             int64_t zeros_stride, int64_t N, int64_t K, int64_t group, void *packed, cudaStream_t stream);
void matmul_w4(int dtype, const void *X, int64_t ldx, const void *packed, const void *bias, void *Y, int64_t ldy, int64_t M,
               int64_t N, int64_t K, int64_t group, int has_zeros, int relu, cudaStream_t stream);

} // namespace gcb
