// Launch parameters of the rotary kernels (omni_rotary.cu) and of the append into a paged cache, which is the same kernel.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace omni {

// One of q, k, v: [B, heads, N, D] with the strides given (in elements; D is contiguous). y is contiguous
// [B, heads, N, D], or the pages [num_pages, heads, page_size, D] of a cache.
struct RotarySegment {
  const void* x;
  void* y;
  long long xs_b, xs_h, xs_n;
  const void* w;   // norm weight [D] or [heads, D], null = no norm
  int heads;
};

struct RotaryParams {
  RotarySegment seg[3];      // q, k, v (v: copied into the cache)
  const double* inv_freq;    // [rotary_dim / 2]
  const void* positions;     // int32 or int64, null = lengths[b] + n (lengths null: n)
  long long pos_stride_b, pos_stride_n;
  const int32_t* lengths;    // append: tokens of each sequence that are in the cache, else null
  const int32_t* counts;     // append: new tokens of each sequence, null = N
  const int32_t* page_table; // append: [B, max_pages]
  long long table_stride;
  int32_t* status;
  long long tokens;          // B * N
  int N;
  int rotary_dim;
  int max_pages, num_pages, page_shift;
  int heads_total;
  unsigned units, span;      // (tile of tokens, head) units, and how many a CTA takes
  float factor, sign, eps;
  int pos64, w_f32, w_per_head, bf16;
};

struct RotaryBwdParams {
  RotaryParams f;            // seg[0], seg[1]: x as in the forward, y = its gradient
  RotarySegment g[2];        // gradients of the results (x and strides)
  void* dw[2];
  float* partial;            // [CTA + sum, D]: the sums a CTA has shares in follow one another
  unsigned tiles;
  int sums;                  // weight rows
};

// dtype: 0 fp16, 1 bf16, 2 fp32. vec: every row starts on a 16-byte boundary, and in the half layout rotary_dim is a
// multiple of 16; else elements are loaded one by one.
cudaError_t launch_rotary(int dtype, int head_dim, bool half, bool vec, bool paged, const RotaryParams& p, cudaStream_t stream);
cudaError_t launch_rotary_bwd(int dtype, int head_dim, bool half, bool vec, const RotaryBwdParams& p, cudaStream_t stream);
// floats of RotaryBwdParams::partial
long long rotary_bwd_partials(const RotaryParams& p, int head_dim);

// Whether the call's units can be counted in 31 bits.
bool rotary_fits(const RotaryParams& p, int head_dim);

}  // namespace omni
