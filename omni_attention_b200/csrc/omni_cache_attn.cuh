// Launch parameters of the attention over a paged key/value cache (omni_cache_attn.cu).
#pragma once
#include <cuda.h>

#include <cstdint>
#include <cuda_runtime.h>

namespace omni {

struct CacheAttnParams {
  const void* q;                // [B, H, T, D], strides in elements, every row 16-byte aligned
  long long qs_b, qs_h, qs_t;
  void* out;                    // [B, H, T, D] contiguous
  float* lse;                   // [B, H, T] or null
  const void* k_pages;          // [num_pages, Hkv, page_size, D]
  const void* v_pages;
  const int32_t* page_table;    // [B, max_pages]
  long long table_stride;
  const int32_t* lengths;       // [B] tokens before this call's T
  const int32_t* counts;        // [B] or null (= T)
  const int32_t* limits;        // [B, T] keys a row sees, or null
  int32_t* status;
  float* partial;               // workspace, see omni_cache_attn.cu
  long long capacity;           // max_pages * page_size
  int B, H, Hkv, G, T;
  int max_pages, num_pages, page_shift;
  int prefix;                   // tokens that all sequences have in the same pages (multiple of the page size), or 0
  int causal;
  float scale;                  // softmax scale
  float softcap;                // 0 = none
  long long wait_cycles;        // cycle budget of one bounded wait
};

// One launch over some of the segments (omni_cache_line.cuh).
struct CacheLaunch {
  int rows;                     // of a row tile
  int ctas;
  int prefix, own;              // which segments
  int rt_prefix, rt_own;        // row tiles of the prefix (0 without it), of a sequence
  unsigned per_cta;             // triples / ctas, rounded up
  unsigned uncut;               // kUncutTiles or kUncutTilesPrefix
  unsigned even;                // CTAs for each triple, if there are that many (Line::even)
  int late_wait;                // 0: waits for its predecessor before it reads anything; 1: only before it ends
  long long share0;             // its shares in the workspace, in floats
};

cudaError_t launch_cache_attn(int head_dim, bool bf16, const CacheAttnParams& p, cudaStream_t stream);
long long cache_attn_workspace_bytes(int B, int H, int Hkv, int T, int head_dim, bool prefix, long long capacity);

// Tensor maps of k_pages and v_pages (omni_abi.cu): the pages as a matrix of rows, one box = 64 columns of
// min(page_size, 128) tokens of one page and head.
cudaError_t make_page_maps(const CacheAttnParams& p, int head_dim, bool bf16, CUtensorMap* tmK, CUtensorMap* tmV);

constexpr int kTileKeys = 128;     // of both kernels
constexpr int kNarrowRows = 16, kWideRows = 128;   // most rows of the narrow kernel's tile: 8 or 16
constexpr int kCacheCtas = 148;    // one CTA per SM
// What cutting costs, in tiles of keys: the shares' way through memory and the kernel that joins them (with a prefix they are
// joined in any case). 8 triples of 3 tiles: uncut 7.0 us, cut 7.3; of 5 tiles 8.7 and 7.9; of 16 tiles 16.5 and 11.4.
constexpr int kUncutTiles = 2, kUncutTilesPrefix = 0;
// What a second piece costs a CTA, in tiles: its queries, the first tile's way through the chain, the join of its shares.
// 40 triples of 64 tiles on 148 CTAs: in even spans 34.8 us, three CTAs for each triple 32.8.
constexpr int kPieceTiles = 4;
// Tiles of 128 rows on the tcgen05 tensor cores (omni_cache_wide.cu).
cudaError_t launch_cache_wide(int head_dim, bool bf16, const CUtensorMap& tmK, const CUtensorMap& tmV, const CacheAttnParams& p,
                              const CacheLaunch& how, cudaStream_t stream);
// Whether the call's line of units can be counted in 31 bits.
bool cache_attn_fits(const CacheAttnParams& p);

// A programmatic dependent launch: may start before its predecessor on the stream has ended (omni_cache_line.cuh: grid_wait).
template <typename... P, typename... A>
inline cudaError_t launch_chained(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace omni
