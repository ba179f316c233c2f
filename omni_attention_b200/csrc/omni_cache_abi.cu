// C-ABI layer of the rotary and paged-cache entry points: argument checks as error codes, before anything is launched,
// and the kernels' launch parameters.
#include <cmath>
#include <cstdint>

#include "../../include/omni_attn_sm100.h"
#include "omni_cache_attn.cuh"
#include "omni_launch.h"
#include "omni_rotary.cuh"

namespace omni {
namespace {

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// Every row of the tensor starts on a 16-byte boundary.
bool rows_aligned(const omni_attn_heads& t, int size) {
  return !misaligned(t.data) && (t.stride_b * size) % 16 == 0 && (t.stride_h * size) % 16 == 0 && (t.stride_n * size) % 16 == 0;
}

int check_rotary(const omni_attn_rotary* r, int head_dim) {
  if (r == nullptr) return OMNI_OK;
  if (r->rotary_dim < 0 || r->rotary_dim > head_dim || r->rotary_dim % 2 != 0 || (r->rotary_dim > 0 && r->inv_freq == nullptr)) {
    return OMNI_ERR_ROTARY;
  }
  return OMNI_OK;
}

int check_cache(const omni_attn_paged_cache* c) {
  if (c == nullptr || c->k_pages == nullptr || c->v_pages == nullptr || c->page_table == nullptr || c->lengths == nullptr) {
    return OMNI_ERR_NULL_POINTER;
  }
  if (c->num_pages <= 0 || c->max_pages <= 0 || c->heads <= 0 || c->page_size < 16 || c->page_size > 1024 ||
      (c->page_size & (c->page_size - 1)) != 0) {
    return OMNI_ERR_CACHE;
  }
  if (static_cast<long long>(c->max_pages) * c->page_size > 0x7FFF0000LL) return OMNI_ERR_TOO_LONG;   // token numbers are int32
  if (static_cast<long long>(c->num_pages) * c->heads * c->page_size >= (1LL << 31)) return OMNI_ERR_TOO_LONG;   // and so are rows of the pages
  if (misaligned(c->k_pages) || misaligned(c->v_pages)) return OMNI_ERR_ALIGNMENT;
  return OMNI_OK;
}

int check_sizes(int B, int N, int head_dim) {
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return OMNI_ERR_HEAD_DIM;
  if (B <= 0 || N <= 0 || static_cast<long long>(B) * N >= (1LL << 31)) return OMNI_ERR_SHAPE;
  return OMNI_OK;
}

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

int ended(cudaError_t e) {
  if (e == cudaSuccess) return OMNI_OK;
  set_last_cuda_error(static_cast<int>(e));
  return OMNI_ERR_CUDA;
}

void set_segment(RotarySegment& s, const omni_attn_heads* t, void* y, const void* w) {
  s = RotarySegment{};
  if (t == nullptr) return;
  s.x = t->data;
  s.y = y;
  s.xs_b = t->stride_b;
  s.xs_h = t->stride_h;
  s.xs_n = t->stride_n;
  s.w = w;
  s.heads = t->heads;
}

void set_rotary(RotaryParams& p, const omni_attn_rotary* r, int B, int N, int dtype) {
  p.factor = 1.f;
  p.sign = 1.f;
  p.N = N;
  p.tokens = static_cast<long long>(B) * N;
  p.bf16 = dtype == OMNI_DTYPE_BF16;
  if (r == nullptr) return;
  p.inv_freq = r->inv_freq;
  p.rotary_dim = r->rotary_dim;
  p.factor = r->factor;
  p.positions = r->positions;
  p.pos64 = r->positions_64;
  p.pos_stride_b = r->pos_stride_b;
  p.pos_stride_n = r->pos_stride_n;
  p.w_f32 = r->weight_f32 || dtype == OMNI_DTYPE_F32;
  p.w_per_head = r->weight_per_head;
  p.eps = r->eps;
}

bool vectors(const omni_attn_rotary* r, std::initializer_list<const omni_attn_heads*> in, std::initializer_list<const void*> out,
             int size) {
  if (r != nullptr && r->half_layout && r->rotary_dim % 16 != 0) return false;
  for (const omni_attn_heads* t : in) {
    if (t != nullptr && !rows_aligned(*t, size)) return false;
  }
  for (const void* o : out) {
    if (misaligned(o)) return false;
  }
  return r == nullptr || (!misaligned(r->q_weight) && !misaligned(r->k_weight));
}

// The kernels form scale / softcap to the sixth power, its inverse, and softcap * log2(e), all in 32 bits.
bool soft_cap_fits(float softcap, float scale) { return softcap <= 1e37f && softcap >= 1e-6 * scale && softcap <= 1e30 * scale; }

int heads_of(const omni_attn_heads* t) { return t == nullptr ? 0 : t->heads; }

}  // namespace
}  // namespace omni

extern "C" {

int omni_attn_rotary_sm100(const omni_attn_heads* q, const omni_attn_heads* k, void* q_out, void* k_out,
                           const omni_attn_rotary* rotary, int B, int N, int head_dim, int dtype, int inverse,
                           void* cuda_stream) {
  using namespace omni;
  if (rotary == nullptr || (q == nullptr && k == nullptr) || (q != nullptr && (q->data == nullptr || q_out == nullptr)) ||
      (k != nullptr && (k->data == nullptr || k_out == nullptr))) {
    return OMNI_ERR_NULL_POINTER;
  }
  if (dtype != OMNI_DTYPE_F16 && dtype != OMNI_DTYPE_BF16 && dtype != OMNI_DTYPE_F32) return OMNI_ERR_DTYPE;
  int rc = check_sizes(B, N, head_dim);
  if (rc != OMNI_OK) return rc;
  if ((rc = check_rotary(rotary, head_dim)) != OMNI_OK) return rc;
  if ((q != nullptr && q->heads <= 0) || (k != nullptr && k->heads <= 0) || heads_of(q) + heads_of(k) > 65535) return OMNI_ERR_SHAPE;
  if (inverse && (rotary->q_weight != nullptr || rotary->k_weight != nullptr)) return OMNI_ERR_ROTARY;
  RotaryParams p{};
  set_rotary(p, rotary, B, N, dtype);
  if (inverse) p.sign = -1.f;
  set_segment(p.seg[0], q, q_out, rotary->q_weight);
  set_segment(p.seg[1], k, k_out, rotary->k_weight);
  p.heads_total = heads_of(q) + heads_of(k);
  const bool vec = vectors(rotary, {q, k}, {q_out, k_out}, dtype == OMNI_DTYPE_F32 ? 4 : 2);
  if (!rotary_fits(p, head_dim)) return OMNI_ERR_SHAPE;
  return ended(launch_rotary(dtype, head_dim, rotary->half_layout != 0, vec, false, p, static_cast<cudaStream_t>(cuda_stream)));
}

long long omni_attn_rotary_bwd_workspace_bytes(int q_heads, int k_heads, int B, int N, int head_dim, int weight_per_head) {
  using namespace omni;
  if (q_heads < 0 || k_heads < 0 || q_heads + k_heads <= 0 || check_sizes(B, N, head_dim) != OMNI_OK) return 0;
  RotaryParams p{};
  p.tokens = static_cast<long long>(B) * N;
  p.seg[0].heads = q_heads;
  p.seg[1].heads = k_heads;
  p.w_per_head = weight_per_head;
  return rotary_bwd_partials(p, head_dim) * 4;
}

int omni_attn_rotary_bwd_sm100(const omni_attn_heads* q, const omni_attn_heads* k, const omni_attn_heads* d_q_out,
                               const omni_attn_heads* d_k_out, void* dq, void* dk, void* dq_weight, void* dk_weight,
                               const omni_attn_rotary* rotary, int B, int N, int head_dim, int dtype, void* workspace,
                               long long workspace_bytes, void* cuda_stream) {
  using namespace omni;
  if (rotary == nullptr || workspace == nullptr || (q == nullptr && k == nullptr)) return OMNI_ERR_NULL_POINTER;
  if (q != nullptr && (q->data == nullptr || d_q_out == nullptr || d_q_out->data == nullptr || dq == nullptr ||
                       dq_weight == nullptr || rotary->q_weight == nullptr)) {
    return OMNI_ERR_NULL_POINTER;
  }
  if (k != nullptr && (k->data == nullptr || d_k_out == nullptr || d_k_out->data == nullptr || dk == nullptr ||
                       dk_weight == nullptr || rotary->k_weight == nullptr)) {
    return OMNI_ERR_NULL_POINTER;
  }
  if (dtype != OMNI_DTYPE_F16 && dtype != OMNI_DTYPE_BF16 && dtype != OMNI_DTYPE_F32) return OMNI_ERR_DTYPE;
  int rc = check_sizes(B, N, head_dim);
  if (rc != OMNI_OK) return rc;
  if ((rc = check_rotary(rotary, head_dim)) != OMNI_OK) return rc;
  if ((q != nullptr && (q->heads <= 0 || d_q_out->heads != q->heads)) || (k != nullptr && (k->heads <= 0 || d_k_out->heads != k->heads)) ||
      heads_of(q) + heads_of(k) > 65535) {
    return OMNI_ERR_SHAPE;
  }
  if (misaligned(workspace)) return OMNI_ERR_ALIGNMENT;
  if (workspace_bytes < omni_attn_rotary_bwd_workspace_bytes(heads_of(q), heads_of(k), B, N, head_dim, rotary->weight_per_head)) {
    return OMNI_ERR_WORKSPACE;
  }
  RotaryBwdParams bp{};
  set_rotary(bp.f, rotary, B, N, dtype);
  bp.f.sign = -1.f;
  set_segment(bp.f.seg[0], q, dq, rotary->q_weight);
  set_segment(bp.f.seg[1], k, dk, rotary->k_weight);
  set_segment(bp.g[0], q != nullptr ? d_q_out : nullptr, nullptr, nullptr);
  set_segment(bp.g[1], k != nullptr ? d_k_out : nullptr, nullptr, nullptr);
  bp.dw[0] = dq_weight;
  bp.dw[1] = dk_weight;
  bp.partial = static_cast<float*>(workspace);
  const bool vec = vectors(rotary, {q, k, q != nullptr ? d_q_out : nullptr, k != nullptr ? d_k_out : nullptr}, {dq, dk},
                           dtype == OMNI_DTYPE_F32 ? 4 : 2);
  if (!rotary_fits(bp.f, head_dim)) return OMNI_ERR_SHAPE;
  return ended(launch_rotary_bwd(dtype, head_dim, rotary->half_layout != 0, vec, bp, static_cast<cudaStream_t>(cuda_stream)));
}

int omni_attn_cache_append_sm100(const omni_attn_heads* q, const omni_attn_heads* k, const omni_attn_heads* v,
                                 void* q_out, const omni_attn_paged_cache* cache, const int32_t* counts,
                                 const omni_attn_rotary* rotary, int B, int N, int head_dim, int dtype,
                                 void* cuda_stream, int32_t* status) {
  using namespace omni;
  if (k == nullptr || v == nullptr || k->data == nullptr || v->data == nullptr || (q != nullptr && (q->data == nullptr || q_out == nullptr))) {
    return OMNI_ERR_NULL_POINTER;
  }
  if (dtype != OMNI_DTYPE_F16 && dtype != OMNI_DTYPE_BF16) return OMNI_ERR_DTYPE;
  int rc = check_sizes(B, N, head_dim);
  if (rc != OMNI_OK) return rc;
  if ((rc = check_rotary(rotary, head_dim)) != OMNI_OK || (rc = check_cache(cache)) != OMNI_OK) return rc;
  if (k->heads != cache->heads || v->heads != cache->heads) return OMNI_ERR_CACHE;
  if ((q != nullptr && q->heads <= 0) || heads_of(q) + 2LL * cache->heads > 65535) return OMNI_ERR_SHAPE;
  RotaryParams p{};
  set_rotary(p, rotary, B, N, dtype);
  set_segment(p.seg[0], q, q_out, rotary != nullptr ? rotary->q_weight : nullptr);
  set_segment(p.seg[1], k, cache->k_pages, rotary != nullptr ? rotary->k_weight : nullptr);
  set_segment(p.seg[2], v, cache->v_pages, nullptr);
  p.heads_total = heads_of(q) + 2 * cache->heads;
  p.lengths = cache->lengths;
  p.counts = counts;
  p.page_table = cache->page_table;
  p.table_stride = cache->table_stride;
  p.max_pages = cache->max_pages;
  p.num_pages = cache->num_pages;
  p.page_shift = shift_of(cache->page_size);
  p.status = status;
  const bool vec = vectors(rotary, {q, k, v}, {q_out}, 2);
  if (!rotary_fits(p, head_dim)) return OMNI_ERR_SHAPE;
  const bool half = rotary != nullptr && rotary->half_layout != 0;
  return ended(launch_rotary(dtype, head_dim, half, vec, true, p, static_cast<cudaStream_t>(cuda_stream)));
}

long long omni_attn_cache_attention_workspace_bytes(int B, int H, int kv_heads, int T, int head_dim, int shared_prefix,
                                                    long long capacity) {
  if (B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads != 0 || T <= 0 || capacity <= 0) return 0;
  return omni::cache_attn_workspace_bytes(B, H, kv_heads, T, head_dim, shared_prefix > 0, capacity);
}

int omni_attn_cache_attention_sm100(const omni_attn_heads* q, void* out, float* lse, const omni_attn_paged_cache* cache,
                                    const int32_t* counts, const int32_t* limits, int causal, int B, int T, int head_dim,
                                    int dtype, float scale, float softcap, int shared_prefix, void* workspace,
                                    long long workspace_bytes, void* cuda_stream, int32_t* status) {
  using namespace omni;
  if (q == nullptr || q->data == nullptr || out == nullptr) return OMNI_ERR_NULL_POINTER;
  if (dtype != OMNI_DTYPE_F16 && dtype != OMNI_DTYPE_BF16) return OMNI_ERR_DTYPE;
  int rc = check_sizes(B, T, head_dim);
  if (rc != OMNI_OK) return rc;
  if ((rc = check_cache(cache)) != OMNI_OK) return rc;
  if (q->heads <= 0 || q->heads % cache->heads != 0) return OMNI_ERR_CACHE;
  if (static_cast<long long>(B) * q->heads * T >= (1LL << 31) - 64) return OMNI_ERR_SHAPE;
  const float scale_used = scale > 0.f ? scale : 1.f / std::sqrt(static_cast<float>(head_dim));
  if (!(softcap >= 0.f) || (softcap > 0.f && !soft_cap_fits(softcap, scale_used))) return OMNI_ERR_SOFTCAP;
  if (!rows_aligned(*q, 2) || misaligned(out) || misaligned(workspace)) return OMNI_ERR_ALIGNMENT;
  if (shared_prefix < 0) return OMNI_ERR_SEQLEN;
  CacheAttnParams p{};
  p.prefix = shared_prefix / cache->page_size * cache->page_size;
  p.capacity = static_cast<long long>(cache->max_pages) * cache->page_size;
  if (p.prefix > p.capacity) return OMNI_ERR_SEQLEN;
  const long long need = cache_attn_workspace_bytes(B, q->heads, cache->heads, T, head_dim, p.prefix > 0, p.capacity);
  if (need > 0 && workspace == nullptr) return OMNI_ERR_NULL_POINTER;
  if (workspace_bytes < need) return OMNI_ERR_WORKSPACE;
  p.q = q->data;
  p.qs_b = q->stride_b;
  p.qs_h = q->stride_h;
  p.qs_t = q->stride_n;
  p.out = out;
  p.lse = lse;
  p.k_pages = cache->k_pages;
  p.v_pages = cache->v_pages;
  p.page_table = cache->page_table;
  p.table_stride = cache->table_stride;
  p.lengths = cache->lengths;
  p.counts = counts;
  p.limits = limits;
  p.status = status;
  p.partial = static_cast<float*>(workspace);
  p.B = B;
  p.H = q->heads;
  p.Hkv = cache->heads;
  p.G = q->heads / cache->heads;
  p.T = T;
  p.max_pages = cache->max_pages;
  p.num_pages = cache->num_pages;
  p.page_shift = shift_of(cache->page_size);
  p.causal = causal;
  p.scale = scale_used;
  p.softcap = softcap;
  p.wait_cycles = wait_cycle_budget();
  if (!cache_attn_fits(p)) return OMNI_ERR_TOO_LONG;
  return ended(launch_cache_attn(head_dim, dtype == OMNI_DTYPE_BF16, p, static_cast<cudaStream_t>(cuda_stream)));
}

}  // extern "C"
