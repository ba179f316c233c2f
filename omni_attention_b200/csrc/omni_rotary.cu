// Rotary positions with optional RMS norms of the heads, forward and backward, and the same work done on the way into a
// paged key/value cache.
//
// Mathematics, for one head row x of D elements at position t:
//   norm (optional)  r = (mean(x^2) + eps)^(-1/2),  y = x * r * w
//   rotation         pair p < rotary_dim / 2 at the angle a = t * inv_freq[p]:
//                    (y1, y2) -> factor * (y1 cos a - y2 sin a, y1 sin a + y2 cos a)
//                    members of a pair: 2p and 2p + 1 (interleaved) or p and p + rotary_dim / 2 (half)
//   backward         g' = the rotation by -a of the gradient, dw = sum over rows g' * x * r,
//                    dx = r * (g' w - x r * mean(g' w * x r))
// The angle is a product and a reduction to one turn in 64 bits (t * inv_freq is exact to 2^-53 of itself; in 32 bits a
// position of 100 000 would be off by 1e-2), its cosine and sine, the norm and everything else are in 32 bits, and each
// result is rounded once.
//
// Bound: memory - each element is read once and written once, about ten operations between. A thread owns 8 pairs (16
// elements) of a token and keeps their cosines and sines in registers while it walks over the heads, so that these are
// computed once per token and group of heads, not once per row; D / 16 threads are a row, and the norm's sums go through
// that many lanes' shuffles.
#include "omni_common.cuh"
#include "omni_launch.h"
#include "omni_rotary.cuh"

namespace omni {

namespace {

constexpr int kRotThreads = 256;

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <>
struct Elem<float> {
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What a thread holds of one row as it lies in memory: 16 elements in two chunks of 8 (VEC), 16-byte loads.
template <typename T>
struct Raw {
  uint4 c[sizeof(T) == 4 ? 4 : 2];
};

// Which elements of a row a thread owns. Pair j (of 8) has the members first(j) and second(j). VEC: they lie in two runs
// of 8 that start at o0 and o1; interleaved, a run holds four whole pairs; half, the runs hold the first and the second
// members (beyond the rotated part the two runs are neighbours and a "pair" is only two elements that pass through).
template <int D, bool HALF>
struct Place {
  int lane, o0, o1, rd2;   // lane of the row, run starts, rotary_dim / 2
  __device__ __forceinline__ Place(int lane_, int rd) : lane(lane_), rd2(rd >> 1) {
    const bool rotated = 8 * lane < rd2;
    o0 = HALF && rotated ? 8 * lane : 16 * lane;
    o1 = HALF && rotated ? rd2 + 8 * lane : 16 * lane + 8;
  }
  __device__ __forceinline__ int pair(int j) const { return 8 * lane + j; }
  // element numbers for the path that loads one element at a time; the same as above where both paths could be taken, so
  // that sums over a thread's elements have one order
  __device__ __forceinline__ int first(int j) const {
    const int p = pair(j);
    return !HALF ? 2 * p : p < rd2 ? p : 8 * lane >= rd2 ? 16 * lane + j : 2 * p;
  }
  __device__ __forceinline__ int second(int j) const {
    const int p = pair(j);
    return !HALF ? 2 * p + 1 : p < rd2 ? p + rd2 : 8 * lane >= rd2 ? 16 * lane + 8 + j : 2 * p + 1;
  }
};

template <typename T, bool VEC, typename P>
__device__ __forceinline__ void load_raw(const T* row, const P& at, Raw<T>& raw) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      raw.c[0] = __ldg(reinterpret_cast<const uint4*>(row + at.o0));
      raw.c[1] = __ldg(reinterpret_cast<const uint4*>(row + at.o0) + 1);
      raw.c[2] = __ldg(reinterpret_cast<const uint4*>(row + at.o1));
      raw.c[3] = __ldg(reinterpret_cast<const uint4*>(row + at.o1) + 1);
    } else {
      raw.c[0] = __ldg(reinterpret_cast<const uint4*>(row + at.o0));
      raw.c[1] = __ldg(reinterpret_cast<const uint4*>(row + at.o1));
    }
  } else {
    T* e = reinterpret_cast<T*>(raw.c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = row[at.first(j)];
      e[8 + j] = row[at.second(j)];
    }
  }
}

// a[j], b[j]: the members of pair j.
template <typename T, bool HALF, bool VEC>
__device__ __forceinline__ void to_pairs(const Raw<T>& raw, float (&a)[8], float (&b)[8]) {
  float u[8], v[8];
  if constexpr (sizeof(T) == 4) {
    const float* e = reinterpret_cast<const float*>(raw.c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = e[j];
      v[j] = e[8 + j];
    }
  } else {
    unpack8(raw.c[0], u, T());
    unpack8(raw.c[1], v, T());
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (HALF || !VEC) {
      a[j] = u[j];
      b[j] = v[j];
    } else {
      a[j] = j < 4 ? u[2 * (j & 3)] : v[2 * (j & 3)];
      b[j] = j < 4 ? u[2 * (j & 3) + 1] : v[2 * (j & 3) + 1];
    }
  }
}

template <typename T, bool HALF, bool VEC, typename P>
__device__ __forceinline__ void store_pairs(T* row, const P& at, const float (&a)[8], const float (&b)[8]) {
  if constexpr (VEC) {
    float u[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (HALF) {
        u[j] = a[j];
        v[j] = b[j];
      } else {
        u[j] = (j & 1) ? b[j >> 1] : a[j >> 1];
        v[j] = (j & 1) ? b[4 + (j >> 1)] : a[4 + (j >> 1)];
      }
    }
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(row + at.o0)[0] = make_float4(u[0], u[1], u[2], u[3]);
      reinterpret_cast<float4*>(row + at.o0)[1] = make_float4(u[4], u[5], u[6], u[7]);
      reinterpret_cast<float4*>(row + at.o1)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(row + at.o1)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 x, y;
      x.x = pack2(u[0], u[1], T());
      x.y = pack2(u[2], u[3], T());
      x.z = pack2(u[4], u[5], T());
      x.w = pack2(u[6], u[7], T());
      y.x = pack2(v[0], v[1], T());
      y.y = pack2(v[2], v[3], T());
      y.z = pack2(v[4], v[5], T());
      y.w = pack2(v[6], v[7], T());
      *reinterpret_cast<uint4*>(row + at.o0) = x;
      *reinterpret_cast<uint4*>(row + at.o1) = y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      Elem<T>::store(row + at.first(j), a[j]);
      Elem<T>::store(row + at.second(j), b[j]);
    }
  }
}

// The weight of the thread's elements, from a row of D weights in 32 bits or in the data's type.
template <typename T, int D, bool HALF, bool VEC>
__device__ __forceinline__ void load_weight(const void* w, bool f32, long long row, const Place<D, HALF>& at,
                                            float (&a)[8], float (&b)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int e0, e1;
    if constexpr (VEC && !HALF) {
      e0 = 2 * at.pair(j);
      e1 = e0 + 1;
    } else if constexpr (VEC) {
      e0 = at.o0 + j;
      e1 = at.o1 + j;
    } else {
      e0 = at.first(j);
      e1 = at.second(j);
    }
    if (f32) {
      a[j] = __ldg(static_cast<const float*>(w) + row * D + e0);
      b[j] = __ldg(static_cast<const float*>(w) + row * D + e1);
    } else {
      a[j] = Elem<T>::load(static_cast<const T*>(w) + row * D + e0);
      b[j] = Elem<T>::load(static_cast<const T*>(w) + row * D + e1);
    }
  }
}

// Cosines and sines of the thread's pairs at position `pos`, with the factor; 1 and 0 for what is not rotated.
template <int D, bool HALF>
__device__ __forceinline__ void turn_of(const RotaryParams& p, const Place<D, HALF>& at, long long pos, float (&c)[8],
                                        float (&s)[8]) {
  const double t = static_cast<double>(pos) * 0.15915494309189533577;   // 1 / (2 pi)
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (at.pair(j) < at.rd2) {
      double turns = t * __ldg(p.inv_freq + at.pair(j));
      turns -= rint(turns);
      float sn, cs;
      sincospif(2.f * static_cast<float>(turns), &sn, &cs);
      c[j] = cs * p.factor;
      s[j] = sn * p.factor * p.sign;
    } else {
      c[j] = 1.f;
      s[j] = 0.f;
    }
  }
}

__device__ __forceinline__ long long position_of(const RotaryParams& p, int b, int n) {
  if (p.positions == nullptr) return (p.lengths != nullptr ? max(__ldg(p.lengths + b), 0) : 0) + static_cast<long long>(n);
  const long long i = b * p.pos_stride_b + n * p.pos_stride_n;
  return p.pos64 ? __ldg(static_cast<const long long*>(p.positions) + i) : __ldg(static_cast<const int*>(p.positions) + i);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Forward, and with sign = -1 the backward of a rotation without a norm. grid.x: tiles of tokens (all batch elements in
// one row of tokens), grid.y: groups of heads. PAGED: k and v go into the pages of a cache, rows beyond a sequence's
// count are not stored there and are zero in q's result.
template <typename T, int D, bool HALF, bool VEC, bool PAGED>
__global__ void __launch_bounds__(kRotThreads) omni_rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int LPR = D / 16;                       // lanes of a row
  constexpr int ROWS = kRotThreads / LPR;
  const Place<D, HALF> at(threadIdx.x % LPR, p.rotary_dim);
  const long long token = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / LPR;
  const bool inside = token < p.tokens;
  const int b = inside ? static_cast<int>(token / p.N) : 0;
  const int n = inside ? static_cast<int>(token % p.N) : 0;

  float c[8], s[8];
  turn_of<D, HALF>(p, at, position_of(p, b, n), c, s);

  bool live = inside;
  long long slot = -1;                              // row of the token's slot in head 0 of its page
  if constexpr (PAGED) {
    if (p.counts != nullptr && n >= __ldg(p.counts + b)) live = false;
    if (live) {
      const long long key = static_cast<long long>(max(__ldg(p.lengths + b), 0)) + n;
      const long long entry = key >> p.page_shift;
      const int page = entry < p.max_pages ? __ldg(p.page_table + b * p.table_stride + entry) : -1;
      if (page >= 0 && page < p.num_pages) {
        slot = ((static_cast<long long>(page) * p.seg[1].heads) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
      } else if (p.status != nullptr && at.lane == 0) {
        atomicCAS(p.status, 0, kStatusBadIndex);
      }
    }
  }

  const int h_end = min(p.heads_total, (static_cast<int>(blockIdx.y) + 1) * p.heads_per_group);
  const int hq = p.seg[0].heads, hk = p.seg[1].heads;
  auto segment = [&](int h) { return h < hq ? 0 : h < hq + hk ? 1 : 2; };
  auto local = [&](int h, int g) { return h - (g == 0 ? 0 : g == 1 ? hq : hq + hk); };
  auto source = [&](int h) {
    const int g = segment(h);
    const RotarySegment& sg = p.seg[g];
    return static_cast<const T*>(sg.x) + b * sg.xs_b + local(h, g) * sg.xs_h + n * sg.xs_n;
  };

  Raw<T> next;
  int h = blockIdx.y * p.heads_per_group;
  if (h < h_end) load_raw<T, VEC>(source(h), at, next);
  float wa[8], wb[8];
  int weight_of = -1;
  for (; h < h_end; ++h) {
    const Raw<T> raw = next;
    if (h + 1 < h_end) load_raw<T, VEC>(source(h + 1), at, next);
    const int g = segment(h);
    const RotarySegment& sg = p.seg[g];
    const int hl = local(h, g);
    float a[8], bb[8];
    to_pairs<T, HALF, VEC>(raw, a, bb);
    if (sg.w != nullptr) {
      if (weight_of != g || p.w_per_head) {
        load_weight<T, D, HALF, VEC>(sg.w, p.w_f32, p.w_per_head ? hl : 0, at, wa, wb);
        weight_of = g;
      }
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq += a[j] * a[j] + bb[j] * bb[j];
      const float r = rsqrtf(row_sum<LPR>(sq) * (1.f / D) + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] *= r * wa[j];
        bb[j] *= r * wb[j];
      }
    }
    if (g < 2) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = a[j], v = bb[j];
        a[j] = u * c[j] - v * s[j];
        bb[j] = u * s[j] + v * c[j];
      }
    }
    if (PAGED && g > 0) {
      if (slot >= 0) {
        T* y = static_cast<T*>(sg.y) + (slot + (static_cast<long long>(hl) << p.page_shift)) * D;
        store_pairs<T, HALF, VEC>(y, at, a, bb);
      }
    } else if (inside) {
      if (PAGED && !live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = bb[j] = 0.f;
      }
      T* y = static_cast<T*>(sg.y) + ((static_cast<long long>(b) * sg.heads + hl) * p.N + n) * D;
      store_pairs<T, HALF, VEC>(y, at, a, bb);
    }
  }
}

// Backward with a norm: dx of every row and, per CTA, the sum over its rows of the weight's gradient (added up by
// omni_rotary_dw_kernel in a fixed order, so the result does not depend on which CTA ran first). grid.x: CTAs that share
// the tiles of tokens, grid.y: groups of heads, none of which holds heads of both q and k.
template <typename T, int D, bool HALF, bool VEC>
__global__ void __launch_bounds__(kRotThreads) omni_rotary_bwd_kernel(const __grid_constant__ RotaryBwdParams bp) {
  constexpr int LPR = D / 16;
  constexpr int ROWS = kRotThreads / LPR;
  const RotaryParams& p = bp.f;
  const Place<D, HALF> at(threadIdx.x % LPR, p.rotary_dim);
  const int group = blockIdx.y;
  const int g = group < bp.groups_q ? 0 : 1;
  const RotarySegment& sg = p.seg[g];
  const int per = g == 0 ? bp.per_q : bp.per_k;
  const int h0 = (g == 0 ? group : group - bp.groups_q) * per, h1 = min(sg.heads, h0 + per);

  float da[8], db[8], wa[8], wb[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) da[j] = db[j] = 0.f;
  load_weight<T, D, HALF, VEC>(sg.w, p.w_f32, p.w_per_head ? h0 : 0, at, wa, wb);

  const long long tiles = (p.tokens + ROWS - 1) / ROWS;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long token = tile * ROWS + threadIdx.x / LPR;
    const bool inside = token < p.tokens;
    const int b = inside ? static_cast<int>(token / p.N) : 0;
    const int n = inside ? static_cast<int>(token % p.N) : 0;
    float c[8], s[8];
    turn_of<D, HALF>(p, at, position_of(p, b, n), c, s);   // sign = -1: the rotation back
    const T* xrow = static_cast<const T*>(sg.x) + b * sg.xs_b + n * sg.xs_n;
    const T* grow = static_cast<const T*>(bp.g[g].x) + b * bp.g[g].xs_b + n * bp.g[g].xs_n;
    Raw<T> nx, ng;
    load_raw<T, VEC>(xrow + h0 * sg.xs_h, at, nx);
    load_raw<T, VEC>(grow + h0 * bp.g[g].xs_h, at, ng);
    for (int h = h0; h < h1; ++h) {
      float a[8], bb[8], ga[8], gb[8];
      to_pairs<T, HALF, VEC>(nx, a, bb);
      to_pairs<T, HALF, VEC>(ng, ga, gb);
      if (h + 1 < h1) {
        load_raw<T, VEC>(xrow + (h + 1) * sg.xs_h, at, nx);
        load_raw<T, VEC>(grow + (h + 1) * bp.g[g].xs_h, at, ng);
      }
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq += a[j] * a[j] + bb[j] * bb[j];
      const float r = rsqrtf(row_sum<LPR>(sq) * (1.f / D) + p.eps);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = ga[j] * c[j] - gb[j] * s[j], v = ga[j] * s[j] + gb[j] * c[j];
        a[j] *= r;
        bb[j] *= r;
        if (inside) {
          da[j] += u * a[j];
          db[j] += v * bb[j];
        }
        ga[j] = u * wa[j];
        gb[j] = v * wb[j];
        dot += ga[j] * a[j] + gb[j] * bb[j];
      }
      dot = row_sum<LPR>(dot) * (1.f / D);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ga[j] = r * (ga[j] - a[j] * dot);
        gb[j] = r * (gb[j] - bb[j] * dot);
      }
      if (inside) {
        T* y = static_cast<T*>(sg.y) + ((static_cast<long long>(b) * sg.heads + h) * p.N + n) * D;
        store_pairs<T, HALF, VEC>(y, at, ga, gb);
      }
    }
  }

  // rows of a warp, then the warps, each in a fixed order
  __shared__ float red[kRotThreads / 32][D];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 16; o >= LPR; o >>= 1) {
      da[j] += __shfl_xor_sync(0xFFFFFFFFu, da[j], o);
      db[j] += __shfl_xor_sync(0xFFFFFFFFu, db[j], o);
    }
  }
  if ((threadIdx.x & 31) < LPR) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int e0, e1;
      if constexpr (VEC && HALF) {
        e0 = at.o0 + j;
        e1 = at.o1 + j;
      } else {
        e0 = at.first(j);
        e1 = at.second(j);
      }
      red[threadIdx.x >> 5][e0] = da[j];
      red[threadIdx.x >> 5][e1] = db[j];
    }
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRotThreads / 32; ++w) sum += red[w][threadIdx.x];
    bp.partial[(static_cast<long long>(group) * gridDim.x + blockIdx.x) * D + threadIdx.x] = sum;
  }
}

// Sums the CTAs' shares of the weights' gradients. One CTA per weight row: `rows_q` of q's, then those of k's.
template <int D>
__global__ void __launch_bounds__(256) omni_rotary_dw_kernel(const __grid_constant__ RotaryBwdParams bp, int rows_q, int ctas) {
  constexpr int LANES = 256 / D;
  __shared__ float red[LANES][D];
  const int row = blockIdx.x;
  const int g = row < rows_q ? 0 : 1;
  const int local = g == 0 ? row : row - rows_q;
  const bool per_head = bp.f.w_per_head;
  const int first_group = (g == 0 ? 0 : bp.groups_q) + (per_head ? local : 0);
  const int groups = per_head ? 1 : (g == 0 ? bp.groups_q : bp.groups_k);
  const float* at = bp.partial + static_cast<long long>(first_group) * ctas * D;
  const int col = threadIdx.x % D, lane = threadIdx.x / D;
  const long long count = static_cast<long long>(groups) * ctas;
  float sum = 0.f;
#pragma unroll 8
  for (long long i = lane; i < count; i += LANES) sum += at[i * D + col];
  red[lane][col] = sum;
  __syncthreads();
  if (threadIdx.x < D) {
    float total = 0.f;
#pragma unroll
    for (int l = 0; l < LANES; ++l) total += red[l][threadIdx.x];
    void* dw = bp.dw[g];
    const long long e = static_cast<long long>(local) * D + threadIdx.x;
    if (bp.f.w_f32) {
      static_cast<float*>(dw)[e] = total;
    } else if (bp.f.bf16) {
      static_cast<__nv_bfloat16*>(dw)[e] = __float2bfloat16_rn(total);
    } else {
      static_cast<__half*>(dw)[e] = __float2half_rn(total);
    }
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return sms;
}

template <typename T, int D, bool HALF, bool VEC>
cudaError_t launch_t(RotaryParams p, bool paged, cudaStream_t stream) {
  constexpr int ROWS = kRotThreads / (D / 16);
  const long long tiles = (p.tokens + ROWS - 1) / ROWS;
  // As many groups of heads as it takes to have four CTAs on every SM, no more: each group computes the cosines and sines again.
  const long long want = (4LL * sm_count() + tiles - 1) / tiles;
  const int groups = static_cast<int>(want < 1 ? 1 : want > p.heads_total ? p.heads_total : want);
  p.heads_per_group = (p.heads_total + groups - 1) / groups;
  const dim3 grid(static_cast<unsigned>(tiles), (p.heads_total + p.heads_per_group - 1) / p.heads_per_group);
  if (paged) {
    omni_rotary_kernel<T, D, HALF, VEC, true><<<grid, kRotThreads, 0, stream>>>(p);
  } else {
    omni_rotary_kernel<T, D, HALF, VEC, false><<<grid, kRotThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

// How the token tiles and heads of a backward with norms are shared out; the workspace holds D floats for each CTA.
void bwd_grid(const RotaryParams& p, int D, RotaryBwdParams& bp, int& ctas) {
  const int rows = kRotThreads / (D / 16);
  const long long tiles = (p.tokens + rows - 1) / rows;
  const int hq = p.seg[0].heads, hk = p.seg[1].heads;
  bp.per_q = bp.per_k = 1;
  if (!p.w_per_head) {
    const long long want = (4LL * 148 + tiles - 1) / tiles;   // groups, as in the forward
    const int total = hq + hk;
    const int per = static_cast<int>((total + want - 1) / want);
    bp.per_q = per < hq ? per : (hq > 0 ? hq : 1);
    bp.per_k = per < hk ? per : (hk > 0 ? hk : 1);
  }
  bp.groups_q = (hq + bp.per_q - 1) / bp.per_q;
  bp.groups_k = (hk + bp.per_k - 1) / bp.per_k;
  const int groups = bp.groups_q + bp.groups_k;
  long long c = (8LL * 148 + groups - 1) / groups;   // CTAs of a group: eight per SM in all
  ctas = static_cast<int>(c < tiles ? c : tiles);
}

template <typename T, int D, bool HALF, bool VEC>
cudaError_t launch_bwd_t(RotaryBwdParams bp, cudaStream_t stream) {
  int ctas = 0;
  bwd_grid(bp.f, D, bp, ctas);
  const dim3 grid(ctas, bp.groups_q + bp.groups_k);
  omni_rotary_bwd_kernel<T, D, HALF, VEC><<<grid, kRotThreads, 0, stream>>>(bp);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int rows_q = bp.f.seg[0].heads == 0 ? 0 : bp.f.w_per_head ? bp.f.seg[0].heads : 1;
  const int rows_k = bp.f.seg[1].heads == 0 ? 0 : bp.f.w_per_head ? bp.f.seg[1].heads : 1;
  omni_rotary_dw_kernel<D><<<rows_q + rows_k, 256, 0, stream>>>(bp, rows_q, ctas);
  return cudaGetLastError();
}

// What the kernels are built for: (type, head_dim, layout, vector or element loads).
template <template <typename, int, bool, bool> class Fn, typename... A>
cudaError_t dispatch(int dtype, int head_dim, bool half, bool vec, A&&... args) {
#define OMNI_ROT_CASE(T, D)                                                                                    \
  return half ? (vec ? Fn<T, D, true, true>::run(args...) : Fn<T, D, true, false>::run(args...))               \
              : (vec ? Fn<T, D, false, true>::run(args...) : Fn<T, D, false, false>::run(args...))
#define OMNI_ROT_TYPE(T)                        \
  do {                                          \
    if (head_dim == 32) { OMNI_ROT_CASE(T, 32); }  \
    if (head_dim == 64) { OMNI_ROT_CASE(T, 64); }  \
    OMNI_ROT_CASE(T, 128);                      \
  } while (0)
  if (dtype == 0) OMNI_ROT_TYPE(__half);
  if (dtype == 1) OMNI_ROT_TYPE(__nv_bfloat16);
  OMNI_ROT_TYPE(float);
#undef OMNI_ROT_TYPE
#undef OMNI_ROT_CASE
}

template <typename T, int D, bool HALF, bool VEC>
struct Forward {
  static cudaError_t run(const RotaryParams& p, bool paged, cudaStream_t s) { return launch_t<T, D, HALF, VEC>(p, paged, s); }
};
template <typename T, int D, bool HALF, bool VEC>
struct Backward {
  static cudaError_t run(const RotaryBwdParams& p, cudaStream_t s) { return launch_bwd_t<T, D, HALF, VEC>(p, s); }
};

}  // namespace

cudaError_t launch_rotary(int dtype, int head_dim, bool half, bool vec, bool paged, const RotaryParams& p, cudaStream_t stream) {
  return dispatch<Forward>(dtype, head_dim, half, vec, p, paged, stream);
}
cudaError_t launch_rotary_bwd(int dtype, int head_dim, bool half, bool vec, const RotaryBwdParams& p, cudaStream_t stream) {
  return dispatch<Backward>(dtype, head_dim, half, vec, p, stream);
}
long long rotary_bwd_partials(const RotaryParams& p, int head_dim) {
  RotaryBwdParams bp;
  int ctas = 0;
  bwd_grid(p, head_dim, bp, ctas);
  return static_cast<long long>(bp.groups_q + bp.groups_k) * ctas * head_dim;
}

}  // namespace omni
