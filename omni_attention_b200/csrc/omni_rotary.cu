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
#include "omni_cache_line.cuh"
#include "omni_launch.h"
#include "omni_rotary.cuh"

namespace omni {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotCtas = 3;        // CTAs of the forward on an SM: 85 registers a thread
constexpr int kSms = 148;

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

// The members of the thread's 8 pairs, two pairs to a packed 32-bit operation: a[i] = first members of pairs 2i and 2i + 1,
// b[i] = the second ones.
struct Pairs {
  float2 a[4], b[4];
};

template <typename T, bool HALF, bool VEC>
__device__ __forceinline__ void to_pairs(const Raw<T>& raw, Pairs& x) {
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
  for (int i = 0; i < 4; ++i) {
    if constexpr (HALF || !VEC) {
      x.a[i] = make_float2(u[2 * i], u[2 * i + 1]);
      x.b[i] = make_float2(v[2 * i], v[2 * i + 1]);
    } else {   // interleaved: four pairs in each run
      const float(&e)[8] = i < 2 ? u : v;
      x.a[i] = make_float2(e[4 * (i & 1)], e[4 * (i & 1) + 2]);
      x.b[i] = make_float2(e[4 * (i & 1) + 1], e[4 * (i & 1) + 3]);
    }
  }
}

template <typename T, bool HALF, bool VEC, typename P>
__device__ __forceinline__ void store_pairs(T* row, const P& at, const Pairs& x) {
  if constexpr (VEC) {
    float u[8], v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (HALF) {
        u[2 * i] = x.a[i].x, u[2 * i + 1] = x.a[i].y;
        v[2 * i] = x.b[i].x, v[2 * i + 1] = x.b[i].y;
      } else {
        float(&e)[8] = i < 2 ? u : v;
        e[4 * (i & 1)] = x.a[i].x, e[4 * (i & 1) + 1] = x.b[i].x;
        e[4 * (i & 1) + 2] = x.a[i].y, e[4 * (i & 1) + 3] = x.b[i].y;
      }
    }
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(row + at.o0)[0] = make_float4(u[0], u[1], u[2], u[3]);
      reinterpret_cast<float4*>(row + at.o0)[1] = make_float4(u[4], u[5], u[6], u[7]);
      reinterpret_cast<float4*>(row + at.o1)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(row + at.o1)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(row + at.o0) =
          make_uint4(pack2(u[0], u[1], T()), pack2(u[2], u[3], T()), pack2(u[4], u[5], T()), pack2(u[6], u[7], T()));
      *reinterpret_cast<uint4*>(row + at.o1) =
          make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Elem<T>::store(row + at.first(2 * i), x.a[i].x);
      Elem<T>::store(row + at.second(2 * i), x.b[i].x);
      Elem<T>::store(row + at.first(2 * i + 1), x.a[i].y);
      Elem<T>::store(row + at.second(2 * i + 1), x.b[i].y);
    }
  }
}

// The weights of the thread's elements, from a row of D weights in 32 bits or in the data's type.
template <typename T, int D, bool HALF, bool VEC>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int row, const Place<D, HALF>& at, Pairs& x) {
  if (f32) {
    Raw<float> raw;
    load_raw<float, VEC>(static_cast<const float*>(w) + static_cast<long long>(row) * D, at, raw);
    to_pairs<float, HALF, VEC>(raw, x);
  } else {
    Raw<T> raw;
    load_raw<T, VEC>(static_cast<const T*>(w) + static_cast<long long>(row) * D, at, raw);
    to_pairs<T, HALF, VEC>(raw, x);
  }
}

// Cosines and sines of the thread's pairs at a position, with the factor; 1 and 0 for what is not rotated.
struct Turn {
  float2 c[4], s[4];
};
template <int D, bool HALF>
__device__ __forceinline__ void turn_of(const RotaryParams& p, const Place<D, HALF>& at, long long pos, Turn& r) {
  const double t = static_cast<double>(pos) * 0.15915494309189533577;   // 1 / (2 pi)
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float sn = 0.f, cs = 1.f;
    if (at.pair(j) < at.rd2) {
      double turns = t * __ldg(p.inv_freq + at.pair(j));
      turns -= rint(turns);
      sincospif(2.f * static_cast<float>(turns), &sn, &cs);
      cs *= p.factor;
      sn *= p.factor * p.sign;
    }
    (j & 1 ? r.c[j >> 1].y : r.c[j >> 1].x) = cs;
    (j & 1 ? r.s[j >> 1].y : r.s[j >> 1].x) = sn;
  }
}
__device__ __forceinline__ void rotate(Pairs& x, const Turn& r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 minus = make_float2(-r.s[i].x, -r.s[i].y);
    const float2 a = __ffma2_rn(x.b[i], minus, __fmul2_rn(x.a[i], r.c[i]));
    x.b[i] = __ffma2_rn(x.b[i], r.c[i], __fmul2_rn(x.a[i], r.s[i]));
    x.a[i] = a;
  }
}
__device__ __forceinline__ void scale_by(Pairs& x, float f) {
  const float2 f2 = make_float2(f, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.a[i] = __fmul2_rn(x.a[i], f2);
    x.b[i] = __fmul2_rn(x.b[i], f2);
  }
}
__device__ __forceinline__ void times(Pairs& x, const Pairs& w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.a[i] = __fmul2_rn(x.a[i], w.a[i]);
    x.b[i] = __fmul2_rn(x.b[i], w.b[i]);
  }
}
__device__ __forceinline__ float dot(const Pairs& x, const Pairs& y) {
  float2 s = __fmul2_rn(x.a[0], y.a[0]), t = __fmul2_rn(x.b[0], y.b[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    s = __ffma2_rn(x.a[i], y.a[i], s);
    t = __ffma2_rn(x.b[i], y.b[i], t);
  }
  return (s.x + s.y) + (t.x + t.y);
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

// Forward, and with sign = -1 the backward of a rotation without a norm. The units (tile of tokens, head), heads inside, are
// cut into equal spans, one per CTA. PAGED: k and v go into the pages of a cache, rows beyond a sequence's count are not
// stored there and are zero in q's result.
template <typename T, int D, bool HALF, bool VEC, bool PAGED>
__global__ void __launch_bounds__(kRotThreads, kRotCtas) omni_rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int LPR = D / 16;                       // lanes of a row
  constexpr int ROWS = kRotThreads / LPR;
  const Place<D, HALF> at(threadIdx.x % LPR, p.rotary_dim);
  grid_wait();
  grid_go();
  unsigned u = blockIdx.x * p.span;
  const unsigned end = min(u + p.span, p.units);
  while (u < end) {
    const unsigned tile = u / p.heads_total;
    const int h0 = static_cast<int>(u - tile * p.heads_total), h1 = static_cast<int>(min(static_cast<unsigned>(p.heads_total), h0 + (end - u)));
    u += h1 - h0;
    const unsigned token = tile * ROWS + threadIdx.x / LPR;
    const bool inside = token < p.tokens;
    const int b = inside ? static_cast<int>(token / p.N) : 0, n = inside ? static_cast<int>(token - static_cast<unsigned>(b) * p.N) : 0;

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
    Turn turn;
    bool turned = false;

    // the heads of one of q, k, v that lie in the span
    int base = 0;
#pragma unroll 1
    for (int g = 0; g < (PAGED ? 3 : 2); ++g) {
      const RotarySegment& sg = p.seg[g];
      const int from = max(h0 - base, 0), to = min(h1 - base, sg.heads);
      base += sg.heads;
      if (from >= to) continue;
      const T* x = static_cast<const T*>(sg.x) + b * sg.xs_b + n * sg.xs_n + from * sg.xs_h;
      Raw<T> next{};
      if (live) load_raw<T, VEC>(x, at, next);   // what is not stored is not read
      if (g < 2 && !turned) {   // the first rows are on their way meanwhile
        turn_of<D, HALF>(p, at, position_of(p, b, n), turn);
        turned = true;
      }
      T* y;
      long long ys;
      bool store = inside;
      if (PAGED && g > 0) {
        y = static_cast<T*>(sg.y) + (slot + (static_cast<long long>(from) << p.page_shift)) * D;
        ys = static_cast<long long>(D) << p.page_shift;
        store = slot >= 0;
      } else {
        y = static_cast<T*>(sg.y) + ((static_cast<long long>(b) * sg.heads + from) * p.N + n) * D;
        ys = static_cast<long long>(p.N) * D;
      }
      const bool zero = PAGED && g == 0 && !live;
      const bool norm = sg.w != nullptr;
      Pairs w;
      if (norm) load_weight<T, D, HALF, VEC>(sg.w, p.w_f32, p.w_per_head ? from : 0, at, w);
#pragma unroll 1
      for (int h = from; h < to; ++h) {
        Pairs v;
        to_pairs<T, HALF, VEC>(next, v);
        x += sg.xs_h;
        if (h + 1 < to && live) load_raw<T, VEC>(x, at, next);
        if (norm) {
          const float r = rsqrtf(row_sum<LPR>(dot(v, v)) * (1.f / D) + p.eps);
          times(v, w);
          if (g < 2) rotate(v, turn);
          scale_by(v, r);
          if (p.w_per_head && h + 1 < to) load_weight<T, D, HALF, VEC>(sg.w, p.w_f32, h + 1, at, w);
        } else if (g < 2) {
          rotate(v, turn);
        }
        if (zero) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v.a[i] = v.b[i] = make_float2(0.f, 0.f);
        }
        if (store) store_pairs<T, HALF, VEC>(y, at, v);
        y += ys;
      }
    }
  }
}

// Backward with a norm: dx of every row and, per CTA, the sum over its rows of the weight's gradient (added up by
// omni_rotary_dw_kernel in a fixed order, so the result does not depend on which CTA ran first). The units (tile of tokens,
// head), those of q and then those of k, are cut into equal spans. With one weight for all heads the heads of a tile follow
// one another (its angles are computed once), with a weight for each head the tiles of a head do (its sum stays in registers).
template <typename T, int D, bool HALF, bool VEC, bool PER_HEAD>
__global__ void __launch_bounds__(kRotThreads, 2) omni_rotary_bwd_kernel(const __grid_constant__ RotaryBwdParams bp) {
  constexpr int LPR = D / 16;
  constexpr int ROWS = kRotThreads / LPR;
  __shared__ float red[kRotThreads / 32][D];
  const RotaryParams& p = bp.f;
  const Place<D, HALF> at(threadIdx.x % LPR, p.rotary_dim);
  grid_wait();
  grid_go();
  Pairs dw, w;
  Turn turn;
  const unsigned units_q = bp.tiles * p.seg[0].heads;
  unsigned u = blockIdx.x * p.span;
  const unsigned end = min(u + p.span, p.units);

  // adds up the CTA's rows: those of a warp, then the warps, each in a fixed order
  auto flush = [&](int sum) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = dw.a[i].x, v[2 * i + 1] = dw.a[i].y, v[8 + 2 * i] = dw.b[i].x, v[9 + 2 * i] = dw.b[i].y;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int o = 16; o >= LPR; o >>= 1) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
    }
    if ((threadIdx.x & 31) < LPR) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        red[threadIdx.x >> 5][VEC && HALF ? at.o0 + j : at.first(j)] = v[j];
        red[threadIdx.x >> 5][VEC && HALF ? at.o1 + j : at.second(j)] = v[8 + j];
      }
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < kRotThreads / 32; ++i) total += red[i][threadIdx.x];
      bp.partial[static_cast<long long>(blockIdx.x + sum) * D + threadIdx.x] = total;   // sums of a CTA follow one another: a place each
    }
    __syncthreads();
  };

  int sum_of = -1;   // which sum is in dw: 0 and 1 for q's and k's one weight, else the head (k's behind q's)
  while (u < end) {
    const int g = u < units_q ? 0 : 1;
    const RotarySegment& sg = p.seg[g];
    const unsigned in = g == 0 ? u : u - units_q, per = PER_HEAD ? bp.tiles : sg.heads;
    const unsigned major = in / per, minor = in - major * per;
    const unsigned tile = PER_HEAD ? minor : major;
    const int h0 = static_cast<int>(PER_HEAD ? major : minor);
    const int h1 = PER_HEAD ? h0 + 1 : static_cast<int>(min(static_cast<unsigned>(sg.heads), h0 + (end - u)));
    u += h1 - h0;
    const int sum = PER_HEAD ? h0 + (g == 0 ? 0 : p.seg[0].heads) : g;
    if (sum != sum_of) {
      if (sum_of >= 0) flush(sum_of);
      sum_of = sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) dw.a[i] = dw.b[i] = make_float2(0.f, 0.f);
      load_weight<T, D, HALF, VEC>(sg.w, p.w_f32, PER_HEAD ? h0 : 0, at, w);
    }
    const unsigned token = tile * ROWS + threadIdx.x / LPR;
    const bool inside = token < p.tokens;
    const int b = inside ? static_cast<int>(token / p.N) : 0, n = inside ? static_cast<int>(token - static_cast<unsigned>(b) * p.N) : 0;
    const T* x = static_cast<const T*>(sg.x) + b * sg.xs_b + n * sg.xs_n + h0 * sg.xs_h;
    const T* gx = static_cast<const T*>(bp.g[g].x) + b * bp.g[g].xs_b + n * bp.g[g].xs_n + h0 * bp.g[g].xs_h;
    T* y = static_cast<T*>(sg.y) + ((static_cast<long long>(b) * sg.heads + h0) * p.N + n) * D;
    Raw<T> nx, ng;
    load_raw<T, VEC>(x, at, nx);
    load_raw<T, VEC>(gx, at, ng);
    turn_of<D, HALF>(p, at, position_of(p, b, n), turn);   // sign = -1: the rotation back
#pragma unroll 1
    for (int h = h0; h < h1; ++h) {
      Pairs v, d;
      to_pairs<T, HALF, VEC>(nx, v);
      to_pairs<T, HALF, VEC>(ng, d);
      if (h + 1 < h1) {
        x += sg.xs_h;
        gx += bp.g[g].xs_h;
        load_raw<T, VEC>(x, at, nx);
        load_raw<T, VEC>(gx, at, ng);
      }
      const float r = rsqrtf(row_sum<LPR>(dot(v, v)) * (1.f / D) + p.eps);
      rotate(d, turn);
      scale_by(v, r);   // x_hat
      if (inside) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dw.a[i] = __ffma2_rn(d.a[i], v.a[i], dw.a[i]);
          dw.b[i] = __ffma2_rn(d.b[i], v.b[i], dw.b[i]);
        }
      }
      times(d, w);
      const float m = -row_sum<LPR>(dot(d, v)) * (1.f / D);
      const float2 m2 = make_float2(m, m);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d.a[i] = __ffma2_rn(v.a[i], m2, d.a[i]);
        d.b[i] = __ffma2_rn(v.b[i], m2, d.b[i]);
      }
      scale_by(d, r);
      if (inside) store_pairs<T, HALF, VEC>(y, at, d);
      y += static_cast<long long>(p.N) * D;
    }
  }
  if (sum_of >= 0) flush(sum_of);
}

// Adds up the CTAs' shares of each weight row's gradient, 32 columns to a CTA, in the order of the CTAs.
template <int D>
__global__ void __launch_bounds__(1024) omni_rotary_dw_kernel(const __grid_constant__ RotaryBwdParams bp) {
  __shared__ float red[32][33];
  const RotaryParams& p = bp.f;
  const int sum = blockIdx.x, hq = p.seg[0].heads;
  const bool per_head = p.w_per_head;
  const int g = per_head ? (sum < hq ? 0 : 1) : (bp.sums == 2 ? sum : (hq > 0 ? 0 : 1));
  const int row = per_head ? sum - (g == 0 ? 0 : hq) : 0;
  const int place = per_head ? sum : g;
  // the units that went into this sum, and the CTAs that had them
  const unsigned u0 = per_head ? bp.tiles * sum : (g == 0 ? 0 : bp.tiles * hq), u1 = per_head ? u0 + bp.tiles : u0 + bp.tiles * p.seg[g].heads;
  const unsigned c0 = u0 / p.span, c1 = (u1 - 1) / p.span;
  const int col = blockIdx.y * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  grid_wait();
  float total = 0.f;
#pragma unroll 4
  for (unsigned c = c0 + lane; c <= c1; c += 32) total += __ldcg(bp.partial + static_cast<long long>(c + place) * D + col);
  red[lane][threadIdx.x & 31] = total;
  __syncthreads();
  if (lane != 0) return;
  total = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) total += red[i][threadIdx.x];
  void* to = bp.dw[g];
  const long long e = static_cast<long long>(row) * D + col;
  if (p.w_f32) {
    static_cast<float*>(to)[e] = total;
  } else if (p.bf16) {
    static_cast<__nv_bfloat16*>(to)[e] = __float2bfloat16_rn(total);
  } else {
    static_cast<__half*>(to)[e] = __float2half_rn(total);
  }
}

// Spans of the units, one per CTA: as many CTAs as `most`, or one per unit.
void cut(RotaryParams& p, long long units, int most, int& ctas) {
  p.units = static_cast<unsigned>(units);
  p.span = static_cast<unsigned>((units + most - 1) / most);
  ctas = static_cast<int>((units + p.span - 1) / p.span);
}
unsigned tiles_of(const RotaryParams& p, int D) {
  const int rows = kRotThreads / (D / 16);
  return static_cast<unsigned>((p.tokens + rows - 1) / rows);
}

template <typename T, int D, bool HALF, bool VEC>
cudaError_t launch_t(RotaryParams p, bool paged, cudaStream_t stream) {
  int ctas = 0;
  cut(p, static_cast<long long>(tiles_of(p, D)) * p.heads_total, kSms * kRotCtas, ctas);
  if constexpr (sizeof(T) == 2) {
    if (paged) return launch_chained(omni_rotary_kernel<T, D, HALF, VEC, true>, ctas, kRotThreads, 0, stream, p);
  }
  return launch_chained(omni_rotary_kernel<T, D, HALF, VEC, false>, ctas, kRotThreads, 0, stream, p);
}

void cut_bwd(RotaryBwdParams& bp, int D, int& ctas) {
  RotaryParams& p = bp.f;
  bp.tiles = tiles_of(p, D);
  bp.sums = p.w_per_head ? p.seg[0].heads + p.seg[1].heads : (p.seg[0].heads > 0) + (p.seg[1].heads > 0);
  cut(p, static_cast<long long>(bp.tiles) * (p.seg[0].heads + p.seg[1].heads), kSms * 2, ctas);
}

template <typename T, int D, bool HALF, bool VEC>
cudaError_t launch_bwd_t(RotaryBwdParams bp, cudaStream_t stream) {
  int ctas = 0;
  cut_bwd(bp, D, ctas);
  const cudaError_t e = launch_chained(bp.f.w_per_head ? omni_rotary_bwd_kernel<T, D, HALF, VEC, true> : omni_rotary_bwd_kernel<T, D, HALF, VEC, false>,
                                       ctas, kRotThreads, 0, stream, bp);
  if (e != cudaSuccess) return e;
  return launch_chained(omni_rotary_dw_kernel<D>, dim3(bp.sums, D / 32), 1024, 0, stream, bp);
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
  RotaryBwdParams bp{};
  bp.f = p;
  int ctas = 0;
  cut_bwd(bp, head_dim, ctas);
  return static_cast<long long>(ctas + p.seg[0].heads + p.seg[1].heads + 1) * head_dim;
}
bool rotary_fits(const RotaryParams& p, int head_dim) {
  return static_cast<long long>(tiles_of(p, head_dim)) * (p.seg[0].heads + p.seg[1].heads + p.seg[2].heads) < (1LL << 31);
}

}  // namespace omni
