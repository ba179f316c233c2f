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
// that many lanes' shuffles. Measured, 64 heads of 128, 8 192 tokens, bf16: forward 47 us for 268 MB, backward with norms 67 us
// for 402 MB (5.7 and 6.0 TB/s) and 5 to 7 us for the weights' sums; fp32: 106 us for 537 MB, with norms 155 us in all for 805 MB
// (5.1 and 5.2), without 97 us for 537 MB.
#include "omni_cache_line.cuh"
#include "omni_launch.h"
#include "omni_rotary.cuh"

namespace omni {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotCtas = 2;        // CTAs on an SM: 128 registers a thread
constexpr int kSms = 148;
constexpr int kRotAhead = 4;       // heads that a thread of the forward has on their way
constexpr int kRotBwdStages = 3;   // stages of the backward's ring

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <>
struct Elem<float> {
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

// A warp's ring in shared memory for the rows that the backward is going to need (VEC), copied there with cp.async, so that
// several heads are on their way without taking registers, of which it has none to spare (the forward, with half the rows,
// keeps kRotAhead heads in registers: 46 us against 50 with this ring; the backward 71 against 79 with one head ahead in
// registers). A copy's 32 lanes read whole neighbouring 32-byte sectors - in the threads' own places of an interleaved row half
// of each was read twice, 116 us - so lanes copy for one another: a __syncwarp stands between the wait and the reads. The
// 16-byte chunks are spread over the banks (place), for the copies and for the threads' own reads.
template <typename T, int D, int STAGES>
struct RowRing {
  static constexpr int kLanes = D / 16;                            // of a row
  static constexpr int kRow = D * static_cast<int>(sizeof(T)) / 16;   // chunks of a row
  static constexpr int kCopies = kRow / kLanes;                    // chunks that a lane copies, and that it reads
  static constexpr int kStage = 32 * kCopies * 16;                 // bytes of a warp
  static constexpr int kBytes = STAGES * kStage * (kRotThreads / 32);
  uint32_t base;
  uint32_t own[kCopies];    // where this thread's chunks are
  const T* from[kCopies];   // what it copies next
  uint32_t live;            // bit i: copy i is of a row that is needed

  static __device__ __forceinline__ uint32_t place(int chunk) {
    const int line = chunk >> 3;
    return (line * 8 + ((chunk & 7) ^ (line & 3))) * 16;
  }
  template <typename P>
  __device__ __forceinline__ RowRing(uint32_t smem, const P& at) : base(smem + (threadIdx.x >> 5) * (STAGES * kStage)), live(0) {
    const int row = (threadIdx.x & 31) / kLanes;
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < kCopies; ++c) own[c] = base + place(row * kRow + (c < kCopies / 2 ? at.o0 : at.o1) / E + c % (kCopies / 2));
  }
  // `x`: the first row that this thread itself is going to need; `needed`: whether it is.
  __device__ __forceinline__ void start(const T* x, bool needed) {
    const int lane = threadIdx.x & 31;
    const unsigned all = __ballot_sync(0xFFFFFFFFu, needed);
    live = 0;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int chunk = lane + 32 * i, owner = chunk / kRow * kLanes;
      from[i] = reinterpret_cast<const T*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(x), owner)) + chunk % kRow * (16 / sizeof(T));
      live |= (all >> owner & 1u) << i;
    }
  }
  // Copies a head's rows, and steps to the next head's.
  __device__ __forceinline__ void issue(int stage, long long step) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      if (live >> i & 1u) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + stage * kStage + place(lane + 32 * i)), "l"(from[i]) : "memory");
      }
      from[i] += step;
    }
  }
  __device__ __forceinline__ void read(int stage, Raw<T>& raw) const {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < kCopies; ++c) raw.c[c] = lds_v4(own[c] + stage * kStage);
  }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ring_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

struct Turn {
  float2 c[4], s[4];
};
// Cosines and sines of two angles given in turns, at most half a turn: Taylor's series about the nearest quarter turn, |x| <= pi / 4,
// to x^9 and x^10 (what is left out is below 2^-28). The turns are off by 2^-26, which is 2^-23.4 of an angle; x by its product's
// rounding and 2 pi's, 2^-25 each; the sums by 2^-24: together less than 2^-22 (on 8 million angles 2^-22.7).
__device__ __forceinline__ void sincos_turns(float2 turns, float2& sn, float2& cs) {
  auto both = [](float v) { return make_float2(v, v); };
  constexpr float kBig = 12582912.f;   // 1.5 * 2^23: a sum with it is rounded to whole numbers
  const float2 sum = __ffma2_rn(turns, both(4.f), both(kBig));
  const float2 quarters = __fadd2_rn(sum, both(-kBig));
  const float2 x = __fmul2_rn(__ffma2_rn(quarters, both(-0.25f), turns), both(6.2831853071795865f));
  const float2 z = __fmul2_rn(x, x);
  float2 s = __ffma2_rn(z, both(1.f / 362880.f), both(-1.f / 5040.f));
  s = __ffma2_rn(s, z, both(1.f / 120.f));
  s = __ffma2_rn(s, z, both(-1.f / 6.f));
  s = __ffma2_rn(__fmul2_rn(s, z), x, x);
  float2 c = __ffma2_rn(z, both(-1.f / 3628800.f), both(1.f / 40320.f));
  c = __ffma2_rn(c, z, both(-1.f / 720.f));
  c = __ffma2_rn(c, z, both(1.f / 24.f));
  c = __ffma2_rn(c, z, both(-0.5f));
  c = __ffma2_rn(c, z, both(1.f));
  auto place = [](int k, float s1, float c1, float& sin_out, float& cos_out) {
    const float a = k & 1 ? c1 : s1, b = k & 1 ? s1 : c1;
    sin_out = k & 2 ? -a : a;
    cos_out = (k + 1) & 2 ? -b : b;
  };
  place(__float_as_int(sum.x), s.x, c.x, sn.x, cs.x);
  place(__float_as_int(sum.y), s.y, c.y, sn.y, cs.y);
}
// Cosines and sines of the thread's pairs at a position, with the factor. EXACT: as above, for results in 32 bits: fp32 data, and
// gradients of fp32 weights whatever the data's type. Else the special function unit's sine and cosine, which take
// fewer instructions: the unit's own 2^-21.2 for angles within half a turn, 2^-23.4 of the turns, 2^-23 of the product with 2 pi and
// 2^-23.4 of 2 pi itself, less than 2^-20.4 together. Forward, bf16, head_dim 128: 64 heads of 8 192 tokens 47.3 us EXACT and 46.9,
// 8 heads of 65 536 53.3 and 51.0, 2 heads of 262 144 92.6 and 84.4.
template <bool EXACT, int D, bool HALF>
__device__ __forceinline__ void turn_of(const RotaryParams& p, const Place<D, HALF>& at, long long pos, Turn& r) {
  const double t = static_cast<double>(pos) * 0.15915494309189533577;   // 1 / (2 pi)
  auto turns_of = [&](int j) {
    if (at.pair(j) >= at.rd2) return 0.f;   // (not used)
    const double turns = t * __ldg(p.inv_freq + at.pair(j));
    return static_cast<float>(turns - rint(turns));
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 turns = make_float2(turns_of(2 * i), turns_of(2 * i + 1));
    if constexpr (EXACT) {
      sincos_turns(turns, r.s[i], r.c[i]);
    } else {
      __sincosf(6.2831853071795865f * turns.x, &r.s[i].x, &r.c[i].x);
      __sincosf(6.2831853071795865f * turns.y, &r.s[i].y, &r.c[i].y);
    }
    r.c[i] = __fmul2_rn(r.c[i], make_float2(p.factor, p.factor));
    r.s[i] = __fmul2_rn(r.s[i], make_float2(p.factor * p.sign, p.factor * p.sign));
  }
}
// Pairs behind the rotated part pass through as they are (a turn by cosine 1 and sine 0 would make the neighbour of an infinite
// element NaN). With vector loads in the half layout all of a thread's pairs are rotated or none.
template <bool VEC, int D, bool HALF>
__device__ __forceinline__ void rotate(Pairs& x, const Turn& r, const Place<D, HALF>& at) {
  const int n = at.rd2 - at.pair(0);   // how many are rotated
  if constexpr (VEC) {
    if (n <= 0) return;
  }
  Pairs y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 minus = make_float2(-r.s[i].x, -r.s[i].y);
    y.a[i] = __ffma2_rn(x.b[i], minus, __fmul2_rn(x.a[i], r.c[i]));
    y.b[i] = __ffma2_rn(x.b[i], r.c[i], __fmul2_rn(x.a[i], r.s[i]));
    if constexpr (!VEC) {   // fewer registers: fp32, a weight for each head, half layout, rows off their boundaries 342 us with the branches, 315 so
      x.a[i] = make_float2(2 * i < n ? y.a[i].x : x.a[i].x, 2 * i + 1 < n ? y.a[i].y : x.a[i].y);
      x.b[i] = make_float2(2 * i < n ? y.b[i].x : x.b[i].x, 2 * i + 1 < n ? y.b[i].y : x.b[i].y);
    }
  }
  if constexpr (VEC && HALF) {
    x = y;
  } else if constexpr (VEC) {
    if (n >= 8) {
      x = y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i < n) x.a[i].x = y.a[i].x, x.b[i].x = y.b[i].x;
        if (2 * i + 1 < n) x.a[i].y = y.a[i].y, x.b[i].y = y.b[i].y;
      }
    }
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
  constexpr int kAhead = sizeof(T) == 4 ? 2 : kRotAhead;
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

    // The span's heads in order, of q, then k, then v, kAhead of them on their way. What is not stored is not read.
    int rd = h0, rd_end = 0, rd_seg = -1;   // next head to be read, where its segment ends
    const T* rd_x = nullptr;
    long long rd_step = 0;
    auto read = [&](Raw<T>& raw) {
      if (rd >= h1) return;
      if (rd >= rd_end) {   // the same in all threads
        do {
          ++rd_seg;
          rd_end += p.seg[rd_seg].heads;
        } while (rd >= rd_end);
        const RotarySegment& sg = p.seg[rd_seg];
        rd_step = sg.xs_h;
        rd_x = static_cast<const T*>(sg.x) + b * sg.xs_b + n * sg.xs_n + (rd - (rd_end - sg.heads)) * rd_step;
      }
      if (live) load_raw<T, VEC>(rd_x, at, raw);
      rd_x += rd_step;
      ++rd;
    };
    Raw<T> raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      raw[i] = Raw<T>{};
      read(raw[i]);
    }

    int seg = -1, seg_end = 0, hl = 0;   // of the head at hand; its number in the segment
    T* y = nullptr;
    long long ys = 0;
    bool store = false, zero = false, norm = false;
    Pairs w;
#pragma unroll 1
    for (int h = h0; h < h1;) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i, ++h) {
        if (h >= h1) break;
        if (h >= seg_end) {
          do {
            ++seg;
            seg_end += p.seg[seg].heads;
          } while (h >= seg_end);
          const RotarySegment& sg = p.seg[seg];
          hl = h - (seg_end - sg.heads);
          if (PAGED && seg > 0) {
            y = static_cast<T*>(sg.y) + (slot + (static_cast<long long>(hl) << p.page_shift)) * D;
            ys = static_cast<long long>(D) << p.page_shift;
            store = slot >= 0;
            zero = false;
          } else {
            y = static_cast<T*>(sg.y) + ((static_cast<long long>(b) * sg.heads + hl) * p.N + n) * D;
            ys = static_cast<long long>(p.N) * D;
            store = inside;
            zero = PAGED && !live;
          }
          norm = sg.w != nullptr;
          if (norm) load_weight<T, D, HALF, VEC>(sg.w, p.w_f32, p.w_per_head ? hl : 0, at, w);
          if (seg < 2 && !turned) {
            turn_of<sizeof(T) == 4>(p, at, position_of(p, b, n), turn);
            turned = true;
          }
        }
        Pairs v;
        to_pairs<T, HALF, VEC>(raw[i], v);
        read(raw[i]);
        if (norm) {
          const float r = rsqrtf(row_sum<LPR>(dot(v, v)) * (1.f / D) + p.eps);
          times(v, w);
          if (seg < 2) rotate<VEC>(v, turn, at);
          scale_by(v, r);
          if (p.w_per_head && h + 1 < min(h1, seg_end)) load_weight<T, D, HALF, VEC>(p.seg[seg].w, p.w_f32, ++hl, at, w);
        } else if (seg < 2) {
          rotate<VEC>(v, turn, at);
        }
        if (zero) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v.a[j] = v.b[j] = make_float2(0.f, 0.f);
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
__global__ void __launch_bounds__(kRotThreads, kRotCtas) omni_rotary_bwd_kernel(const __grid_constant__ RotaryBwdParams bp) {
  constexpr int LPR = D / 16;
  constexpr int ROWS = kRotThreads / LPR;
  constexpr int kStages = kRotBwdStages;
  __shared__ float red[kRotThreads / 32][D];
  extern __shared__ __align__(16) uint8_t rotary_smem[];
  const RotaryParams& p = bp.f;
  const Place<D, HALF> at(threadIdx.x % LPR, p.rotary_dim);
  RowRing<T, D, kStages> ring_x(smem_u32(rotary_smem), at), ring_g(smem_u32(rotary_smem) + RowRing<T, D, kStages>::kBytes, at);
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
    const int n_rows = h1 - h0;
    if constexpr (VEC) {
      __syncwarp();
      ring_x.start(x, inside);
      ring_g.start(gx, inside);
    }
    auto read_ahead = [&](int i) {   // row i of the run
      if constexpr (VEC) {
        if (i < n_rows) {
          ring_x.issue(i % kStages, sg.xs_h);
          ring_g.issue(i % kStages, bp.g[g].xs_h);
        }
        ring_commit();
      }
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) read_ahead(i);
    // sign = -1: the rotation back. A weight for each head means angles for each row: 106 us with the unit's sines, 117 EXACT (64 heads
    // of 8 192 tokens, bf16, half layout).
    if (sizeof(T) == 4 || p.w_f32) {
      turn_of<true>(p, at, position_of(p, b, n), turn);
    } else {
      turn_of<false>(p, at, position_of(p, b, n), turn);
    }
#pragma unroll 1
    for (int i = 0; i < n_rows; ++i) {
      Pairs v, d;
      {
        Raw<T> raw_x, raw_g;
        if constexpr (VEC) {
          ring_wait<kStages - 2>();
          ring_x.read(i % kStages, raw_x);
          ring_g.read(i % kStages, raw_g);
        } else {
          load_raw<T, false>(x + i * sg.xs_h, at, raw_x);
          load_raw<T, false>(gx + i * bp.g[g].xs_h, at, raw_g);
        }
        to_pairs<T, HALF, VEC>(raw_x, v);
        to_pairs<T, HALF, VEC>(raw_g, d);
      }
      read_ahead(i + kStages - 1);
      const float r = rsqrtf(row_sum<LPR>(dot(v, v)) * (1.f / D) + p.eps);
      rotate<VEC>(d, turn, at);
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
    if constexpr (VEC) ring_wait<0>();
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

// A launch with `smem` bytes of rings, chained to its predecessor.
template <int SMEM, typename K, typename P>
cudaError_t launch_ring(K kern, int ctas, cudaStream_t stream, const P& p, SmemAttrOnce (&once)[kMaxDevices]) {
  if constexpr (SMEM > 32 * 1024) {   // (beside what a kernel has statically)
    const cudaError_t e = ensure_smem_attr(kern, SMEM, once);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(kern, ctas, kRotThreads, SMEM, stream, p);
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
  cut(p, static_cast<long long>(bp.tiles) * (p.seg[0].heads + p.seg[1].heads), kSms * kRotCtas, ctas);
}

template <typename T, int D, bool HALF, bool VEC>
cudaError_t launch_bwd_t(RotaryBwdParams bp, cudaStream_t stream) {
  int ctas = 0;
  cut_bwd(bp, D, ctas);
  constexpr int kSmem = VEC ? 2 * RowRing<T, D, kRotBwdStages>::kBytes : 0;
  static SmemAttrOnce once_shared[kMaxDevices], once_head[kMaxDevices];
  const cudaError_t e = bp.f.w_per_head ? launch_ring<kSmem>(omni_rotary_bwd_kernel<T, D, HALF, VEC, true>, ctas, stream, bp, once_head)
                                        : launch_ring<kSmem>(omni_rotary_bwd_kernel<T, D, HALF, VEC, false>, ctas, stream, bp, once_shared);
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
