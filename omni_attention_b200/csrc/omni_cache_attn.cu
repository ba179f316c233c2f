// Attention of a few new tokens over a paged key/value cache: out = softmax(cap(q k^T * scale)) v for T query tokens of
// each sequence, H query heads sharing Hkv key/value heads, every row with its own number of visible keys.
//
// Bound: memory. Every key and value is read once and serves G * T query rows (G = H / Hkv), 2 * G * T operations per
// byte: with 16 rows that is a twentieth of what the card computes in the time of the read. So the query rows of a
// key/value head go through the tensor cores together as one 16-row tile (mma.sync: 16 rows would fill an eighth of a
// tcgen05 tile), and all that matters is that enough reads are in flight on every SM.
//
// Split: the keys of all (sequence, key/value head, 16-row tile) triples, in tiles of kTileKeys, form one line of units
// that is cut into equal spans, one per CTA; lengths are read on the device, so the cut is even however ragged the batch
// is, and the launch does not depend on them (it can be captured once and replayed as the cache grows). A span may end
// inside a triple: then its rows' (maximum, sum, O) go to the workspace and omni_cache_join_kernel puts the shares
// together, in the order of the keys. A triple inside one span is written out directly.
//
// Inside a CTA each warp has its own 16 keys of a tile, its own ring of cp.async stages and its own running maximum, sum
// and O (no barrier between warps until the end of a triple, where the warps' shares are joined through shared memory).
// The maximum moves only when it would grow by more than 2^8 (scores are in the log2 domain), P goes into the product as
// a 16-bit value plus the 16-bit rest (two products; the tensor cores have the room), so the only rounding that shows
// is that of the result.
#include "omni_cache_line.cuh"
#include "omni_launch.h"

namespace omni {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTileKeys = 16 * kWarps;
constexpr int kRows = 16;

template <int D>
struct CacheCfg {
  static constexpr int kStages = 3;
  static constexpr int kStageBytes = 2 * 16 * D * 2;                       // K and V of 16 keys
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kJoin = kWarps * kRows * (D + 4) * 4;               // O shares, over the ring
  static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
};

// ---------------------------------------------------------------------------------------------------------------------
// instructions
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? 16 : 0;   // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t u) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
}

// Byte offset of 16-byte chunk c of row r in a [16][D] tile whose chunks are spread over the banks: eight rows read at
// the same chunk (what ldmatrix does) touch all 32 banks once.
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  if constexpr (D >= 64) {
    return static_cast<uint32_t>(r * (D * 2) + ((c ^ (r & 7)) << 4));
  } else {   // two rows of 64 bytes to a line of 128
    const int line = r >> 1;
    return static_cast<uint32_t>(line * 128 + (((((r & 1) << 2) + c) ^ (line & 7)) << 4));
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------------------------------------------------
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads) omni_cache_attn_kernel(const __grid_constant__ CacheAttnParams p, const __grid_constant__ CacheLaunch how) {
  using Cfg = CacheCfg<D>;
  constexpr int KS = D / 16;        // steps of Q K^T
  constexpr int CH = D / 8;         // 16-byte chunks of a row
  constexpr int ITEMS = 16 * CH / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int quad = lane >> 2, pos = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * (Cfg::kStages * Cfg::kStageBytes);
  const float scale_log2 = p.scale * 1.4426950408889634f;
  Walk walk(p, how);
  Piece pc;
  while (walk.next(p, pc)) {
    const int hk = pc.hk, rows = pc.rows, tile0 = pc.tile0, tile1 = pc.tile1;

    // this thread's two rows: their queries as mma operands, their numbers of visible keys
    uint32_t qf[KS][4];
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = pc.rt * kRows + quad + 8 * i;
      lim[i] = 0;
      const uint32_t* src = nullptr;
      if (r < rows) {
        const RowId id = row_of(p, pc.prefix, pc.seg, r);
        lim[i] = min(limit_of(p, id.b, id.t), pc.total);
        src = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + id.b * p.qs_b +
                                                (static_cast<long long>(hk) * p.G + id.g) * p.qs_h + id.t * p.qs_t);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[k][i] = src != nullptr ? __ldg(src + 8 * k + pos) : 0u;
        qf[k][2 + i] = src != nullptr ? __ldg(src + 8 * k + 4 + pos) : 0u;
      }
    }
    int lim_max = max(lim[0], lim[1]), lim_min = min(lim[0], lim[1]);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      lim_max = max(lim_max, __shfl_xor_sync(0xFFFFFFFFu, lim_max, o));
      lim_min = min(lim_min, __shfl_xor_sync(0xFFFFFFFFu, lim_min, o));
    }

    float o_acc[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o_acc[i][0] = o_acc[i][1] = o_acc[i][2] = o_acc[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // this warp's 16 keys of tile t begin at key_at(t)
    auto key_at = [&](int t) { return pc.key0 + t * kTileKeys + warp * 16; };
    auto page_at = [&](int t) -> int {
      const int key = key_at(t);
      return t < tile1 && key < lim_max ? __ldg(p.page_table + pc.table_of * p.table_stride + (key >> p.page_shift)) : -1;
    };
    uint32_t there = 0;   // bit (tile & 31): the tile's page exists
    auto issue = [&](int t, int page) {
      if (t < tile1) {
        const int key = key_at(t);
        const bool ok = page >= 0 && page < p.num_pages;
        if (!ok && key < lim_max && p.status != nullptr && lane == 0) atomicCAS(p.status, 0, kStatusBadIndex);
        there = (there & ~(1u << (t & 31))) | (static_cast<uint32_t>(ok) << (t & 31));
        const long long row = ok ? (((static_cast<long long>(page) * p.Hkv + hk) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * D : 0;
        const uint16_t* ks = static_cast<const uint16_t*>(p.k_pages) + row;
        const uint16_t* vs = static_cast<const uint16_t*>(p.v_pages) + row;
        const uint32_t dst = ring + (t % Cfg::kStages) * Cfg::kStageBytes;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          const int item = lane + 32 * i, r = item / CH, c = item % CH;
          const bool read = ok && key + r < lim_max;   // what no row sees is zero, whatever the page holds there
          const uint32_t off = tile_offset<D>(r, c);
          cp_async16(dst + off, ks + (read ? item * 8 : 0), read);
          cp_async16(dst + 16 * D * 2 + off, vs + (read ? item * 8 : 0), read);
        }
      }
      cp_async_commit();
    };

    int pages[Cfg::kStages];
#pragma unroll
    for (int i = 0; i < Cfg::kStages - 1; ++i) pages[i] = page_at(tile0 + i);
    int page_next = page_at(tile0 + Cfg::kStages - 1);
#pragma unroll
    for (int i = 0; i < Cfg::kStages - 1; ++i) issue(tile0 + i, pages[i]);

    for (int t = tile0; t < tile1; ++t) {
      cp_async_wait<Cfg::kStages - 2>();
      __syncwarp();
      issue(t + Cfg::kStages - 1, page_next);   // into the stage that the last round read
      page_next = page_at(t + Cfg::kStages);
      const int key = key_at(t);
      if (key >= lim_max || !(there >> (t & 31) & 1u)) continue;   // the same in all lanes
      const uint32_t sk = ring + (t % Cfg::kStages) * Cfg::kStageBytes, sv = sk + 16 * D * 2;

      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t b[4];
        ldmatrix4(sk + tile_offset<D>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)), b);
        mma16816<BF16>(s[0], qf[k], b[0], b[1]);
        mma16816<BF16>(s[1], qf[k], b[2], b[3]);
      }
      const bool masked = key + 16 > lim_min;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[j][e];
          if (p.softcap > 0.f) {
            x = tanhf(x * (p.scale / p.softcap)) * (p.softcap * 1.4426950408889634f);
          } else {
            x *= scale_log2;
          }
          if (masked && key + 8 * j + 2 * pos + (e & 1) >= lim[e >> 1]) x = -INFINITY;
          s[j][e] = x;
        }
      }
      // running maximum: moved only when it would grow by more than 8 (p <= 2^8 in 32 bits and in either 16-bit type)
      bool move = false;
      float top[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
        v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
        v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
        top[i] = v;
        move |= v > m[i] + 8.f;
      }
      if (__any_sync(0xFFFFFFFFu, move)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float to = fmaxf(m[i], top[i]);
          const float f = m[i] == -INFINITY ? 0.f : ex2_approx(m[i] - to);
          m[i] = to;
          l[i] *= f;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            o_acc[d][2 * i] *= f;
            o_acc[d][2 * i + 1] *= f;
          }
        }
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float at = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float a = ex2_approx(s[j][2 * i] - at), b = ex2_approx(s[j][2 * i + 1] - at);
          l[i] += a + b;
          hi[2 * j + i] = pack16<BF16>(a, b);
          const float2 h = unpack16<BF16>(hi[2 * j + i]);
          lo[2 * j + i] = pack16<BF16>(a - h.x, b - h.y);
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldmatrix4_trans(sv + tile_offset<D>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * d + (lane >> 4)), b);
        mma16816<BF16>(o_acc[2 * d], hi, b[0], b[1]);
        mma16816<BF16>(o_acc[2 * d + 1], hi, b[2], b[3]);
        mma16816<BF16>(o_acc[2 * d], lo, b[0], b[1]);
        mma16816<BF16>(o_acc[2 * d + 1], lo, b[2], b[3]);
      }
    }
    cp_async_wait<0>();

    // ---- the warps' shares of the triple, joined ----
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
      l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
      if (pos == 0) {
        s_m[warp][quad + 8 * i] = m[i];
        s_l[warp][quad + 8 * i] = l[i];
      }
    }
    __syncthreads();   // every warp is through with its stages: the shares go over them
    float* so = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<float2*>(so + (warp * kRows + quad + 8 * i) * (D + 4) + 8 * d + 2 * pos) =
            make_float2(o_acc[d][2 * i], o_acc[d][2 * i + 1]);
      }
    }
    __syncthreads();
    constexpr int LPR = D / 4;    // threads of a row, 4 columns each
    for (int r = threadIdx.x / LPR; r < kRows; r += kThreads / LPR) {
      const int row = pc.rt * kRows + r, col = (threadIdx.x % LPR) * 4;
      if (row >= rows) break;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
      const float at = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2_approx(s_m[w][r] - at);
        const float4 v = *reinterpret_cast<const float4*>(so + (w * kRows + r) * (D + 4) + col);
        sum += f * s_l[w][r];
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
      }
      if (pc.share >= 0) {
        float* to = share_at(p, how, pc.share, D);
        *reinterpret_cast<float4*>(to + r * D + col) = acc;
        if (col == 0) {
          to[kRows * D + r] = top;
          to[kRows * D + kRows + r] = sum;
        }
      } else {
        const long long at_row = out_row(p, row_of(p, pc.prefix, pc.seg, row), hk);
        const bool any = !(sum == 0.f);   // NaN shows
        const float inv = 1.f / sum;
        uint2 out = make_uint2(0u, 0u);
        if (any) {
          out.x = pack16<BF16>(acc.x * inv, acc.y * inv);
          out.y = pack16<BF16>(acc.z * inv, acc.w * inv);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at_row * D + col) = out;
        if (p.lse != nullptr && col == 0) p.lse[at_row] = any ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
      }
    }
    __syncthreads();   // the shares are read: the next triple's stages may go over them
  }
}

// Joins the shares of the rows that no single span covered. One CTA per (sequence, key/value head, 16 rows), a warp per
// row. `pre` is the launch that had the prefix (if there is one), `own` the one that had the sequences' own keys; they may
// be the same launch.
template <int D, bool BF16>
__global__ void __launch_bounds__(128) omni_cache_join_kernel(const __grid_constant__ CacheAttnParams p, const __grid_constant__ CacheLaunch pre,
                                                              const __grid_constant__ CacheLaunch own) {
  constexpr int V = D / 32;   // columns of a lane
  const int rows = p.G * p.T;
  const int groups = (rows + kRows - 1) / kRows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seq = static_cast<int>(blockIdx.x / (static_cast<long long>(p.Hkv) * groups));
  const int in_seq = static_cast<int>(blockIdx.x - static_cast<long long>(seq) * p.Hkv * groups);
  const int hk = in_seq / groups, group = in_seq % groups;

  const Line lo = make_line(p, own);
  long long before = 0;
  for (int b = lane; b < seq; b += 32) before += lo.own_units(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
  const long long tiles = lo.tiles_between(p.prefix, total_of(p, seq));
  const long long triple = static_cast<long long>(hk) * lo.rt_own + group * kRows / own.rows;
  const long long first = lo.prefix_units + before + triple * tiles;
  const long long c0 = first / lo.span, c1 = (first + tiles - 1) / lo.span;
  if (p.prefix == 0 && c0 == c1) return;   // written by the one CTA that had it
  Line lp = lo;
  if (p.prefix > 0) {
    lp = make_line(p, pre);
    if (p.status != nullptr && in_seq == 0) {   // is the prefix in the same pages?
      const int pages = (min(p.prefix, total_of(p, seq)) + (1 << p.page_shift) - 1) >> p.page_shift;
      bool same = true;
      for (int i = threadIdx.x; i < pages; i += blockDim.x) {
        same &= __ldg(p.page_table + seq * p.table_stride + i) == __ldg(p.page_table + lp.prefix_seq * p.table_stride + i);
      }
      if (!same) atomicCAS(p.status, 0, kStatusBadIndex);
    }
  }

  for (int r = warp; r < kRows; r += 4) {
    const int row = group * kRows + r;
    if (row >= rows) break;
    float top = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    auto add = [&](const CacheLaunch& how, long long share, int in) {
      const float* from = share_at(p, how, share, D);
      const float m2 = __ldcg(from + how.rows * D + in), l2 = __ldcg(from + how.rows * D + how.rows + in);
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __ldcg(from + in * D + lane + 32 * i);
      const float to = fmaxf(top, m2), at = to == -INFINITY ? 0.f : to;
      const float f1 = ex2_approx(top - at), f2 = ex2_approx(m2 - at);
      sum = sum * f1 + l2 * f2;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = acc[i] * f1 + v[i] * f2;
      top = to;
    };
    auto add_triple = [&](const CacheLaunch& how, long long from, long long n, long long span, long long whole, int in) {
      const long long i0 = from / span, i1 = (from + n - 1) / span;
      if (i0 == i1) {
        add(how, whole, in);
      } else {
        for (long long i = i0; i <= i1; ++i) add(how, 2 * i + (i == i0 ? 1 : 0), in);
      }
    };
    if (p.prefix > 0) {
      const long long gr = static_cast<long long>(seq) * rows + row;   // the row in the prefix segment
      const long long pt = static_cast<long long>(hk) * lp.rt_prefix + gr / pre.rows;
      add_triple(pre, pt * lp.tiles_prefix, lp.tiles_prefix, lp.span, 2LL * pre.ctas + pt, static_cast<int>(gr % pre.rows));
    }
    add_triple(own, first, tiles, lo.span, 2LL * own.ctas + static_cast<long long>(p.Hkv) * (lo.rt_prefix + static_cast<long long>(seq) * lo.rt_own) + triple,
               row % own.rows);
    const long long at_row = out_row(p, row_of(p, false, seq, row), hk);
    const bool any = !(sum == 0.f);   // NaN shows
    const float inv = 1.f / sum;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float o = any ? acc[i] * inv : 0.f;
      uint16_t* to = static_cast<uint16_t*>(p.out) + at_row * D + lane + 32 * i;
      if constexpr (BF16) {
        *reinterpret_cast<__nv_bfloat16*>(to) = __float2bfloat16_rn(o);
      } else {
        *reinterpret_cast<__half*>(to) = __float2half_rn(o);
      }
    }
    if (p.lse != nullptr && lane == 0) p.lse[at_row] = any ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
  }
}

constexpr int kNarrowCtas = 148 * 2;   // two CTAs on each SM at head_dim 128

// The launches of a call: one over everything, or one over the prefix and one over the sequences' own keys where only one
// of the two has more than 16 rows to a key/value head (the 16-row tile would read its keys once for every 16 rows).
struct Plan {
  CacheLaunch of[2];   // the prefix's, the sequences'; equal if one launch has both
  bool wide[2];
  long long floats;
};

Plan make_plan(int B, int Hkv, long long per, int head_dim, bool prefix, long long capacity) {
  Plan pl;
  pl.floats = 0;
  const long long rows[2] = {B * per, per};
  for (int i = 0; i < 2; ++i) pl.wide[i] = rows[i] > kRows;
  if (!prefix) pl.wide[0] = pl.wide[1];
  const bool one = !prefix || pl.wide[0] == pl.wide[1];
  for (int i = 0; i < 2; ++i) {
    CacheLaunch& how = pl.of[i];
    how.rows = pl.wide[i] ? kWideRows : kRows;
    how.keys = pl.wide[i] ? kWideKeys : kTileKeys;
    how.prefix = prefix && (one || i == 0);
    how.own = one || i == 1;
    if (i == 1 && one) {
      how = pl.of[0];
      break;
    }
    long long triples = 0;
    if (how.prefix) triples += Hkv * ((rows[0] + how.rows - 1) / how.rows);
    if (how.own) triples += static_cast<long long>(B) * Hkv * ((rows[1] + how.rows - 1) / how.rows);
    const long long most = triples * ((capacity + how.keys - 1) / how.keys);
    const int limit = pl.wide[i] ? kWideCtas : kNarrowCtas;
    how.ctas = static_cast<int>(most < limit ? most : limit);
    how.share0 = pl.floats;
    pl.floats += (2LL * limit + (prefix ? triples : 0)) * how.rows * (head_dim + 2);
  }
  return pl;
}

template <int D, bool BF16>
cudaError_t launch_narrow(const CacheAttnParams& p, const CacheLaunch& how, cudaStream_t stream) {
  using Cfg = CacheCfg<D>;
  auto kern = omni_cache_attn_kernel<D, BF16>;
  static SmemAttrOnce attr_once[kMaxDevices];
  cudaError_t e = ensure_smem_attr(kern, Cfg::kSmem, attr_once);
  if (e != cudaSuccess) return e;
  kern<<<how.ctas, kThreads, Cfg::kSmem, stream>>>(p, how);
  return cudaGetLastError();
}

template <int D, bool BF16>
cudaError_t launch_t(const CacheAttnParams& p, cudaStream_t stream) {
  const long long per = p.G * static_cast<long long>(p.T);
  const Plan pl = make_plan(p.B, p.Hkv, per, D, p.prefix > 0, p.capacity);
  CUtensorMap tmK, tmV;
  if (pl.wide[0] || pl.wide[1]) {
    cudaError_t e = make_page_maps(p, D, BF16, &tmK, &tmV);
    if (e != cudaSuccess) return e;
  }
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && pl.of[0].own) break;
    const cudaError_t e = pl.wide[i] ? launch_cache_wide(D, BF16, tmK, tmV, p, pl.of[i], stream) : launch_narrow<D, BF16>(p, pl.of[i], stream);
    if (e != cudaSuccess) return e;
  }
  omni_cache_join_kernel<D, BF16><<<static_cast<unsigned>(p.B * static_cast<long long>(p.Hkv) * ((per + kRows - 1) / kRows)), 128, 0, stream>>>(
      p, pl.of[0], pl.of[1]);
  return cudaGetLastError();
}

}  // namespace

long long cache_attn_workspace_bytes(int B, int H, int Hkv, int T, int head_dim, bool prefix) {
  return make_plan(B, Hkv, static_cast<long long>(H / Hkv) * T, head_dim, prefix, 1 << 30).floats * 4;
}

cudaError_t launch_cache_attn(int head_dim, bool bf16, const CacheAttnParams& p, cudaStream_t stream) {
  if (head_dim == 32) return bf16 ? launch_t<32, true>(p, stream) : launch_t<32, false>(p, stream);
  if (head_dim == 64) return bf16 ? launch_t<64, true>(p, stream) : launch_t<64, false>(p, stream);
  return bf16 ? launch_t<128, true>(p, stream) : launch_t<128, false>(p, stream);
}

}  // namespace omni
