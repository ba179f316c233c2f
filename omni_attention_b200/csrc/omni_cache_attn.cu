// Attention of a few new tokens over a paged key/value cache: out = softmax(cap(q k^T * scale)) v for T query tokens of
// each sequence, H query heads sharing Hkv key/value heads, every row with its own number of visible keys.
//
// Bound: memory. Every key and value is read once and serves G * T query rows (G = H / Hkv), 2 * G * T operations per
// byte: with 16 rows that is a twentieth of what the card computes in the time of the read. So the query rows of a
// key/value head go through the tensor cores together, as one tile of 8 or 16 rows (mma.sync: 16 rows would fill an eighth of
// a tcgen05 tile), and all that matters is that enough reads are in flight on every SM. (More rows: omni_cache_wide.cu.)
// Measured, 8 key/value heads of 128, bf16: 2 sequences of 131 072 tokens 159 us = 6.8 TB/s; 16 of up to 8 192 61-65 us by card = 5.5-5.9 TB/s,
// 7 us of it before the first and after the last tile; 16 heads of 64, one sequence of 513 tokens 7.7 us, all of it latency.
//
// Split: the keys of all (sequence, key/value head, row tile) triples, in tiles of kTileKeys, form one line of units that is
// cut among the CTAs; lengths are read on the device, so the cut is even however ragged the batch is, and the launch does not
// depend on them (it can be captured once and replayed as the cache grows). A CTA's piece may be a part of a triple: then its
// rows' (maximum, sum, O) go to the workspace and omni_cache_join_kernel puts the shares together, in the order of the keys.
// A triple inside one piece is written out directly.
//
// A CTA (one per SM): one warp brings in the tiles of K and V, page by page with TMA, through a ring of 160 to 192 KB, running
// ahead over the ends of triples, so that the reads do not pause where a sequence ends; another the queries (cp.async) and
// what is known of the rows. Eight warps compute, each on its own 16 keys of a tile with its own running maximum, sum and O
// (no barrier between them until the end of a piece, where their shares are joined through shared memory, half of the
// columns at a time). P goes into the product as a 16-bit value plus the 16-bit rest (two products; the tensor cores have the
// room), so the only rounding that shows is that of the result. Every wait on a barrier is bounded, as in the forward kernels.
#include "omni_cache_line.cuh"
#include "omni_launch.h"

namespace omni {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32 + 64;

template <int D>
struct CacheCfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kChunks = D / 64;
  static constexpr int kSlots = D == 128 ? 3 : 5;                            // pairs of K and V tiles
  static constexpr int kRound = D / 2;                                       // columns of a round of the join, 8 rows
  static constexpr int kJoin = kWarps * 8 * (kRound + 8) * 4;                // (16 rows: half of the columns)
  static constexpr int kQ = kNarrowRows * D * 2;                             // queries of a triple
  static constexpr int kSmem = kSlots * 2 * kTile + kJoin + 2 * kQ + 2560;       // + barriers, descriptions
};

// What the computing warps are told of a piece.
struct PieceInfo {
  int n, key0, rows, lim_max;   // tiles of keys (-1: no more pieces), first key, rows, most keys that a row sees
  int table_of, hk;             // whose page table, which key/value head
  long long share;
  int lim[kNarrowRows];         // keys that a row sees
  int out[kNarrowRows];         // where it is written
};

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

// Transposes an 8 x 8 matrix of 16-bit values, two of a row to a thread.
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Arrives on `bar` (one of the arrivals it was initialised for) when this thread's cp.asyncs have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Byte offset of 16-byte chunk c of row r in [64 columns][rows][128 bytes] with the 128-byte swizzle; `pitch` = rows * 128.
__device__ __forceinline__ uint32_t swizzled(int r, int c, int pitch) {
  return static_cast<uint32_t>((c >> 3) * pitch + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// What the infinite and NaN values of column `col` in keys key0 .. key1 add up to, 0 without any: the result of a row that sees
// these keys, whatever the products made of them. Everything from memory.
template <bool BF16>
__device__ __noinline__ float not_finite_sum(const CacheAttnParams& p, int table_of, int hk, int key0, int key1, int d, int col) {
  const int in_page = (1 << p.page_shift) - 1;
  const int* table = p.page_table + table_of * p.table_stride;
  float sum = 0.f;
  for (int key = key0; key < key1; key += 16) {   // 16 keys from a multiple of 16 on are in one page
    const int page = __ldg(table + (key >> p.page_shift));
    if (page < 0 || page >= p.num_pages) continue;
    const uint16_t* v = static_cast<const uint16_t*>(p.v_pages) +
                        (((static_cast<long long>(page) * p.Hkv + hk) << p.page_shift) + (key & in_page)) * d + col;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t raw = __ldg(v + i * d);
      if ((raw & kExponent<BF16>) == kExponent<BF16> && key + i < key1) sum += unpack16<BF16>(raw).x;
    }
  }
  return sum;
}

// Barrier of the eight computing warps.
__device__ __forceinline__ void compute_sync() { named_barrier_sync(1, kWarps * 32); }

// The same, and whether `ok` holds in all of them.
__device__ __forceinline__ bool compute_vote(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.and.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok)), "n"(kWarps * 32)
      : "memory");
  return all != 0;
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
omni_cache_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CacheAttnParams p,
                       const __grid_constant__ CacheLaunch how, int d_real) {
  using Cfg = CacheCfg<D>;
  constexpr int KS = D / 16;        // steps of K Q^T, and 16-column tiles of O
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(1024) uint8_t smem[];   // what the 128-byte swizzle wants
  if ((smem_u32(smem) & 1023u) != 0) {
    if (p.status != nullptr && threadIdx.x == 0) atomicExch(p.status, kStatusWaitTimeout | (69 << 8));
    return;
  }
  const uint32_t sRing = smem_u32(smem), sQ = sRing + Cfg::kSlots * 2 * Cfg::kTile;
  float* s_join = reinterpret_cast<float*>(smem + Cfg::kSlots * 2 * Cfg::kTile + 2 * Cfg::kQ);
  uint8_t* rest = smem + Cfg::kSlots * 2 * Cfg::kTile + 2 * Cfg::kQ + Cfg::kJoin;
  uint64_t* bars = reinterpret_cast<uint64_t*>(rest);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * Cfg::kSlots;
  const uint32_t bar_q = bar_empty + 8 * Cfg::kSlots;      // [2] a piece's description and queries are there
  const uint32_t bar_free = bar_q + 16;                    // [2] and not needed any more
  volatile int* taken_out = reinterpret_cast<volatile int*>(rest + 240);   // [2] of a piece's V, something that is not finite
  volatile int* abort_flag = reinterpret_cast<volatile int*>(rest + 248);
  uint32_t(*s_valid)[4] = reinterpret_cast<uint32_t(*)[4]>(rest + 256);   // [kSlots]
  PieceInfo* info = reinterpret_cast<PieceInfo*>(rest + 512);             // [2]
  float* s_m = reinterpret_cast<float*>(rest + 1024);                     // [8][16]
  float* s_l = s_m + kWarps * kNarrowRows;                                // [8][16]

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kSlots; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q + 8 * i, 64);
      mbar_init(bar_free + 8 * i, kWarps);
    }
    *abort_flag = 0;
    taken_out[0] = taken_out[1] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (!how.late_wait) grid_wait();   // lengths, queries and pages may be the predecessor's work
  grid_go();
  __syncthreads();
  const long long limit = p.wait_cycles;
  const Ring<Cfg::kTile, Cfg::kChunks, Cfg::kSlots, true> ring{sRing, bar_full, bar_empty, s_valid, abort_flag};
  RingState st;

  if (warp >= kWarps) {
    Walk walk(p, how);
    Piece pc;
    if (warp == kWarps) {
      // =========================== K and V ========================================================
      while (st.alive && walk.next(p, pc)) ring.stream(p, &tmK, &tmV, pc, pc.tile1, st, 61);
    }
    // =========================== queries and what is known of the rows ============================
    for (int piece = 0; warp > kWarps; ++piece) {
      const int buf = piece & 1;
      if (piece >= 2) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait_lim(bar_free + 8 * buf, ((piece >> 1) - 1) & 1, abort_flag, p.status, 60, limit);
        if (!__shfl_sync(0xFFFFFFFFu, ok, 0)) break;
      }
      PieceInfo& to = info[buf];
      if (!walk.next(p, pc)) {
        if (lane == 0) to.n = -1;
        mbar_arrive(bar_q + 8 * buf);
        mbar_arrive(bar_q + 8 * buf);
        break;
      }
      // lane = row
      const int row = pc.rt * ROWS + lane;
      int lim = 0;
      const uint16_t* src = nullptr;
      if (lane < ROWS && row < pc.rows) {
        const RowId id = row_of(p, pc.prefix, pc.seg, row);
        lim = min(limit_of(p, id.b, id.t), pc.total);
        if (lim > 0) {   // a row that sees nothing may hold anything, and moves no other row's maximum
          src = static_cast<const uint16_t*>(p.q) + id.b * p.qs_b + (static_cast<long long>(pc.hk) * p.G + id.g) * p.qs_h + id.t * p.qs_t;
        }
        to.out[lane] = static_cast<int>(out_row(p, id, pc.hk));
      }
      constexpr int CH = D / 8;
#pragma unroll 1   // code that runs once comes at about 7 cycles an instruction
      for (int i = 0; i < ROWS * CH / 32; ++i) {
        const int item = lane + 32 * i, r = item / CH, c = item % CH;
        const uint16_t* from = reinterpret_cast<const uint16_t*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(src), r));
        const bool ok = from != nullptr && c * 8 < d_real;
        cp_async16(sQ + buf * Cfg::kQ + swizzled(r, c, ROWS * 128), ok ? static_cast<const void*>(from + c * 8) : p.q, ok);
      }
      cp_async_arrive(bar_q + 8 * buf);
      const int lim_max = __reduce_max_sync(0xFFFFFFFFu, lim);
      if (lane < ROWS) to.lim[lane] = lim;
      if (lane == 0) {
        to.n = pc.tile1 - pc.tile0;
        to.key0 = pc.key0 + pc.tile0 * kTileKeys;
        to.rows = min(ROWS, pc.rows - pc.rt * ROWS);
        to.lim_max = lim_max;
        to.table_of = pc.table_of;
        to.hk = pc.hk;
        to.share = pc.share;
      }
      mbar_arrive(bar_q + 8 * buf);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // =========================== computation ======================================================
    // S^T = K Q^T (16 keys x 8 rows a warp and product), O^T += V^T P^T (16 columns x 8 rows): the keys and columns fill the
    // products' 16 rows, the query rows, which are few, their 8 columns. On this card a product of this kind takes about 16
    // cycles of a quarter of an SM, and with the query rows as the 16 there were twice as many: 1 550 cycles a tile
    // against 2 750 that the card's memory needs for it.
    const int quad = lane >> 2, pos = lane & 3;
    const float scale_log2 = p.scale * 1.4426950408889634f;
    const float cap_in = p.softcap > 0.f ? p.scale / p.softcap : 0.f, cap_out = p.softcap * 1.4426950408889634f;
    uint32_t fill = 0;
    for (int piece = 0;; ++piece) {
      const int buf = piece & 1;
      bool alive = true;
      if (lane == 0) alive = mbar_wait_lim(bar_q + 8 * buf, (piece >> 1) & 1, abort_flag, p.status, 62, limit);
      alive = __shfl_sync(0xFFFFFFFFu, alive, 0);
      if (!compute_vote(alive)) break;   // all warps leave together: none waits for another at a barrier
      const PieceInfo& in = info[buf];
      const int n = in.n;
      if (n < 0) break;
      const int key0 = in.key0 + warp * 16, rows = in.rows, lim_max = in.lim_max;
      // this thread's rows: 8 j + 2 pos + {0, 1}
      int lim[2 * NT], lim_min = 0x7FFFFFFF;
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j) {
        const int r = 8 * (j >> 1) + 2 * pos + (j & 1);
        lim[j] = in.lim[r];
        if (r < rows && lim[j] > 0) lim_min = min(lim_min, lim[j]);   // rows that see nothing are zeroed at the end
      }
      lim_min = __reduce_min_sync(0xFFFFFFFFu, lim_min);
      uint32_t qf[KS][2 * NT];   // Q^T, two steps to an ldmatrix for 8 rows, one for 16
#pragma unroll
      for (int k = 0; k < KS; k += 2 / NT) {
        uint32_t b[4];
        if constexpr (NT == 1) {
          ldmatrix4(sQ + buf * Cfg::kQ + swizzled(lane & 7, 2 * k + (lane >> 3), ROWS * 128), b);
          qf[k][0] = b[0];
          qf[k][1] = b[1];
          qf[k + 1][0] = b[2];
          qf[k + 1][1] = b[3];
        } else {
          ldmatrix4(sQ + buf * Cfg::kQ + swizzled((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1), ROWS * 128), b);
#pragma unroll
          for (int i = 0; i < 4; ++i) qf[k][i] = b[i];
        }
      }
      float o_acc[KS][NT][4];
#pragma unroll
      for (int i = 0; i < KS; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) o_acc[i][j][0] = o_acc[i][j][1] = o_acc[i][j][2] = o_acc[i][j][3] = 0.f;
      }
      float m[2 * NT], l[2 * NT];
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.f;
      }

      for (int t = 0; t < n; ++t, ++fill) {
        const uint32_t slot = fill % Cfg::kSlots;
        const int key = key0 + t * kTileKeys;
        if (lane == 0) mbar_wait_lim(bar_full + 8 * slot, (fill / Cfg::kSlots) & 1, abort_flag, p.status, 63, limit);
        __syncwarp();
        const bool there = *const_cast<volatile uint32_t*>(&s_valid[slot][warp >> 1]) >> (16 * (warp & 1)) & 1u;   // a page has 16 keys at least
        if (key < lim_max && there) {   // else: nothing for this warp in the tile
          const uint32_t sk = sRing + slot * (2 * Cfg::kTile), sv = sk + Cfg::kTile;
          float s[NT][4], s2[NT][4];   // [rows 8 j ..]: keys quad (0, 1) and quad + 8 (2, 3), rows 2 pos and 2 pos + 1
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
            s2[j][0] = s2[j][1] = s2[j][2] = s2[j][3] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t a[4];
            ldmatrix4(sk + swizzled(warp * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * k + (lane >> 4), 128 * 128), a);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma16816<BF16>(k & 1 ? s2[j] : s[j], a, qf[k][2 * j], qf[k][2 * j + 1]);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] += s2[j][e];
          }
          if (key + 16 > lim_max) {   // V that no row sees may be anything: 0 * NaN
#pragma unroll
            for (int i = 0; i < 16 * Cfg::kChunks * 8 / 32; ++i) {
              const int item = lane + 32 * i, r = item & 15, c = item >> 4;
              if (key + r >= lim_max) {
                *reinterpret_cast<uint4*>(smem + slot * (2 * Cfg::kTile) + Cfg::kTile + swizzled(warp * 16 + r, c, 128 * 128)) = make_uint4(0u, 0u, 0u, 0u);
              }
            }
            fence_async_smem();   // the ring's next copy goes over it
            __syncwarp();
          }
          if (p.softcap > 0.f) {
            float big = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                s[j][e] *= cap_in;
                big = fmaxf(big, fabsf(s[j][e]));
              }
            }
            const bool small = !__any_sync(0xFFFFFFFFu, big > kTanhPolyLimit);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const float2 y = make_float2(s[j][e], s[j][e + 1]);
                float2 t = tanh_small2(y);
                if (!small) {   // which form a score takes depends on nothing but itself: keys that are not there are among these
                  t.x = fabsf(y.x) <= kTanhPolyLimit ? t.x : tanh_exact(y.x);
                  t.y = fabsf(y.y) <= kTanhPolyLimit ? t.y : tanh_exact(y.y);
                }
                s[j][e] = t.x * cap_out;
                s[j][e + 1] = t.y * cap_out;
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int e = 0; e < 4; ++e) s[j][e] *= scale_log2;
            }
          }
          if (key + 16 > lim_min) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (key + quad + 4 * (e & 2) >= lim[2 * j + (e & 1)]) s[j][e] = -INFINITY;
              }
            }
          }
          // Running maximum: looked for and moved only when a score is above it by more than 8 (p <= 2^8 in 32 bits and in
          // either 16-bit type).
          bool move = false;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) move |= s[j][e] > m[2 * j + (e & 1)] + 8.f;
          }
          if (__any_sync(0xFFFFFFFFu, move)) {
#pragma unroll
            for (int j = 0; j < 2 * NT; ++j) {
              float to = fmaxf(m[j], fmaxf(s[j >> 1][j & 1], s[j >> 1][2 + (j & 1)]));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) to = fmaxf(to, __shfl_xor_sync(0xFFFFFFFFu, to, o));
              const float f = m[j] == -INFINITY ? 0.f : ex2_approx(m[j] - to);
              m[j] = to;
              l[j] *= f;
#pragma unroll
              for (int d = 0; d < KS; ++d) {
                o_acc[d][j >> 1][j & 1] *= f;
                o_acc[d][j >> 1][2 + (j & 1)] *= f;
              }
            }
          }
          uint32_t hi[NT][2], lo[NT][2];   // P^T: keys 0-7 and 8-15 of the warp's, turned so that a thread has two keys of a row
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const float at0 = m[2 * j] == -INFINITY ? 0.f : m[2 * j], at1 = m[2 * j + 1] == -INFINITY ? 0.f : m[2 * j + 1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float a = ex2_approx(s[j][2 * h] - at0), b = ex2_approx(s[j][2 * h + 1] - at1);
              s[j][2 * h] = a;
              s[j][2 * h + 1] = b;
              l[2 * j] += a;
              l[2 * j + 1] += b;
              const uint32_t w = pack16<BF16>(a, b);
              const float2 v = unpack16<BF16>(w);
              hi[j][h] = movmatrix(w);
              lo[j][h] = movmatrix(pack16<BF16>(a - v.x, b - v.y));
            }
          }
          if (key + 16 > lim_min && lim_min < lim_max) {
            // An infinite or NaN value must not reach the rows that do not see its key (0 * NaN): it is taken out of the product
            // and added at the end of the piece. Looked for only where rows of the tile see different numbers of keys.
            bool bad = false;
#pragma unroll 1
            for (int c = lane >> 4; c < Cfg::kChunks * 8; c += 2) {
              uint4* v = reinterpret_cast<uint4*>(smem + slot * (2 * Cfg::kTile) + Cfg::kTile + swizzled(warp * 16 + (lane & 15), c, 128 * 128));
              if (not_finite<BF16>(*v)) {
                *v = finite_part<BF16>(*v);
                bad = true;
              }
            }
            if (__any_sync(0xFFFFFFFFu, bad)) {
              if (lane == 0) taken_out[buf] = 1;
              fence_async_smem();
              __syncwarp();
            }
          }
#pragma unroll
          for (int d = 0; d < KS; ++d) {
            uint32_t a[4];   // V^T: 16 columns x 16 keys
            ldmatrix4_trans(sv + swizzled(warp * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1), 128 * 128), a);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma16816<BF16>(o_acc[d][j], a, hi[j][0], hi[j][1]);
              mma16816<BF16>(o_acc[d][j], a, lo[j][0], lo[j][1]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + 8 * slot);
      }

      // ---- the warps' shares of the piece, joined: kRound columns at a time ----
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xFFFFFFFFu, l[j], o);
        if (quad == 0) {
          const int r = 8 * (j >> 1) + 2 * pos + (j & 1);
          s_m[warp * kNarrowRows + r] = m[j];
          s_l[warp * kNarrowRows + r] = l[j];
        }
      }
      const long long share = in.share;
      constexpr int C = Cfg::kRound / NT, TR = 256 / ROWS, V = C / TR;   // columns of a round, threads of a row, columns of a thread
      constexpr int P = C + 4;                                           // pitch of a row
      const int r = threadIdx.x / TR;                                    // the row this thread finishes
      const long long at_row = in.out[r];
      const bool sees = in.lim[r] > 0;
      float f[kWarps], top = -INFINITY, sum = 0.f;
      bool odd = false;   // values were taken out, or an element is not finite though its row's sum is
#pragma unroll
      for (int round = 0; round < D / C; ++round) {
        if (round * C >= d_real) break;
#pragma unroll
        for (int d = 0; d < C / 16; ++d) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int rr = 8 * j + 2 * pos + (e & 1);
              if (rr < rows) s_join[(warp * ROWS + rr) * P + 16 * d + quad + 4 * (e & 2)] = o_acc[round * (C / 16) + d][j][e];
            }
          }
        }
        compute_sync();
        if (round == 0) {
          odd = taken_out[buf] != 0;
          if (threadIdx.x == 0) taken_out[buf ^ 1] = 0;   // the piece before is done with it, the next one has not begun
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * kNarrowRows + r]);
          const float at = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            f[w] = ex2_approx(s_m[w * kNarrowRows + r] - at);
            sum += f[w] * s_l[w * kNarrowRows + r];
          }
          if (!sees) {
            top = -INFINITY;
            sum = 0.f;
          }
        }
        const int in_round = (threadIdx.x % TR) * V, col = round * C + in_round;
        if (r < rows && col < d_real) {
          float acc[V];
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += f[w] * s_join[(w * ROWS + r) * P + in_round + i];
          }
          float z = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) z = fmaf(acc[i], 0.f, z);
          odd |= z != z && sum == sum;
          if (share >= 0) {
            float* to = share_at(p, how, share, d_real) + r * d_real + col;
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = sees ? acc[i] : 0.f;
          } else {
            const bool any = !(sum == 0.f);   // NaN shows
            const float inv = 1.f / sum;
            uint16_t* to = static_cast<uint16_t*>(p.out) + at_row * d_real + col;
            if constexpr (V == 2) {
              *reinterpret_cast<uint32_t*>(to) = any ? pack16<BF16>(acc[0] * inv, acc[1] * inv) : 0u;
            } else {
              *to = any ? static_cast<uint16_t>(pack16<BF16>(acc[0] * inv, 0.f)) : static_cast<uint16_t>(0);
            }
          }
        }
        compute_sync();   // the next round goes over what was read
      }
      // Of values that are not finite some were taken out of the products, the others came in as p * inf with p in two parts, of
      // which the second may be zero or negative: an element whose row sees such values in its column is what they add up to.
      if (odd && r < rows) {
#pragma unroll 1
        for (int e = 0; e < d_real / TR; ++e) {
          const int col = e / V * C + threadIdx.x % TR * V + e % V;   // what this thread wrote
          const float x = not_finite_sum<BF16>(p, in.table_of, in.hk, in.key0, min(in.lim[r], in.key0 + n * kTileKeys), d_real, col);
          if (x == 0.f) continue;
          if (share >= 0) {
            share_at(p, how, share, d_real)[r * d_real + col] = x;
          } else {
            static_cast<uint16_t*>(p.out)[at_row * d_real + col] = static_cast<uint16_t>(pack16<BF16>(x, 0.f));
          }
        }
      }
      if (r < rows && threadIdx.x % TR == 0) {
        if (share >= 0) {
          float* to = share_at(p, how, share, d_real) + how.rows * d_real;
          to[r] = top;
          to[how.rows + r] = sum;
        } else if (p.lse != nullptr) {
          p.lse[at_row] = !(sum == 0.f) ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_free + 8 * buf);
    }
  }
  __syncthreads();
  if (*abort_flag && warp == kWarps) ring.drain(st);
  if (how.late_wait) grid_wait();
}

// Joins the shares of the rows that no single span covered, a warp per row. `pre` is the launch that had the prefix (if
// there is one), `own` the one that had the sequences' own keys; they may be the same launch.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) omni_cache_join_kernel(const __grid_constant__ CacheAttnParams p, const __grid_constant__ CacheLaunch pre,
                                                              const __grid_constant__ CacheLaunch own) {
  constexpr int V = D / 32;   // columns of a lane
  constexpr int AHEAD = 4;    // shares whose O is read before their maxima are known
  const int lane = threadIdx.x & 31;
  const Line lo = make_line(p, own);
  if (p.prefix == 0 && lo.uncut) {   // everything was written by the one CTA that had it
    grid_wait();
    return;
  }
  const Line lp = p.prefix > 0 ? make_line(p, pre) : lo;
  if (p.prefix > 0 && p.status != nullptr) {   // is the prefix in the same pages?
    for (int seq = blockIdx.x; seq < p.B; seq += gridDim.x) {
      const int pages = (min(p.prefix, total_of(p, seq)) + (1 << p.page_shift) - 1) >> p.page_shift;
      bool same = true;
      for (int i = threadIdx.x; i < pages; i += blockDim.x) {
        same &= __ldg(p.page_table + seq * p.table_stride + i) == __ldg(p.page_table + lp.prefix_seq * p.table_stride + i);
      }
      if (!same) atomicCAS(p.status, 0, kStatusBadIndex);
    }
  }
  const int rows = p.G * p.T;
  const unsigned per_seq = static_cast<unsigned>(p.Hkv) * rows, all = per_seq * p.B;   // below 2^31
  bool waited = false;
  for (unsigned item = blockIdx.x * 8 + (threadIdx.x >> 5); item < all; item += gridDim.x * 8) {
    const int seq = p.B == 1 ? 0 : static_cast<int>(item / per_seq);
    const int in_seq = static_cast<int>(item - seq * per_seq), hk = in_seq / rows, row = in_seq - hk * rows;
    unsigned before = 0;
    if (!lo.even) {
      for (int b = lane; b < seq; b += 32) before += lo.own_units(p, b);
      before = __reduce_add_sync(0xFFFFFFFFu, before);
    }
    const unsigned units = lo.units_between(p.prefix, total_of(p, seq));
    const unsigned triple = static_cast<unsigned>(hk) * lo.rt_own + row / own.rows;
    unsigned c0, n1;
    if (lo.even) {
      c0 = lo.first_cta(p, seq, triple);
      n1 = lo.parts(units);
    } else {
      const unsigned first = lo.prefix_units + before + triple * units;
      c0 = first / lo.span;
      n1 = (first + units - 1) / lo.span - c0 + 1;
    }
    if (p.prefix == 0 && n1 == 1) continue;   // written already
    // the row's shares: n0 of the prefix, then n1 of its own keys
    unsigned d0 = 0, n0 = 0, pt = 0;
    int in0 = 0;
    if (p.prefix > 0) {
      const unsigned gr = static_cast<unsigned>(seq) * rows + row;   // the row in the prefix segment
      pt = static_cast<unsigned>(hk) * lp.rt_prefix + gr / pre.rows;
      in0 = static_cast<int>(gr % pre.rows);
      const unsigned pu = lp.units_between(0, lp.prefix_end), f = pt * pu;
      d0 = lp.even ? lp.first_cta(p, -1, pt) : f / lp.span;
      n0 = lp.even ? lp.parts(pu) : (f + pu - 1) / lp.span - d0 + 1;
    }
    const long long whole0 = 2LL * pre.ctas + pt;
    const long long whole1 = 2LL * own.ctas + static_cast<long long>(p.Hkv) * (lo.rt_prefix + static_cast<long long>(seq) * lo.rt_own) + triple;
    if (!waited) grid_wait();
    waited = true;

    float top = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (unsigned j0 = 0; j0 < n0 + n1; j0 += 32) {
      // lane = share: maximum, sum and place of up to 32 of them at once
      const unsigned j = j0 + lane;
      const int n = min(32, static_cast<int>(n0 + n1 - j0));
      float m2 = -INFINITY, l2 = 0.f;
      unsigned long long at = 0;
      if (j < n0 + n1) {
        const bool first_part = j < n0;
        const unsigned i = first_part ? j : j - n0;
        const int tile_rows = first_part ? pre.rows : own.rows;
        const long long share = (first_part ? n0 : n1) == 1 ? (first_part ? whole0 : whole1) : 2LL * ((first_part ? d0 : c0) + i) + (i == 0 ? 1 : 0);
        const int in = first_part ? in0 : row % own.rows;
        const float* from = p.partial + (first_part ? pre.share0 : own.share0) + share * (tile_rows * (D + 2));
        m2 = __ldcg(from + tile_rows * D + in);
        l2 = __ldcg(from + tile_rows * D + tile_rows + in);
        at = reinterpret_cast<unsigned long long>(from + in * D);
      }
      auto read = [&](int i, float (&v)[V]) {
        const float* from = reinterpret_cast<const float*>(__shfl_sync(0xFFFFFFFFu, at, i)) + lane * V;
        if constexpr (V == 4) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(from));
          v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        } else if constexpr (V == 2) {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(from));
          v[0] = x.x, v[1] = x.y;
        } else {
          v[0] = __ldcg(from);
        }
      };
      float early[AHEAD][V];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (i < n) read(i, early[i]);
      }
      float to = fmaxf(top, m2);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xFFFFFFFFu, to, o));
      const float ref = to == -INFINITY ? 0.f : to;
      // A share's weight is not 0 while it has keys: 0 * inf. (2^-126 of the largest shows in nothing else.)
      constexpr float kLeast = 1.17549435e-38f;
      const float f1 = top == -INFINITY ? 0.f : fmaxf(ex2_approx(top - ref), kLeast), f2 = m2 == -INFINITY ? 0.f : fmaxf(ex2_approx(m2 - ref), kLeast);
      float part = l2 * f2;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xFFFFFFFFu, part, o);
      sum = sum * f1 + part;
      top = to;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f1;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (i < n) {
          const float f = __shfl_sync(0xFFFFFFFFu, f2, i);
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += f * early[i][k];
        }
      }
#pragma unroll 4
      for (int i = AHEAD; i < n; ++i) {
        float v[V];
        read(i, v);
        const float f = __shfl_sync(0xFFFFFFFFu, f2, i);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += f * v[k];
      }
    }
    const long long at_row = out_row(p, row_of(p, false, seq, row), hk);
    const bool any = !(sum == 0.f);   // NaN shows
    const float inv = 1.f / sum;
    uint16_t* to = static_cast<uint16_t*>(p.out) + at_row * D + lane * V;
    if constexpr (V == 4) {
      *reinterpret_cast<uint2*>(to) = any ? make_uint2(pack16<BF16>(acc[0] * inv, acc[1] * inv), pack16<BF16>(acc[2] * inv, acc[3] * inv)) : make_uint2(0u, 0u);
    } else if constexpr (V == 2) {
      *reinterpret_cast<uint32_t*>(to) = any ? pack16<BF16>(acc[0] * inv, acc[1] * inv) : 0u;
    } else {
      *to = any ? static_cast<uint16_t>(pack16<BF16>(acc[0] * inv, 0.f)) : static_cast<uint16_t>(0);
    }
    if (p.lse != nullptr && lane == 0) p.lse[at_row] = any ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
  }
  if (!waited) grid_wait();
}

// The launches of a call: one over everything, or one over the prefix and one over the sequences' own keys where only one
// of the two has more than 16 rows to a key/value head (the narrow kernel would read its keys once for every 16 rows).
// 8 sequences of 4K keys, 8 key/value heads of 128: 16 rows 29.7 us here and 34.4 on 128-row tiles, 32 rows 38.4 and 34.4.
struct Plan {
  CacheLaunch of[2];   // the prefix's, the sequences'; equal if one launch has both
  bool join;
  long long floats, units;
};

Plan make_plan(int B, int Hkv, long long per, int head_dim, int prefix, long long capacity) {
  Plan pl{};
  const long long rows[2] = {B * per, per};
  auto tile = [](long long n) { return n > kNarrowRows ? kWideRows : n > 8 ? 16 : 8; };
  const bool one = prefix == 0 || (rows[0] > kNarrowRows) == (rows[1] > kNarrowRows);
  const long long tiles = (capacity + kTileKeys - 1) / kTileKeys;
  for (int i = 0; i < 2; ++i) {
    CacheLaunch& how = pl.of[i];
    if (i == 1 && one) {
      how = pl.of[0];
      break;
    }
    how.prefix = prefix > 0 && (one || i == 0);
    how.own = one || i == 1;
    how.rows = tile(rows[how.prefix ? 0 : 1]);
    how.uncut = prefix > 0 ? kUncutTilesPrefix : kUncutTiles;
    how.late_wait = i;
    how.rt_prefix = how.prefix ? static_cast<int>((rows[0] + how.rows - 1) / how.rows) : 0;
    how.rt_own = static_cast<int>((rows[1] + how.rows - 1) / how.rows);
    const long long triples = Hkv * (how.rt_prefix + (how.own ? static_cast<long long>(B) * how.rt_own : 0)), most = triples * tiles;
    pl.units += most;
    how.ctas = static_cast<int>(most < kCacheCtas ? most : kCacheCtas);
    how.per_cta = static_cast<unsigned>((triples + how.ctas - 1) / how.ctas);
    how.even = static_cast<unsigned>(how.ctas / triples);
    how.share0 = pl.floats;
    pl.floats += (2LL * kCacheCtas + (prefix > 0 ? triples : 0)) * how.rows * (head_dim + 2);
    pl.join = prefix > 0 || how.per_cta * tiles > 1 + kUncutTiles;   // else it is never cut
  }
  return pl;
}

template <int D, int NT, bool BF16>
cudaError_t launch_narrow(const CUtensorMap& tmK, const CUtensorMap& tmV, const CacheAttnParams& p, const CacheLaunch& how, int d_real,
                          cudaStream_t stream) {
  using Cfg = CacheCfg<D>;
  auto kern = omni_cache_attn_kernel<D, NT, BF16>;
  static SmemAttrOnce attr_once[kMaxDevices];
  const cudaError_t e = ensure_smem_attr(kern, Cfg::kSmem, attr_once);
  if (e != cudaSuccess) return e;
  return launch_chained(kern, how.ctas, kThreads, Cfg::kSmem, stream, tmK, tmV, p, how, d_real);
}

template <int D, bool BF16>
cudaError_t launch_t(const CacheAttnParams& p, cudaStream_t stream) {
  constexpr int C = D == 128 ? 128 : 64;   // head_dim 32 is computed as 64: the TMA unit fills the missing columns with zeros
  const Plan pl = make_plan(p.B, p.Hkv, p.G * static_cast<long long>(p.T), D, p.prefix, p.capacity);
  CUtensorMap tmK, tmV;
  cudaError_t e = make_page_maps(p, D, BF16, &tmK, &tmV);
  for (int i = 0; e == cudaSuccess && i < 2; ++i) {
    const CacheLaunch& how = pl.of[i];
    if (i == 1 && pl.of[0].own) break;
    e = how.rows == kWideRows ? launch_cache_wide(D, BF16, tmK, tmV, p, how, stream)
        : how.rows == 16      ? launch_narrow<C, 2, BF16>(tmK, tmV, p, how, D, stream)
                              : launch_narrow<C, 1, BF16>(tmK, tmV, p, how, D, stream);
  }
  if (e != cudaSuccess || !pl.join) return e;
  const long long ctas = (static_cast<long long>(p.B) * p.H * p.T + 7) / 8;
  return launch_chained(omni_cache_join_kernel<D, BF16>, static_cast<unsigned>(ctas < 4 * kCacheCtas ? ctas : 4 * kCacheCtas), 256, 0, stream, p, pl.of[0], pl.of[1]);
}

}  // namespace

long long cache_attn_workspace_bytes(int B, int H, int Hkv, int T, int head_dim, bool prefix, long long capacity) {
  const Plan pl = make_plan(B, Hkv, static_cast<long long>(H / Hkv) * T, head_dim, prefix ? 1 : 0, capacity);
  return pl.join ? pl.floats * 4 : 0;
}

bool cache_attn_fits(const CacheAttnParams& p) {
  return make_plan(p.B, p.Hkv, p.G * static_cast<long long>(p.T), 128, p.prefix, p.capacity).units < (1LL << 31);
}

cudaError_t launch_cache_attn(int head_dim, bool bf16, const CacheAttnParams& p, cudaStream_t stream) {
  if (head_dim == 32) return bf16 ? launch_t<32, true>(p, stream) : launch_t<32, false>(p, stream);
  if (head_dim == 64) return bf16 ? launch_t<64, true>(p, stream) : launch_t<64, false>(p, stream);
  return bf16 ? launch_t<128, true>(p, stream) : launch_t<128, false>(p, stream);
}

}  // namespace omni
