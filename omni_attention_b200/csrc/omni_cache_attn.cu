// Attention of a few new tokens over a paged key/value cache: out = softmax(cap(q k^T * scale)) v for T query tokens of
// each sequence, H query heads sharing Hkv key/value heads, every row with its own number of visible keys.
//
// Bound: memory. Every key and value is read once and serves G * T query rows (G = H / Hkv), 2 * G * T operations per
// byte: with 16 rows that is a twentieth of what the card computes in the time of the read. So the query rows of a
// key/value head go through the tensor cores together as one 16-row tile (mma.sync: 16 rows would fill an eighth of a
// tcgen05 tile), and all that matters is that enough reads are in flight on every SM. (More rows: omni_cache_wide.cu.)
//
// Split: the keys of all (sequence, key/value head, 16-row tile) triples, in tiles of kTileKeys, form one line of units
// that is cut into equal spans, one per CTA; lengths are read on the device, so the cut is even however ragged the batch
// is, and the launch does not depend on them (it can be captured once and replayed as the cache grows). A span may end
// inside a triple: then its rows' (maximum, sum, O) go to the workspace and omni_cache_join_kernel puts the shares
// together, in the order of the keys. A triple inside one span is written out directly.
//
// A CTA (one per SM): one warp brings in the queries (cp.async) and, page by page with TMA, the tiles of K and V through a
// ring of 160 to 192 KB, running ahead over the ends of triples, so that the reads do not pause where a sequence ends. Eight
// warps compute, each on its own 16 keys of a tile with its own running maximum, sum and O (no barrier between them until
// the end of a triple, where their shares are joined through shared memory, a quarter of the columns at a time). The maximum
// moves only when it would grow by more than 2^8 (scores are in the log2 domain), P goes into the product as a 16-bit value
// plus the 16-bit rest (two products; the tensor cores have the room), so the only rounding that shows is that of the result.
// Every wait on a barrier is bounded, as in the forward kernels.
#include "omni_cache_line.cuh"
#include "omni_launch.h"

namespace omni {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kRows = kNarrowRows;

template <int D>
struct CacheCfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kChunks = D / 64;
  static constexpr int kSlots = D == 128 ? 6 : 10;
  static constexpr int kRound = D / 4;                                       // columns of a round of the join
  static constexpr int kJoin = kWarps * kRows * (kRound + 4) * 4;
  static constexpr int kQ = kRows * D * 2;                                   // queries of a triple
  static constexpr int kSmem = kSlots * kTile + kJoin + 2 * kQ + 2560;       // + barriers, descriptions
};

// What the loading warp tells the others of a piece.
struct PieceInfo {
  int n, key0, rows, hk;      // tiles of keys, first key, rows of the tile, -1 in n: no more pieces
  int lim_max, pad;
  long long share;
  int lim[kRows];             // keys that a row sees
  long long out[kRows];       // where it is written
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? 16 : 0;   // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives on `bar` (one of the arrivals it was initialised for) when this thread's cp.asyncs have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Byte offset of 16-byte chunk c of row r in [64 columns][rows][128 bytes] with the 128-byte swizzle; `pitch` = rows * 128.
__device__ __forceinline__ uint32_t swizzled(int r, int c, int pitch) {
  return static_cast<uint32_t>((c >> 3) * pitch + r * 128 + (((c & 7) ^ (r & 7)) << 4));
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

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
omni_cache_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CacheAttnParams p,
                       const __grid_constant__ CacheLaunch how, int d_real) {
  using Cfg = CacheCfg<D>;
  constexpr int KS = D / 16;        // steps of Q K^T
  extern __shared__ __align__(1024) uint8_t smem[];   // what the 128-byte swizzle wants
  if ((smem_u32(smem) & 1023u) != 0) {
    if (p.status != nullptr && threadIdx.x == 0) atomicExch(p.status, kStatusWaitTimeout | (69 << 8));
    return;
  }
  const uint32_t sRing = smem_u32(smem), sQ = sRing + Cfg::kSlots * Cfg::kTile;
  float* s_join = reinterpret_cast<float*>(smem + Cfg::kSlots * Cfg::kTile + 2 * Cfg::kQ);
  uint8_t* rest = smem + Cfg::kSlots * Cfg::kTile + 2 * Cfg::kQ + Cfg::kJoin;
  uint64_t* bars = reinterpret_cast<uint64_t*>(rest);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * Cfg::kSlots;
  const uint32_t bar_q = bar_empty + 8 * Cfg::kSlots;      // [2] a piece's description and queries are there
  const uint32_t bar_free = bar_q + 16;                    // [2] and not needed any more
  volatile int* abort_flag = reinterpret_cast<volatile int*>(rest + 248);
  uint32_t(*s_valid)[4] = reinterpret_cast<uint32_t(*)[4]>(rest + 256);   // [kSlots]
  PieceInfo* info = reinterpret_cast<PieceInfo*>(rest + 512);             // [2]
  float* s_m = reinterpret_cast<float*>(rest + 1024);                     // [8][16]
  float* s_l = s_m + kWarps * kRows;                                      // [8][16]

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
    mbar_fence_init();
  }
  __syncthreads();
  grid_go();
  const long long limit = p.wait_cycles;

  if (warp == kWarps) {
    // =========================== loads ============================================================
    const Ring<Cfg::kTile, Cfg::kChunks, Cfg::kSlots> ring{sRing, bar_full, bar_empty, s_valid, abort_flag};
    Walk walk(p, how);
    Piece pc;
    RingState st;
    for (int piece = 0;; ++piece) {
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
      // rows: lane = row
      const int row = pc.rt * kRows + lane;
      int lim = 0;
      const uint16_t* src = nullptr;
      long long out = 0;
      if (lane < kRows && row < pc.rows) {
        const RowId id = row_of(p, pc.prefix, pc.seg, row);
        lim = min(limit_of(p, id.b, id.t), pc.total);
        out = out_row(p, id, pc.hk);
        src = static_cast<const uint16_t*>(p.q) + id.b * p.qs_b + (static_cast<long long>(pc.hk) * p.G + id.g) * p.qs_h + id.t * p.qs_t;
      }
      const int lim_max = __reduce_max_sync(0xFFFFFFFFu, lim);
      constexpr int CH = D / 8;
#pragma unroll
      for (int i = 0; i < kRows * CH / 32; ++i) {
        const int item = lane + 32 * i, r = item / CH, c = item % CH;
        const uint16_t* from = reinterpret_cast<const uint16_t*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(src), r));
        const bool ok = from != nullptr && c * 8 < d_real;
        cp_async16(sQ + buf * Cfg::kQ + swizzled(r, c, kRows * 128), ok ? from + c * 8 : p.q, ok);
      }
      cp_async_arrive(bar_q + 8 * buf);
      // tiles of keys that no row sees are not read
      const int first = pc.key0 + pc.tile0 * kTileKeys;
      const int seen = lim_max > first ? (lim_max - first + kTileKeys - 1) / kTileKeys : 0;
      const int n = min(pc.tile1 - pc.tile0, seen);
      if (lane < kRows) {
        to.lim[lane] = lim;
        to.out[lane] = out;
      }
      if (lane == 0) {
        to.n = n;
        to.key0 = first;
        to.rows = min(kRows, pc.rows - pc.rt * kRows);
        to.lim_max = lim_max;
        to.share = pc.share;
      }
      mbar_arrive(bar_q + 8 * buf);
      ring.stream(p, &tmK, &tmV, pc, pc.tile0 + n, st, 61);
      if (!st.alive) break;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    ring.drain(st);
  } else {
    // =========================== computation ======================================================
    const int quad = lane >> 2, pos = lane & 3;
    const float scale_log2 = p.scale * 1.4426950408889634f;
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
      const int lim[2] = {in.lim[quad], in.lim[quad + 8]};
      int lim_min = min(quad < rows ? lim[0] : lim_max, quad + 8 < rows ? lim[1] : lim_max);
      lim_min = __reduce_min_sync(0xFFFFFFFFu, lim_min);
      uint32_t qf[KS][4];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        ldmatrix4(sQ + buf * Cfg::kQ + swizzled((lane & 7) + (((lane >> 3) & 1) << 3), 2 * k + (lane >> 4), kRows * 128), qf[k]);
      }
      float o_acc[D / 8][4];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o_acc[i][0] = o_acc[i][1] = o_acc[i][2] = o_acc[i][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

      for (int t = 0; t < n; ++t, fill += 2) {
        const uint32_t ks = fill % Cfg::kSlots, vs = (fill + 1) % Cfg::kSlots;
        const int key = key0 + t * kTileKeys;
        if (lane == 0) mbar_wait_lim(bar_full + 8 * ks, (fill / Cfg::kSlots) & 1, abort_flag, p.status, 63, limit);
        __syncwarp();
        float s[2][4];
        if (key < lim_max) {   // else: nothing for this warp in the tile
          const uint32_t sk = sRing + ks * Cfg::kTile;
#pragma unroll
          for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t b[4];
            ldmatrix4(sk + swizzled(warp * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1), 128 * 128), b);
            mma16816<BF16>(s[0], qf[k], b[0], b[1]);
            mma16816<BF16>(s[1], qf[k], b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_empty + 8 * ks);
          mbar_wait_lim(bar_full + 8 * vs, ((fill + 1) / Cfg::kSlots) & 1, abort_flag, p.status, 64, limit);
        }
        __syncwarp();
        const bool there = *const_cast<volatile uint32_t*>(&s_valid[vs][warp >> 1]) >> (16 * (warp & 1)) & 1u;   // a page has 16 keys at least
        if (key < lim_max && there) {
          const uint32_t sv = sRing + vs * Cfg::kTile;
          if (key + 16 > lim_max) {   // V that no row sees may be anything: 0 * NaN
#pragma unroll
            for (int i = 0; i < 16 * Cfg::kChunks * 8 / 32; ++i) {
              const int item = lane + 32 * i, r = item & 15, c = item >> 4;
              if (key + r >= lim_max) {
                *reinterpret_cast<uint4*>(smem + vs * Cfg::kTile + swizzled(warp * 16 + r, c, 128 * 128)) = make_uint4(0u, 0u, 0u, 0u);
              }
            }
            fence_async_smem();   // the ring's next copy goes over it
            __syncwarp();
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
            ldmatrix4_trans(sv + swizzled(warp * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * d + (lane >> 4), 128 * 128), b);
            mma16816<BF16>(o_acc[2 * d], hi, b[0], b[1]);
            mma16816<BF16>(o_acc[2 * d + 1], hi, b[2], b[3]);
            mma16816<BF16>(o_acc[2 * d], lo, b[0], b[1]);
            mma16816<BF16>(o_acc[2 * d + 1], lo, b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + 8 * vs);
      }

      // ---- the warps' shares of the piece, joined ----
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
        if (pos == 0) {
          s_m[warp * kRows + quad + 8 * i] = m[i];
          s_l[warp * kRows + quad + 8 * i] = l[i];
        }
      }
      const long long share = in.share;
      const int r = threadIdx.x >> 4;                // the row this thread finishes, and which columns of a round
      const long long at_row = in.out[r];
      float f[kWarps], top = -INFINITY, sum = 0.f;
      constexpr int C = Cfg::kRound, V = C / 16;     // columns of a round, of a thread
#pragma unroll
      for (int round = 0; round < 4; ++round) {
#pragma unroll
        for (int d = 0; d < C / 8; ++d) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (quad + 8 * i < rows) {
              *reinterpret_cast<float2*>(s_join + (warp * kRows + quad + 8 * i) * (C + 4) + 8 * d + 2 * pos) =
                  make_float2(o_acc[round * (C / 8) + d][2 * i], o_acc[round * (C / 8) + d][2 * i + 1]);
            }
          }
        }
        compute_sync();
        if (round == 0) {
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * kRows + r]);
          const float at = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            f[w] = ex2_approx(s_m[w * kRows + r] - at);
            sum += f[w] * s_l[w * kRows + r];
          }
        }
        const int col = round * C + (threadIdx.x & 15) * V;
        if (r < rows && col < d_real) {
          float acc[V];
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += f[w] * s_join[(w * kRows + r) * (C + 4) + (threadIdx.x & 15) * V + i];
          }
          if (share >= 0) {
            float* to = share_at(p, how, share, d_real) + r * d_real + col;
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = acc[i];
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
      if (r < rows && (threadIdx.x & 15) == 0) {
        if (share >= 0) {
          float* to = share_at(p, how, share, d_real) + kRows * d_real;
          to[r] = top;
          to[kRows + r] = sum;
        } else if (p.lse != nullptr) {
          p.lse[at_row] = !(sum == 0.f) ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_free + 8 * buf);
    }
  }
  __syncthreads();
  grid_wait();   // a launch that was allowed to start early ends after its predecessor
}

// Joins the shares of the rows that no single span covered. One CTA of 16 warps per (sequence, key/value head, 16 rows):
// with fewer rows several warps take a row's shares in turn. `pre` is the launch that had the prefix (if there is one),
// `own` the one that had the sequences' own keys; they may be the same launch.
template <int D, bool BF16>
__global__ void __launch_bounds__(512) omni_cache_join_kernel(const __grid_constant__ CacheAttnParams p, const __grid_constant__ CacheLaunch pre,
                                                              const __grid_constant__ CacheLaunch own) {
  constexpr int V = D / 32;   // columns of a lane
  __shared__ float s_acc[16][D], s_top[16], s_sum[16];
  const int rows = p.G * p.T;
  const int groups = (rows + kRows - 1) / kRows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seq = static_cast<int>(blockIdx.x / (static_cast<unsigned>(p.Hkv) * groups));
  const int in_seq = static_cast<int>(blockIdx.x - static_cast<unsigned>(seq) * p.Hkv * groups);
  const int hk = in_seq / groups, group = in_seq % groups;

  const Line lo = make_line(p, own);
  unsigned before = 0;
  for (int b = lane; b < seq; b += 32) before += lo.own_units(p, b);
  before = __reduce_add_sync(0xFFFFFFFFu, before);
  const unsigned units = lo.units_between(p.prefix, total_of(p, seq));
  const unsigned triple = static_cast<unsigned>(hk) * lo.rt_own + group * kRows / own.rows;
  const unsigned first = lo.prefix_units + before + triple * units;
  const unsigned c0 = first / lo.span, c1 = (first + units - 1) / lo.span;
  if (p.prefix == 0 && c0 == c1) {   // written by the one CTA that had it
    grid_wait();
    return;
  }
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
  // warps of a row, this warp's row and turn
  const int here = min(kRows, rows - group * kRows);
  const int shift = here > 8 ? 0 : here > 4 ? 1 : here > 2 ? 2 : here > 1 ? 3 : 4;
  const int r = warp >> shift, part = warp & ((1 << shift) - 1);
  const bool mine = r < here;
  const int row = group * kRows + r;

  // the row's shares: n0 of the prefix, then n1 of its own keys
  unsigned d0 = 0, n0 = 0, pt = 0;
  int in0 = 0;
  if (p.prefix > 0) {
    const unsigned gr = static_cast<unsigned>(seq) * rows + row;   // the row in the prefix segment
    pt = static_cast<unsigned>(hk) * lp.rt_prefix + gr / pre.rows;
    in0 = static_cast<int>(gr % pre.rows);
    const unsigned pu = lp.units_between(0, lp.prefix_end), f = pt * pu;
    d0 = f / lp.span;
    n0 = (f + pu - 1) / lp.span - d0 + 1;
  }
  const unsigned n1 = c1 - c0 + 1;
  const long long whole0 = 2LL * pre.ctas + pt;
  const long long whole1 = 2LL * own.ctas + static_cast<long long>(p.Hkv) * (lo.rt_prefix + static_cast<long long>(seq) * lo.rt_own) + triple;
  grid_wait();

  float top = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  if (mine) {
    for (unsigned j0 = part; j0 < n0 + n1; j0 += 32u << shift) {
      // lane = share: maximum, sum and place of up to 32 of them at once
      const unsigned j = j0 + (static_cast<unsigned>(lane) << shift);
      float m2 = -INFINITY, l2 = 0.f;
      unsigned long long at = 0;
      if (j < n0 + n1) {
        const bool first_part = j < n0;
        const unsigned i = first_part ? j : j - n0;
        const CacheLaunch& how = first_part ? pre : own;
        const long long share = (first_part ? n0 : n1) == 1 ? (first_part ? whole0 : whole1) : 2LL * ((first_part ? d0 : c0) + i) + (i == 0 ? 1 : 0);
        const int in = first_part ? in0 : row % own.rows;
        const float* from = share_at(p, how, share, D);
        m2 = __ldcg(from + how.rows * D + in);
        l2 = __ldcg(from + how.rows * D + how.rows + in);
        at = reinterpret_cast<unsigned long long>(from + in * D);
      }
      float to = fmaxf(top, m2);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xFFFFFFFFu, to, o));
      const float ref = to == -INFINITY ? 0.f : to;
      const float f1 = ex2_approx(top - ref), f2 = ex2_approx(m2 - ref);
      float part_sum = l2 * f2;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part_sum += __shfl_xor_sync(0xFFFFFFFFu, part_sum, o);
      sum = sum * f1 + part_sum;
      top = to;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f1;
      const int n = min(32, static_cast<int>((n0 + n1 - j0 + (1u << shift) - 1) >> shift));
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float* from = reinterpret_cast<const float*>(__shfl_sync(0xFFFFFFFFu, at, i)) + lane * V;
        const float f = __shfl_sync(0xFFFFFFFFu, f2, i);
        if constexpr (V == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(from));
          acc[0] += f * v.x;
          acc[1] += f * v.y;
          acc[2] += f * v.z;
          acc[3] += f * v.w;
        } else if constexpr (V == 2) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(from));
          acc[0] += f * v.x;
          acc[1] += f * v.y;
        } else {
          acc[0] += f * __ldcg(from);
        }
      }
    }
  }
  if (shift > 0) {   // the warps of a row, in order
#pragma unroll
    for (int i = 0; i < V; ++i) s_acc[warp][lane * V + i] = acc[i];
    if (lane == 0) {
      s_top[warp] = top;
      s_sum[warp] = sum;
    }
    __syncthreads();
    if (part != 0) return;
    float to = top;
    for (int w = 1; w < 1 << shift; ++w) to = fmaxf(to, s_top[warp + w]);
    const float ref = to == -INFINITY ? 0.f : to;
    const float f0 = ex2_approx(top - ref);
    sum *= f0;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] *= f0;
    for (int w = 1; w < 1 << shift; ++w) {
      const float f = ex2_approx(s_top[warp + w] - ref);
      sum += f * s_sum[warp + w];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += f * s_acc[warp + w][lane * V + i];
    }
    top = to;
  }
  if (!mine) return;
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

// The launches of a call: one over everything, or one over the prefix and one over the sequences' own keys where only one
// of the two has more than 16 rows to a key/value head (the 16-row tile would read its keys once for every 16 rows).
struct Plan {
  CacheLaunch of[2];   // the prefix's, the sequences'; equal if one launch has both
  bool wide[2];
  bool join;
  long long floats, units;
};

Plan make_plan(int B, int Hkv, long long per, int head_dim, int prefix, long long capacity) {
  Plan pl{};
  const long long rows[2] = {B * per, per};
  for (int i = 0; i < 2; ++i) pl.wide[i] = rows[i] > kRows;
  if (prefix == 0) pl.wide[0] = pl.wide[1];
  const bool one = prefix == 0 || pl.wide[0] == pl.wide[1];
  for (int i = 0; i < 2; ++i) {
    CacheLaunch& how = pl.of[i];
    how.rows = pl.wide[i] ? kWideRows : kRows;
    how.keys = kTileKeys;
    how.prefix = prefix > 0 && (one || i == 0);
    how.own = one || i == 1;
    if (i == 1 && one) {
      how = pl.of[0];
      break;
    }
    long long triples = 0;
    if (how.prefix) triples += Hkv * ((rows[0] + how.rows - 1) / how.rows);
    if (how.own) triples += static_cast<long long>(B) * Hkv * ((rows[1] + how.rows - 1) / how.rows);
    const long long most = triples * ((capacity + how.keys - 1) / how.keys);
    pl.units += most;
    how.ctas = static_cast<int>(most < kCacheCtas ? most : kCacheCtas);
    how.share0 = pl.floats;
    pl.floats += (2LL * kCacheCtas + (prefix > 0 ? triples : 0)) * how.rows * (head_dim + 2);
  }
  pl.join = prefix > 0 || capacity > kUncutTiles * kTileKeys;
  return pl;
}

template <int D, bool BF16>
cudaError_t launch_narrow(const CUtensorMap& tmK, const CUtensorMap& tmV, const CacheAttnParams& p, const CacheLaunch& how, int d_real, bool chained,
                          cudaStream_t stream) {
  using Cfg = CacheCfg<D>;
  auto kern = omni_cache_attn_kernel<D, BF16>;
  static SmemAttrOnce attr_once[kMaxDevices];
  const cudaError_t e = ensure_smem_attr(kern, Cfg::kSmem, attr_once);
  if (e != cudaSuccess) return e;
  return launch_chained(kern, how.ctas, kThreads, Cfg::kSmem, chained, stream, tmK, tmV, p, how, d_real);
}

template <int D, bool BF16>
cudaError_t launch_t(const CacheAttnParams& p, cudaStream_t stream) {
  const long long per = p.G * static_cast<long long>(p.T);
  const Plan pl = make_plan(p.B, p.Hkv, per, D, p.prefix, p.capacity);
  CUtensorMap tmK, tmV;
  cudaError_t e = make_page_maps(p, D, BF16, &tmK, &tmV);
  for (int i = 0; e == cudaSuccess && i < 2; ++i) {
    if (i == 1 && pl.of[0].own) break;
    e = pl.wide[i] ? launch_cache_wide(D, BF16, tmK, tmV, p, pl.of[i], i == 1, stream)
                   : launch_narrow<D == 128 ? 128 : 64, BF16>(tmK, tmV, p, pl.of[i], D, i == 1, stream);   // head_dim 32 as 64
  }
  if (e != cudaSuccess || !pl.join) return e;
  const unsigned grid = static_cast<unsigned>(p.B * static_cast<long long>(p.Hkv) * ((per + kRows - 1) / kRows));
  return launch_chained(omni_cache_join_kernel<D, BF16>, grid, 512, 0, true, stream, p, pl.of[0], pl.of[1]);
}

}  // namespace

long long cache_attn_workspace_bytes(int B, int H, int Hkv, int T, int head_dim, bool prefix) {
  return make_plan(B, Hkv, static_cast<long long>(H / Hkv) * T, head_dim, prefix ? 1 : 0, 1 << 30).floats * 4;
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
