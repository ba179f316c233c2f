// How the work of an attention over a paged cache is cut up, for the kernels that do it and the one that joins the shares.
//
// A segment is a set of keys with the query rows that read it: the shared prefix with the rows of all sequences, or one
// sequence's own keys (those behind the prefix) with its own rows. The rows of a segment and key/value head in tiles of
// `rows`, its keys in tiles of `keys`: a triple (segment, key/value head, row tile) has one unit per tile of keys, and the
// units of all triples form one line, which is cut into equal spans, one per CTA. A span may begin or end inside a triple.
#pragma once
#include "omni_cache_attn.cuh"
#include "omni_common.cuh"

namespace omni {

__device__ __forceinline__ int count_of(const CacheAttnParams& p, int b) {
  return p.counts == nullptr ? p.T : min(max(__ldg(p.counts + b), 0), p.T);
}
// tokens of sequence b that exist once this call's are in: [0, capacity]; 0 for a sequence without new tokens (nobody asks)
__device__ __forceinline__ int total_of(const CacheAttnParams& p, int b) {
  const int c = count_of(p, b);
  const unsigned n = static_cast<unsigned>(max(__ldg(p.lengths + b), 0)) + c;
  return c == 0 ? 0 : static_cast<int>(min(n, static_cast<unsigned>(p.capacity)));
}
// keys row (b, t) sees
__device__ __forceinline__ int limit_of(const CacheAttnParams& p, int b, int t) {
  if (t >= count_of(p, b)) return 0;
  const int total = total_of(p, b);
  if (p.limits != nullptr) return min(max(__ldg(p.limits + static_cast<long long>(b) * p.T + t), 0), total);
  if (!p.causal) return total;
  return static_cast<int>(min(static_cast<unsigned>(max(__ldg(p.lengths + b), 0)) + t + 1, static_cast<unsigned>(total)));
}

struct Line {
  CacheLaunch how;
  unsigned units;           // all of them
  unsigned span;            // of one CTA
  unsigned prefix_units;    // those of the prefix, which come first
  int prefix_seq;           // the sequence whose page table the prefix is read through: the longest
  int prefix_end;
  int rt_prefix, rt_own;
  // The busiest CTA's tiles of keys decide how the line is cut. uncut: a triple is one unit, none is cut and nothing has to
  // be joined (cutting costs how.uncut tiles); even: each triple is cut into that many parts by itself, one per CTA; else
  // even spans of the whole line, where a CTA may have two pieces (kPieceTiles).
  bool uncut;
  unsigned even;   // 0: not so

  __device__ __forceinline__ unsigned part(unsigned units) const { return (units + even - 1) / even; }
  __device__ __forceinline__ unsigned parts(unsigned units) const {
    const unsigned n = part(units);
    return (units + n - 1) / n;
  }
  __device__ __forceinline__ unsigned first_cta(const CacheAttnParams& p, int seq, unsigned triple) const {
    return even * (seq < 0 ? triple : static_cast<unsigned>(p.Hkv) * (rt_prefix + static_cast<unsigned>(seq) * rt_own) + triple);
  }
  __device__ __forceinline__ int tiles_between(int from, int to) const {
    return to > from ? (to - from + kTileKeys - 1) / kTileKeys : 1;   // a triple without keys still has rows to write
  }
  __device__ __forceinline__ unsigned units_between(int from, int to) const { return uncut ? 1u : tiles_between(from, to); }
  __device__ __forceinline__ unsigned own_units(const CacheAttnParams& p, int b) const {
    return how.own ? static_cast<unsigned>(p.Hkv) * rt_own * units_between(p.prefix, total_of(p, b)) : 0u;
  }
};

// All lanes of a warp; every CTA of every kernel comes to the same line. (The host refuses what would have 2^31 units.)
__device__ __forceinline__ Line make_line(const CacheAttnParams& p, const CacheLaunch& how) {
  Line ln;
  ln.how = how;
  ln.rt_own = how.rt_own;
  const int lane = threadIdx.x & 31;
  unsigned sum = 0;
  int most = -1, seq = 0;
  for (int b = lane; b < p.B; b += 32) {
    const int total = total_of(p, b);
    sum += ln.tiles_between(p.prefix, total);
    if (total > most) {
      most = total;
      seq = b;
    }
  }
  sum = __reduce_add_sync(0xFFFFFFFFu, sum);
  const int most_of_all = __reduce_max_sync(0xFFFFFFFFu, most);
  seq = __reduce_min_sync(0xFFFFFFFFu, most == most_of_all ? seq : 0x7FFFFFFF);
  most = most_of_all;
  ln.prefix_seq = seq;
  ln.prefix_end = min(p.prefix, most);
  ln.rt_prefix = how.rt_prefix;
  const unsigned tiles_prefix = how.prefix ? ln.tiles_between(0, ln.prefix_end) : 0u, tiles_own = how.own ? ln.tiles_between(p.prefix, most) : 0u;
  const unsigned heads = p.Hkv, rt_own = how.own ? ln.rt_own : 0;
  const unsigned cut_units = heads * (ln.rt_prefix * tiles_prefix + rt_own * sum), cut_span = (cut_units + how.ctas - 1) / how.ctas;
  const unsigned triples = heads * (ln.rt_prefix + rt_own * p.B), per_cta = how.per_cta;
  const unsigned longest = max(tiles_prefix, tiles_own), even = how.even >= 2 ? (longest + how.even - 1) / how.even : 0xFFFFFFFFu;
  const unsigned cut = min(even, cut_span + kPieceTiles);
  ln.uncut = static_cast<unsigned long long>(per_cta) * longest <= cut + how.uncut;
  ln.even = !ln.uncut && even == cut ? how.even : 0u;
  ln.prefix_units = how.prefix ? heads * ln.rt_prefix * ln.units_between(0, ln.prefix_end) : 0u;
  ln.units = ln.uncut ? triples : cut_units;
  ln.span = ln.uncut ? per_cta : cut_span;
  return ln;
}

// The part of one triple that lies in a CTA's span.
struct Piece {
  bool prefix, whole;
  int seg, hk, rt;           // sequence (-1: the prefix), key/value head, row tile
  int tile0, tile1;          // tiles of keys
  int rows, key0, total, table_of;
  long long share;           // where its rows' shares go in the workspace, -1: it is written out
};

// Walks over the pieces of one CTA. The constructor is for all lanes of a warp, next() for any thread by itself.
struct Walk {
  Line ln;
  unsigned u, u_end, base;
  int seg;

  __device__ __forceinline__ Walk(const CacheAttnParams& p, const CacheLaunch& how) : ln(make_line(p, how)), base(0), seg(-1) {
    if (ln.even) {   // u: the triple, u_end: the part
      u = blockIdx.x / ln.even;
      u_end = blockIdx.x - u * ln.even;
      return;
    }
    u = ln.span * blockIdx.x;
    u_end = min(u + ln.span, ln.units);
    if (u >= u_end || u < ln.prefix_units) return;
    if (p.B == 1) {
      base = ln.prefix_units;
      seg = 0;
      return;
    }
    base = ln.prefix_units;
    const int lane = threadIdx.x & 31;
    for (int b0 = 0;; b0 += 32) {   // ends: u lies in some sequence's units
      const int b = b0 + lane;
      const unsigned mine = b < p.B ? ln.own_units(p, b) : 0;
      unsigned upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned past = __ballot_sync(0xFFFFFFFFu, base + upto > u);
      if (past != 0) {
        const int l = __ffs(past) - 1;
        seg = b0 + l;
        base += __shfl_sync(0xFFFFFFFFu, upto - mine, l);
        break;
      }
      base += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
  }

  __device__ __forceinline__ bool next(const CacheAttnParams& p, Piece& pc) {
    unsigned triple = 0, first, n, rts;
    if (ln.even) {
      const unsigned np = static_cast<unsigned>(p.Hkv) * ln.rt_prefix, per = static_cast<unsigned>(p.Hkv) * ln.rt_own;
      if (u >= np + (ln.how.own ? per * p.B : 0u)) return false;
      seg = u < np ? -1 : static_cast<int>((u - np) / per);
      triple = u < np ? u : u - np - static_cast<unsigned>(seg) * per;
    } else if (u >= u_end) {
      return false;
    }
    pc.prefix = seg < 0;
    pc.seg = seg;
    rts = pc.prefix ? ln.rt_prefix : ln.rt_own;
    pc.table_of = pc.prefix ? ln.prefix_seq : seg;
    pc.key0 = pc.prefix ? 0 : p.prefix;
    pc.total = pc.prefix ? ln.prefix_end : total_of(p, seg);
    pc.rows = pc.prefix ? p.B * p.G * p.T : p.G * p.T;
    const unsigned units = ln.units_between(pc.key0, pc.total);
    if (ln.even) {
      first = u_end * ln.part(units);
      if (first >= units) return false;   // a short triple has fewer parts
      n = min(ln.part(units), units - first);
    } else {
      triple = (u - base) / units;
      first = u - base - triple * units;
      n = min(units - first, u_end - u);
    }
    pc.whole = n == units;
    pc.tile0 = static_cast<int>(first);
    pc.tile1 = ln.uncut ? ln.tiles_between(pc.key0, pc.total) : static_cast<int>(first + n);
    pc.hk = static_cast<int>(rts == 1 ? triple : triple / rts);
    pc.rt = static_cast<int>(triple - pc.hk * rts);
    // CTA i has share 2 i (of a triple that began before its span) and 2 i + 1 (of one that begins in it and goes on after
    // it); with a prefix, triples inside one span have a share of their own behind those: the prefix's, then the sequences'.
    pc.share = -1;
    if (!pc.whole) {
      pc.share = 2LL * blockIdx.x + (first == 0 ? 1 : 0);
    } else if (p.prefix > 0) {
      pc.share = 2LL * ln.how.ctas + triple;
      if (!pc.prefix) pc.share += static_cast<long long>(p.Hkv) * (ln.rt_prefix + static_cast<long long>(seg) * ln.rt_own);
    }
    if (ln.even) {
      u = 0xFFFFFFFFu;   // that was all
      return true;
    }
    u += n;
    if (u - base >= p.Hkv * rts * units) {
      base += p.Hkv * rts * units;
      ++seg;
    }
    return true;
  }
};

// A share in the workspace: O [rows][D], then the rows' maxima [rows] (log2 domain) and sums [rows].
__device__ __forceinline__ float* share_at(const CacheAttnParams& p, const CacheLaunch& how, long long index, int d) {
  return p.partial + how.share0 + index * (how.rows * (d + 2));
}

// Which (batch element, token, query head of the group) row r of a segment is.
struct RowId {
  int b, t, g;
};
__device__ __forceinline__ RowId row_of(const CacheAttnParams& p, bool prefix, int b, int r) {
  RowId id;
  const int per = p.G * p.T;
  id.b = prefix ? r / per : b;
  const int in = prefix ? r - id.b * per : r;
  id.t = p.T == 1 ? 0 : p.G == 1 ? in : in / p.G;
  id.g = in - id.t * p.G;
  return id;
}
__device__ __forceinline__ long long out_row(const CacheAttnParams& p, const RowId& id, int hk) {
  return (static_cast<long long>(id.b) * p.H + static_cast<long long>(hk) * p.G + id.g) * p.T + id.t;
}

// ---------------------------------------------------------------------------------------------------------------------
// pieces of the two kernels
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? 16 : 0;   // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// x: element along head_dim (a multiple of 64), y: row of the matrix of pages.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y)
               : "memory");
}

template <bool BF16>
constexpr uint32_t kExponent = BF16 ? 0x7F80u : 0x7C00u;   // all of its bits set: infinite or NaN

// Whether one of the eight 16-bit values is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool not_finite(const uint4& v) {
  constexpr uint32_t m = kExponent<BF16>;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & m) == m || (w[i] & (m << 16)) == m << 16;
  return bad;
}
// The eight values with zeros in the place of those.
template <bool BF16>
__device__ __forceinline__ uint4 finite_part(const uint4& v) {
  constexpr uint32_t m = kExponent<BF16>;
  auto word = [](uint32_t w) { return w & (((w & m) == m ? 0u : 0xFFFFu) | ((w & (m << 16)) == m << 16 ? 0u : 0xFFFF0000u)); };
  return make_uint4(word(v.x), word(v.y), word(v.z), word(v.w));
}

// Programmatic dependent launch: a kernel so launched may start before its predecessor has ended; what that one wrote is
// there behind grid_wait. grid_go lets a successor start. Both are no-ops without such launches.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The ring of K and V tiles (128 keys, [64 columns][128 rows][128 bytes], 128-byte swizzle) that a warp fills page by page.
struct RingState {
  uint32_t fill = 0;                // entries filled so far
  bool alive = true;
};
// An entry is a tile of K or V (PAIR: K and V of the same keys, one behind the other).
template <int TILE, int CHUNKS, int SLOTS, bool PAIR>
struct Ring {
  uint32_t data, full, empty;       // shared addresses
  uint32_t (*valid)[4];             // [SLOTS]: of an entry with V, which keys are there
  volatile int* abort_flag;

  // All lanes of the producing warp: tiles tile0 .. tile1 of a piece, K then V of each.
  __device__ __forceinline__ void stream(const CacheAttnParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV, const Piece& pc, int tile1,
                                         RingState& st, int where) const {
    const int lane = threadIdx.x & 31;
    const int page_rows = 1 << p.page_shift;
    const int box = page_rows < 128 ? page_rows : 128;   // tokens of a copy
    const int pages = 128 / box;                         // copies of a tile and chunk: lane = copy
    const int* table = p.page_table + pc.table_of * p.table_stride;
    auto page_at = [&](int t) -> int {
      const int key = pc.key0 + t * 128 + lane * box;
      return t < tile1 && lane < pages && key < pc.total ? __ldg(table + (key >> p.page_shift)) : -1;
    };
    int next = page_at(pc.tile0);
    for (int t = pc.tile0; st.alive && t < tile1; ++t) {
      const int page = next, key = pc.key0 + t * 128 + lane * box;
      next = page_at(t + 1);
      const bool ok = page >= 0 && page < p.num_pages;
      if (!ok && lane < pages && key < pc.total && p.status != nullptr) atomicCAS(p.status, 0, kStatusBadIndex);
      const unsigned there = __ballot_sync(0xFFFFFFFFu, ok);
      uint32_t word = 0;   // keys 32 * lane .. of the tile that are there (lanes 0-3)
      if (lane < 4) {
        if (box >= 32) {
          word = there >> (32 * lane / box) & 1u ? 0xFFFFFFFFu : 0u;
        } else {
          word = (there >> (2 * lane) & 1u ? 0x0000FFFFu : 0u) | (there >> (2 * lane + 1) & 1u ? 0xFFFF0000u : 0u);
        }
      }
      const int y = ok ? ((page * p.Hkv + pc.hk) << p.page_shift) + (key & (page_rows - 1)) : 0;
      const uint32_t bytes = __popc(there) * box * 128 * CHUNKS;
#pragma unroll
      for (int kv = 0; kv < (PAIR ? 1 : 2); ++kv, ++st.fill) {
        const uint32_t s = st.fill % SLOTS;
        if (lane == 0 && st.fill >= SLOTS) {
          st.alive = mbar_wait_lim(empty + 8 * s, ((st.fill / SLOTS) - 1) & 1, abort_flag, p.status, where, p.wait_cycles);
        }
        st.alive = __shfl_sync(0xFFFFFFFFu, st.alive, 0) && !*abort_flag;
        st.alive = __all_sync(0xFFFFFFFFu, st.alive);
        if (!st.alive) break;
        if ((PAIR || kv == 1) && lane < 4) valid[s][lane] = word;
        __syncwarp();
        if (lane == 0) {
          if (bytes > 0) {
            mbar_expect_tx(full + 8 * s, PAIR ? 2 * bytes : bytes);
          } else {
            mbar_arrive(full + 8 * s);
          }
        }
        __syncwarp();
        if (ok) {
          const uint32_t to = data + s * (PAIR ? 2 * TILE : TILE) + lane * box * 128;
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) tma_load_2d(to + c * (128 * 128), kv == 0 ? tmK : tmV, full + 8 * s, c * 64, y);
          if constexpr (PAIR) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) tma_load_2d(to + TILE + c * (128 * 128), tmV, full + 8 * s, c * 64, y);
          }
        }
      }
    }
  }

  // A CTA that gave up: nothing may still be on its way into shared memory when it ends. By the producing warp, once no
  // other warp can give up any more.
  __device__ __forceinline__ void drain(const RingState& st) const {
    if ((threadIdx.x & 31) == 0) {
      for (uint32_t s = 0; s < SLOTS && s < st.fill; ++s) {
        const uint32_t last = ((st.fill - 1 - s) / SLOTS) * SLOTS + s;
        mbar_wait_drain(full + 8 * s, (last / SLOTS) & 1, 4000000000LL);
      }
    }
    __syncwarp();
  }
};

}  // namespace omni
