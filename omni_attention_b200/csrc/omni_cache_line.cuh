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
// tokens of sequence b that exist once this call's are in: [0, capacity]
__device__ __forceinline__ int total_of(const CacheAttnParams& p, int b) {
  const long long n = static_cast<long long>(max(__ldg(p.lengths + b), 0)) + count_of(p, b);
  return static_cast<int>(n < p.capacity ? n : p.capacity);
}
// keys row (b, t) sees
__device__ __forceinline__ int limit_of(const CacheAttnParams& p, int b, int t) {
  if (t >= count_of(p, b)) return 0;
  const int total = total_of(p, b);
  if (p.limits != nullptr) return min(max(__ldg(p.limits + static_cast<long long>(b) * p.T + t), 0), total);
  if (!p.causal) return total;
  const long long n = static_cast<long long>(max(__ldg(p.lengths + b), 0)) + t + 1;
  return static_cast<int>(n < total ? n : total);
}

struct Line {
  CacheLaunch how;
  long long units;          // all of them
  long long span;           // of one CTA
  long long prefix_units;   // those of the prefix, which come first
  int prefix_seq;           // the sequence whose page table the prefix is read through: the longest
  int prefix_end;
  int tiles_prefix, rt_prefix, rt_own;

  __device__ __forceinline__ int tiles_between(int from, int to) const {
    return to > from ? (to - from + how.keys - 1) / how.keys : 1;   // a triple without keys still has rows to write
  }
  __device__ __forceinline__ long long own_units(const CacheAttnParams& p, int b) const {
    return how.own ? static_cast<long long>(p.Hkv) * rt_own * tiles_between(p.prefix, total_of(p, b)) : 0;
  }
};

// All lanes of a warp; every CTA of every kernel comes to the same line.
__device__ __forceinline__ Line make_line(const CacheAttnParams& p, const CacheLaunch& how) {
  Line ln;
  ln.how = how;
  ln.rt_own = (p.G * p.T + how.rows - 1) / how.rows;
  const int lane = threadIdx.x & 31;
  long long sum = 0;
  int most = -1, seq = 0;
  for (int b = lane; b < p.B; b += 32) {
    sum += ln.own_units(p, b);
    const int total = total_of(p, b);
    if (total > most) {
      most = total;
      seq = b;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const int m2 = __shfl_xor_sync(0xFFFFFFFFu, most, o), s2 = __shfl_xor_sync(0xFFFFFFFFu, seq, o);
    if (m2 > most || (m2 == most && s2 < seq)) {
      most = m2;
      seq = s2;
    }
  }
  ln.prefix_units = 0;
  ln.prefix_seq = seq;
  ln.prefix_end = min(p.prefix, most);
  ln.tiles_prefix = ln.tiles_between(0, ln.prefix_end);
  ln.rt_prefix = 0;
  if (how.prefix) {
    ln.rt_prefix = static_cast<int>((static_cast<long long>(p.B) * p.G * p.T + how.rows - 1) / how.rows);
    ln.prefix_units = static_cast<long long>(p.Hkv) * ln.rt_prefix * ln.tiles_prefix;
  }
  ln.units = sum + ln.prefix_units;
  ln.span = (ln.units + how.ctas - 1) / how.ctas;
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
  long long u, u_end, base;
  int seg;

  __device__ __forceinline__ Walk(const CacheAttnParams& p, const CacheLaunch& how) : ln(make_line(p, how)), base(0), seg(-1) {
    u = ln.span * blockIdx.x;
    u_end = min(u + ln.span, ln.units);
    if (u >= u_end || u < ln.prefix_units) return;
    base = ln.prefix_units;
    const int lane = threadIdx.x & 31;
    for (int b0 = 0;; b0 += 32) {   // ends: u lies in some sequence's units
      const int b = b0 + lane;
      const long long mine = b < p.B ? ln.own_units(p, b) : 0;
      long long upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
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
    if (u >= u_end) return false;
    pc.prefix = seg < 0;
    pc.seg = seg;
    const int rts = pc.prefix ? ln.rt_prefix : ln.rt_own;
    pc.table_of = pc.prefix ? ln.prefix_seq : seg;
    pc.key0 = pc.prefix ? 0 : p.prefix;
    pc.total = pc.prefix ? ln.prefix_end : total_of(p, seg);
    pc.rows = pc.prefix ? p.B * p.G * p.T : p.G * p.T;
    const int tiles = pc.prefix ? ln.tiles_prefix : ln.tiles_between(pc.key0, pc.total);
    const long long triple = (u - base) / tiles;
    pc.tile0 = static_cast<int>(u - base - triple * tiles);
    pc.tile1 = static_cast<int>(min(static_cast<long long>(tiles), pc.tile0 + (u_end - u)));
    pc.hk = static_cast<int>(triple / rts);
    pc.rt = static_cast<int>(triple - static_cast<long long>(pc.hk) * rts);
    pc.whole = pc.tile0 == 0 && pc.tile1 == tiles;
    // CTA i has share 2 i (of a triple that began before its span) and 2 i + 1 (of one that begins in it and goes on after
    // it); with a prefix, triples inside one span have a share of their own behind those: the prefix's, then the sequences'.
    pc.share = -1;
    if (!pc.whole) {
      pc.share = 2LL * blockIdx.x + (pc.tile0 == 0 ? 1 : 0);
    } else if (p.prefix > 0) {
      pc.share = 2LL * ln.how.ctas + triple;
      if (!pc.prefix) pc.share += static_cast<long long>(p.Hkv) * (ln.rt_prefix + static_cast<long long>(seg) * ln.rt_own);
    }
    u += pc.tile1 - pc.tile0;
    if (u - base >= static_cast<long long>(p.Hkv) * rts * tiles) {
      base += static_cast<long long>(p.Hkv) * rts * tiles;
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
  id.t = in / p.G;
  id.g = in - id.t * p.G;
  return id;
}
__device__ __forceinline__ long long out_row(const CacheAttnParams& p, const RowId& id, int hk) {
  return (static_cast<long long>(id.b) * p.H + static_cast<long long>(hk) * p.G + id.g) * p.T + id.t;
}

}  // namespace omni
