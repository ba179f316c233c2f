// Attention over a paged key/value cache for many query rows to a key/value head: an image's tokens, a draft, or all
// sequences' rows on the prefix they share. The mathematics, the cut of the work and the shares are those of
// omni_cache_attn.cu; a tile is 128 rows by 128 keys, on the tcgen05 tensor cores.
//
// Bound: at 128 rows the read of a tile (64 KB at head_dim 128) takes an SM about as long as the card's HBM rate gives it
// (2 800 cycles), its two products 1 024; from 256 rows on the second row tile finds the keys in L2 and the chain scores ->
// softmax -> P -> product bounds it. So the tiles of keys go to two softmax groups in turn, each with its own scores,
// maximum, sum and O, and one group's chain runs under the other's products; at the end of a piece the groups' halves are
// joined through shared memory. Measured, head_dim 128, bf16: 2 x 32 heads of 256 rows on 4 352 keys 53 us = 690 TFLOP/s (69 with
// the soft-cap): 34 tiles of 1 965 cycles, 20 500 cycles before the first and after the last (start 6 400, queries 4 800, first
// scores 1 100, end 8 200), at 1.74 GHz in a loop (power cap) and up to 1.9 in a short run; the 16 384 shared tokens of 64 sequences,
// 8 key/value heads, 31 us.
//
// Roles of a CTA (one per SM, 384 threads):
//   warps 0-3, 4-7  softmax groups: thread = query row = TMEM lane. They also gather the rows' queries into shared memory
//                   (any strides, rows of one tile may belong to different sequences) and write the result.
//   warp 8          TMA: K and V of each tile of keys page by page into a ring (lane = page of the tile)
//   warp 9          one elected thread issues every tcgen05.mma (warps 10 and 11 only give their registers up)
// Hand-overs go through mbarriers; every wait is bounded as in the forward kernels. TMEM: S of the two groups (P, 16 bit,
// over the first half of S), O of the two groups. P is one 16-bit value, as in the block-mask forward (with its rest as a second
// operand, as in omni_cache_attn.cu, the products would take half as long again, and the rest's columns in TMEM are the next
// scores'): the error against 64 bits is 2.3e-3 of the result's norm where its own rounding to bf16 is 1.7e-3.
//
// A value that is infinite or NaN must not reach the rows that do not see its key (0 * NaN): where rows of a tile see
// different numbers of keys it is taken out of the product. What such values make of the rows that see them is found when
// the piece is written (write_not_finite).
//
// Keys that are not there - behind the last token, in a page that does not exist - are never loaded; what the ring holds in
// their places is zeroed in V (0 * NaN) and masked in S.
#include "omni_cache_line.cuh"
#include "omni_launch.h"

namespace omni {

namespace {

constexpr int kWideThreads = 384;
// Registers: compiled for 168 a thread (what 384 threads can have); the softmax groups take over most of the third
// warpgroup's. The increase must be covered by the decrease, or setmaxnreg.inc waits forever (checked before the launch).
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
constexpr float kLazyLog2 = 8.f;
constexpr long long kDrain = 4000000000LL;

template <int D>
struct WideCfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kChunks = D / 64;
  static constexpr int kChunk = 128 * 128;
  static constexpr int kSlots = D == 128 ? 6 : 10;   // K and V tiles in flight
  // Scores of a tile in two halves of 64 keys: the second half is computed as soon as the group has read the scores before for
  // the last time, under their exponentials, and its maximum is looked for under the first half's product. 2 x 16 heads of 256
  // rows on 4 352 keys: head_dim 64 33.9 -> 31.2 us; head_dim 128 (32 heads) 53.2 -> 55.9 (a product 64 keys wide
  // reads the queries from shared memory twice as often; no counter shows whether that is the reason).
  static constexpr bool kHalves = D == 64;
  static constexpr int kBars = (1 + kSlots) * kTile;
  // Behind the tiles: barriers, flags and limits, which keys are there, row states, the piece's description.
  static constexpr int kFlags = D == 128 ? 256 : 288, kValid = kFlags + 80, kRows = D == 128 ? 512 : 576;
  static constexpr int kPiece = D == 128 ? kValid + 16 * kSlots : kRows + 2560;
  static constexpr int kSmem = kBars + kRows + 2560 + (D == 128 ? 0 : 64);
  static_assert((2 * kSlots + 16) * 8 <= kFlags && (D == 128 ? kPiece + 64 : kValid + 16 * kSlots) <= kRows && kPiece % 16 == 0, "shared memory layout");
};

// Named barrier of the eight softmax warps.
__device__ __forceinline__ void softmax_sync() { named_barrier_sync(1, 256); }

// The first n (may be below 0 or above 32) bits set.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }

template <int COLS>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, float (&f)[COLS]) {
  if constexpr (COLS == 32) {
    uint32_t r[32];
    tmem_ld32(addr, r);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(r[j]);
  } else {
    uint32_t r[16];
    tmem_ld16(addr, r);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(r[j]);
  }
}

// Zeros in the place of scores that are not allowed.
__device__ __forceinline__ void zero_not_allowed64(uint32_t allow0, uint32_t allow1, float (&s)[64]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j] = ((allow0 >> j) & 1u) ? s[j] : 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) s[32 + j] = ((allow1 >> j) & 1u) ? s[32 + j] : 0.f;
}

// Takes what is infinite or NaN out of a row of a V tile (chunks of 128 bytes, `pitch` apart). Whether there was any.
template <bool BF16, int CHUNKS>
__device__ __noinline__ bool take_out_not_finite(uint8_t* row, int r, int pitch) {
  bool bad = false;
#pragma unroll 4
  for (int c = 0; c < CHUNKS * 8; ++c) {
    uint4* at = reinterpret_cast<uint4*>(row + (c >> 3) * pitch + r * 128 + (c & 7) * 16);
    if (not_finite<BF16>(*at)) {
      *at = finite_part<BF16>(*at);
      bad = true;
    }
  }
  return bad;
}

// By the eight softmax warps, when a piece is written: elements whose row sees infinite or NaN values in their column are what
// these add up to (the product has them as zeros, as inf, or as NaN where an fp16 weight is below the type's smallest).
// Keys key0 .. key1, a thread's row (keys below `lim`, columns c0 .. c1, 64 at most) in `out`, or in `share` (32 bit). `keys`: 8
// words in shared memory. From memory, a key to a thread; then the keys that have such values, row by row.
template <bool BF16>
__device__ __noinline__ void write_not_finite(const CacheAttnParams& p, const Piece& pc, int key0, int key1, int lim, int d, int c0, int c1, float* share,
                                              uint16_t* out, volatile uint32_t* keys) {
  const int tid = threadIdx.x, mask = (1 << p.page_shift) - 1;
  const int* table = p.page_table + pc.table_of * p.table_stride;
  unsigned long long plus = 0, minus = 0;   // columns that met +inf or NaN, -inf or NaN: both is NaN
  const unsigned long long all = c1 - c0 == 64 ? ~0ull : (1ull << (c1 - c0)) - 1;
  auto values = [&](int key) -> const uint16_t* {
    const int page = __ldg(table + (key >> p.page_shift));
    if (page < 0 || page >= p.num_pages) return nullptr;
    return static_cast<const uint16_t*>(p.v_pages) + (((static_cast<long long>(page) * p.Hkv + pc.hk) << p.page_shift) + (key & mask)) * d;
  };
  for (int base = key0; base < key1; base += 256) {
    bool bad = false;
    if (base + tid < key1) {
      const uint16_t* v = values(base + tid);
      for (int c = 0; v != nullptr && c < d; c += 8) bad |= not_finite<BF16>(__ldg(reinterpret_cast<const uint4*>(v + c)));
    }
    const uint32_t word = __ballot_sync(0xFFFFFFFFu, bad);
    if ((tid & 31) == 0) keys[tid >> 5] = word;
    softmax_sync();
    for (int w = 0; w < 8; ++w) {
      for (uint32_t left = keys[w]; left != 0; left &= left - 1) {
        const int key = base + 32 * w + __ffs(left) - 1;
        if (key >= lim || (plus & minus) == all) break;
        const uint16_t* v = values(key);
        for (int c = c0; c < c1; c += 8) {
          const uint4 eight = __ldg(reinterpret_cast<const uint4*>(v + c));
          if (!not_finite<BF16>(eight)) continue;
          const uint32_t words[4] = {eight.x, eight.y, eight.z, eight.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t raw = words[i >> 1] >> (16 * (i & 1)) & 0xFFFFu;
            if ((raw & kExponent<BF16>) != kExponent<BF16>) continue;
            const bool nan = (raw & 0x7FFFu) != kExponent<BF16>;
            const unsigned long long bit = 1ull << (c - c0 + i);
            if (nan || !(raw >> 15)) plus |= bit;
            if (nan || raw >> 15) minus |= bit;
          }
        }
      }
    }
    softmax_sync();   // the next words go over these
  }
  for (unsigned long long left = plus | minus; left != 0; left &= left - 1) {
    const int i = __ffsll(left) - 1;
    const bool up = plus >> i & 1u, down = minus >> i & 1u;
    const float x = up && down ? __int_as_float(0x7FFFFFFF) : up ? INFINITY : -INFINITY;
    if (share != nullptr) {
      share[c0 + i] = x;
    } else {
      out[c0 + i] = static_cast<uint16_t>(pack2<BF16>(x, 0.f));
    }
  }
}

template <int D, bool BF16, bool SOFTCAP>
__global__ void __launch_bounds__(kWideThreads, 1)
omni_cache_wide_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ CacheAttnParams p, const __grid_constant__ CacheLaunch how, int d_real) {
  using Cfg = WideCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];   // what the 128-byte swizzle wants; there is no room to align by hand
  if ((smem_u32(smem) & 1023u) != 0) {
    if (p.status != nullptr && threadIdx.x == 0) atomicExch(p.status, kStatusWaitTimeout | (49 << 8));
    return;
  }
  const uint32_t sQ = smem_u32(smem), sRing = sQ + Cfg::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBars);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * Cfg::kSlots;
  const uint32_t bar_q = bar_empty + 8 * Cfg::kSlots;   // the rows' queries are in shared memory
  const uint32_t bar_s = bar_q + 8;                     // [2] scores done
  const uint32_t bar_p = bar_s + 16;                    // [2] P stored
  const uint32_t bar_h = bar_p + 16;                    // [2] P of the tile's first 64 keys stored
  const uint32_t bar_o = bar_h + 16;                    // [2] the group's last product of the piece done
  const uint32_t bar_s2 = bar_o + 16;                   // [2] scores of the tile's last 64 keys done (kHalves)
  const uint32_t bar_e = bar_s2 + 16;                   // [2] and read for the last time
  const uint32_t bar_end = bar_e + 16;                  // drain of a launch that gives up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kBars + Cfg::kFlags);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_lim = reinterpret_cast<int*>(tmem_slot + 2);                                    // [8] largest limit of a warp's rows, [8] smallest
  Piece* s_piece = reinterpret_cast<Piece*>(smem + Cfg::kBars + Cfg::kPiece);
  static_assert(sizeof(Piece) <= 64, "shared memory layout");
  volatile int* s_bad = s_lim + 16;   // [0] a value that is not finite was taken out, [1] an element is not though its row's sum is
  uint32_t(*s_valid)[4] = reinterpret_cast<uint32_t(*)[4]>(smem + Cfg::kBars + Cfg::kValid);      // [kSlots] keys that are there
  float* s_m = reinterpret_cast<float*>(smem + Cfg::kBars + Cfg::kRows);                         // [2][128]
  float* s_l = s_m + 256;                                                                 // [2][128]
  int* s_out = reinterpret_cast<int*>(s_l + 256);                                         // [128] where a row is written

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < Cfg::kSlots; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, 1);
    }
    mbar_init(bar_q, 256);
    for (int g = 0; g < 2; ++g) {
      mbar_init(bar_s + 8 * g, 1);
      mbar_init(bar_p + 8 * g, 128);
      mbar_init(bar_h + 8 * g, 128);
      mbar_init(bar_o + 8 * g, 1);
      mbar_init(bar_s2 + 8 * g, 1);
      mbar_init(bar_e + 8 * g, 128);
    }
    mbar_init(bar_end, 1);
    *abort_flag = 0;
    s_bad[0] = s_bad[1] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Ring<Cfg::kTile, Cfg::kChunks, Cfg::kSlots, false> ring{sRing, bar_full, bar_empty, s_valid, abort_flag};
  const long long limit = p.wait_cycles;
  RingState st;
  if (!how.late_wait) grid_wait();   // lengths, queries and pages may be the predecessor's work
  grid_go();
  Walk walk(p, how);
  Piece pc;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // =========================== softmax groups ===================================================
    const int g = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 128 * g + lanes, tO = tmem + 256 + D * g + lanes;
    const float scale_log2 = p.scale * 1.4426950408889634f, inv_scale_log2 = 1.f / scale_log2;
    const float cap_in = SOFTCAP ? p.scale / p.softcap : 0.f, cap_out = SOFTCAP ? p.softcap / p.scale : 0.f;
    uint32_t n_vis = 0, n_pieces = 0;   // this group's visits and pieces with visits so far = phases of its barriers
    uint32_t fill = 0;                  // ring entries of the pieces before this one
    // The walk is kept in local memory here: it is wanted once a piece, and its twenty registers throughout (spills in the
    // loop otherwise: 532 -> 577 us for 32 heads of 4096 rows on 4K keys).
    Walk own_walk = walk;
    asm volatile("" ::"l"(&own_walk) : "memory");
    while (own_walk.next(p, pc)) {
      const int n = pc.tile1 - pc.tile0;
      // ---- the rows' queries: thread (row tid / 2, half of its chunks). (Two warps of their own with cp.async took longer:
      // their copies stood behind the other warps' polls, 700 cycles each.) ----
      {
        const int row = pc.rt * kWideRows + (tid >> 1);
        const uint4* src = nullptr;
        if (row < pc.rows) {
          const RowId id = row_of(p, pc.prefix, pc.seg, row);
          src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + id.b * p.qs_b +
                                               (static_cast<long long>(pc.hk) * p.G + id.g) * p.qs_h + id.t * p.qs_t);
        }
        const int c0 = (tid & 1) * (D / 16);
        uint4 v[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          v[i] = src != nullptr && (c0 + i) * 8 < d_real ? __ldg(src + c0 + i) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int c = c0 + i, rr = tid >> 1;
          *reinterpret_cast<uint4*>(smem + (c >> 3) * Cfg::kChunk + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[i];
        }
        fence_async_smem();
        mbar_arrive(bar_q);
      }
      const int my_row = pc.rt * kWideRows + r, rows = min(kWideRows, pc.rows - pc.rt * kWideRows);
      int lim = 0;
      if (r < rows) {
        const RowId id = row_of(p, pc.prefix, pc.seg, my_row);
        lim = min(limit_of(p, id.b, id.t), pc.total);
        if (g == 0) s_out[r] = static_cast<int>(out_row(p, id, pc.hk));
      }
      const int warp_max = __reduce_max_sync(0xFFFFFFFFu, lim), warp_min = __reduce_min_sync(0xFFFFFFFFu, lim > 0 ? lim : 0x7FFFFFFF);   // (rows that see nothing are zeroed at the end)
      if (lane == 0) {
        s_lim[warp] = warp_max;
        s_lim[8 + warp] = warp_min;
      }
      if (tid == 0) *s_piece = pc;   // for the piece's end: its registers are wanted in between
      named_barrier_sync(2 + g, 128);
      int lim_max = s_lim[4 * g], lim_min = s_lim[8 + 4 * g];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        lim_max = max(lim_max, s_lim[4 * g + w]);
        lim_min = min(lim_min, s_lim[8 + 4 * g + w]);
      }

      const int key_first = pc.key0 + pc.tile0 * kTileKeys;
      RowState st{-INFINITY, 0.f};
      int mine = 0;   // visits of this group in this piece
      for (int i = g; i < n; i += 2, ++mine, ++n_vis) {
        const uint32_t vs = (fill + 2 * i + 1) % Cfg::kSlots;   // V's place in the ring
        const int key = key_first + i * kTileKeys;
        if (lane == 0) {
          mbar_wait_lim((Cfg::kHalves ? bar_s2 : bar_s) + 8 * g, n_vis & 1, abort_flag, p.status, 40 + g, limit);
          mbar_wait_lim(bar_full + 8 * vs, ((fill + 2 * i + 1) / Cfg::kSlots) & 1, abort_flag, p.status, 42, limit);
        }
        __syncwarp();
        tc_fence_after();
        // Masks only where a row's limit falls into the tile or a page of it is not there.
        uint32_t allow[4];
        const uint4 there = *const_cast<const uint4*>(reinterpret_cast<volatile uint4*>(&s_valid[vs][0])) ;
        const bool masked = key + kTileKeys > lim_min || (there.x & there.y & there.z & there.w) != 0xFFFFFFFFu;
        if (masked) {
          const uint32_t valid[4] = {there.x & low_bits(lim_max - key), there.y & low_bits(lim_max - key - 32),
                                     there.z & low_bits(lim_max - key - 64), there.w & low_bits(lim_max - key - 96)};
#pragma unroll
          for (int w = 0; w < 4; ++w) allow[w] = valid[w] & low_bits(lim - key - 32 * w);
          const int quarter = warp & 3;   // key r of the tile is in word r / 32
          const uint32_t word = quarter == 0 ? valid[0] : quarter == 1 ? valid[1] : quarter == 2 ? valid[2] : valid[3];
          if (!(word >> lane & 1u)) {   // not there, or no row sees it: zero its V
#pragma unroll
            for (int c = 0; c < Cfg::kChunks; ++c) {
              uint4* at = reinterpret_cast<uint4*>(smem + Cfg::kTile * (1 + vs) + c * Cfg::kChunk + r * 128);
#pragma unroll
              for (int j = 0; j < 8; ++j) at[j] = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();
          } else if (key + r >= lim_min) {   // not every row sees it
            if (take_out_not_finite<BF16, Cfg::kChunks>(smem + Cfg::kTile * (1 + vs), r, Cfg::kChunk)) {
              s_bad[0] = 1;
              fence_async_smem();
            }
          }
        }

        float mx = -INFINITY;
#pragma unroll
        for (int h = 1; h >= 0; --h) {   // (halves: the last 64 keys' scores are there first)
          if (Cfg::kHalves && h == 0) {
            if (lane == 0) mbar_wait_lim(bar_s + 8 * g, n_vis & 1, abort_flag, p.status, 58 + g, limit);
            __syncwarp();
            tc_fence_after();
          }
          float s[64];
          load_scores64(tS + 64 * h, s);
          if constexpr (SOFTCAP) {
            // The largest score decides the form of the row's soft-cap: not one that the row does not see, of a key that was never
            // loaded even.
            if (masked) zero_not_allowed64(allow[2 * h], allow[2 * h + 1], s);
            soft_cap_scores(s, cap_in, cap_out);
          }
          if (masked) apply_allow64(allow[2 * h], allow[2 * h + 1], s);
          if constexpr (SOFTCAP) {
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(s[32 * c + j]);
              tmem_st32(tS + 64 * h + 32 * c, w);
            }
          }
          mx = fmaxf(mx, row_max64(s));
        }
        if constexpr (SOFTCAP) tc_wait_st();
        const float alpha = softmax_update(st, mx, scale_log2, kLazyLog2);
        if (mine > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.f)) rescale_o<D>(tO, alpha);
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float s[64];
          uint32_t pk[32];
          load_scores64(tS + 64 * h, s);
          if (Cfg::kHalves && h == 1) {   // the next scores may go over these
            tc_fence_before();
            mbar_arrive(bar_e + 8 * g);
          }
          if (!SOFTCAP && masked) apply_allow64(allow[2 * h], allow[2 * h + 1], s);
          sum += exp_and_pack_n<BF16, 0, 1, 64>(s, st.M, scale_log2, inv_scale_log2, pk);
          tmem_st32(tS + 32 * h, pk);
          if (h == 0) {   // the product over the first 64 keys runs under the second half's exponentials
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(bar_h + 8 * g);
          }
        }
        st.l = st.l * alpha + sum;
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p + 8 * g);
      }
      fill += 2 * n;

      // ---- the groups' halves of the piece, added up in shared memory 32 (head_dim 64: 16) columns at a time and written
      // out row by row, so that a warp's stores are whole lines ----
      if (mine > 0) {
        if (lane == 0) mbar_wait_lim(bar_o + 8 * g, n_pieces & 1, abort_flag, p.status, 44 + g, limit);
        __syncwarp();
        tc_fence_after();
        ++n_pieces;
      }
      s_m[128 * g + r] = st.M;
      s_l[128 * g + r] = st.l;
      softmax_sync();   // (also: every score of the piece is read, its queries are not needed any more)
      bool taken_out = s_bad[0] != 0;
      const float mo = s_m[128 * (1 - g) + r], lo = s_l[128 * (1 - g) + r];
      const float top = lim > 0 ? fmaxf(st.M, mo) : -INFINITY, at = top == -INFINITY ? 0.f : top;
      float f = ex2_approx(st.M - at);
      const float sum = lim > 0 ? st.l * f + lo * ex2_approx(mo - at) : 0.f;
      const bool any = !(sum == 0.f);   // NaN shows
      const long long share_no = *reinterpret_cast<volatile long long*>(&s_piece->share);
      float* share = share_no >= 0 ? share_at(p, how, share_no, d_real) : nullptr;
      const int rows_here = min(kWideRows, *reinterpret_cast<volatile int*>(&s_piece->rows) - *reinterpret_cast<volatile int*>(&s_piece->rt) * kWideRows);
      if (share == nullptr) f *= 1.f / sum;
      const bool have = mine > 0 && any;
      constexpr int C = D / 4, Q4 = C / 4;   // columns of a round, 16-byte pieces of a row
      float4* xchg = reinterpret_cast<float4*>(smem);   // [2][128][Q4], pieces of a row spread over the banks
#pragma unroll 1   // code that runs once comes at about 7 cycles an instruction: little of it counts
      for (int round = 0; round * C < d_real; ++round) {
        float o[C];
        if (mine > 0) {
          tmem_ld_cols<C>(tO + round * C, o);
          float2 z[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int j = 0; j < C / 2; ++j) z[j & 1] = __ffma2_rn(make_float2(o[2 * j], o[2 * j + 1]), make_float2(0.f, 0.f), z[j & 1]);
          const float all = z[0].x + z[0].y + z[1].x + z[1].y;
          if (all != all && sum == sum) s_bad[1] = 1;
        }
#pragma unroll
        for (int j = 0; j < Q4; ++j) {
          xchg[(128 * g + r) * Q4 + (j ^ (r & (Q4 - 1)))] =
              have ? make_float4(o[4 * j] * f, o[4 * j + 1] * f, o[4 * j + 2] * f, o[4 * j + 3] * f) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        softmax_sync();
        if (tid == 0) s_bad[0] = 0;   // everyone has read it, nobody sets it before the next piece
        taken_out |= s_bad[1] != 0;
#pragma unroll
        for (int i = 0; i < 128 * Q4 / 256; ++i) {
          const int item = tid + 256 * i, rr = item / Q4, j = item % Q4;
          if (rr < rows_here) {
            const float4 a = xchg[rr * Q4 + (j ^ (rr & (Q4 - 1)))], b = xchg[(128 + rr) * Q4 + (j ^ (rr & (Q4 - 1)))];
            const float4 v = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
            if (share != nullptr) {
              *reinterpret_cast<float4*>(share + rr * d_real + round * C + 4 * j) = v;
            } else {
              *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + static_cast<long long>(s_out[rr]) * d_real + round * C + 4 * j) =
                  make_uint2(pack2<BF16>(v.x, v.y), pack2<BF16>(v.z, v.w));
            }
          }
        }
        softmax_sync();   // the next round, or the next piece's queries, go over what was read
      }
      if (tid == 0) s_bad[1] = 0;   // as above
      if (taken_out) {
        const Piece whole = *s_piece;
        const int half = d_real / 2;
        write_not_finite<BF16>(p, whole, key_first, min(lim_max, whole.key0 + whole.tile1 * kTileKeys), r < rows_here ? lim : 0, d_real, g * half, (g + 1) * half,
                               share != nullptr ? share + r * d_real : nullptr,
                               static_cast<uint16_t*>(p.out) + static_cast<long long>(s_out[r]) * d_real, reinterpret_cast<volatile uint32_t*>(smem));
      }
      if (r < rows_here && g == 0) {
        if (share != nullptr) {
          share[kWideRows * d_real + r] = top;
          share[kWideRows * d_real + kWideRows + r] = sum;
        } else if (p.lse != nullptr) {
          p.lse[s_out[r]] = any ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // =========================== TMA ============================================================
      while (st.alive && walk.next(p, pc)) ring.stream(p, &tmK, &tmV, pc, pc.tile1, st, 46);
    } else if (warp == 9 && elect_one()) {
      // =========================== MMA issuer =====================================================
      constexpr int fmt = BF16 ? 1 : 0;
      constexpr uint32_t idesc_qk = umma_idesc_f16(128, Cfg::kHalves ? 64 : 128, fmt, 0), idesc_pv = umma_idesc_f16(128, D, fmt, 1);
      constexpr uint32_t hi = umma_desc_hi_sw128(1024);
      constexpr uint32_t kSlot = Cfg::kTile >> 4, kChunk = Cfg::kChunk >> 4;
      const uint32_t q0 = umma_desc_lo(sQ, 16), k0 = umma_desc_lo(sRing, 16), v0 = umma_desc_lo(sRing, Cfg::kChunk);
      uint32_t fill = 0, n_piece = 0, n_p[2] = {0, 0};
      bool alive = true;
      while (alive && walk.next(p, pc)) {
        const int n = pc.tile1 - pc.tile0;
        alive = mbar_wait_lim(bar_q, n_piece & 1, abort_flag, p.status, 50, limit);
        ++n_piece;
        tc_fence_after();
        auto scores = [&](int i, int half) {   // S_g = Q K^T of visit i; kHalves: the keys 64 * half .. of it, the upper half first
          const uint32_t f = fill + 2 * i, s = f % Cfg::kSlots;
          if (!Cfg::kHalves || half == 1) alive = alive && mbar_wait_lim(bar_full + 8 * s, (f / Cfg::kSlots) & 1, abort_flag, p.status, 51, limit);
          if (!alive) return;
          tc_fence_after();
          const uint32_t d = tmem + 128 * (i & 1) + 64 * half, kd = k0 + s * kSlot + half * 512;   // 64 rows = 8192 bytes
          umma_ss_lo<false>(d, q0, kd, hi, idesc_qk);
#pragma unroll
          for (int k = 1; k < D / 16; ++k) {
            const uint32_t off = (k / 4) * kChunk + (k % 4) * 2;
            umma_ss_lo<true>(d, q0 + off, kd + off, hi, idesc_qk);
          }
          if (half == 0) tc_commit(bar_empty + 8 * s);
          tc_commit((half == 0 ? bar_s : bar_s2) + 8 * (i & 1));
        };
        for (int i = 0; i < min(n, 2); ++i) {
          if (Cfg::kHalves) scores(i, 1);
          scores(i, 0);
        }
        for (int i = 0; alive && i < n; ++i) {
          const int g = i & 1;
          const uint32_t f = fill + 2 * i + 1, s = f % Cfg::kSlots;
          const uint32_t par = (g == 0 ? n_p[0] : n_p[1]) & 1;
          alive = mbar_wait_lim(bar_h + 8 * g, par, abort_flag, p.status, 52 + g, limit) &&
                  mbar_wait_lim(bar_full + 8 * s, (f / Cfg::kSlots) & 1, abort_flag, p.status, 54, limit);
          if (!alive) break;
          if (g == 0) {
            ++n_p[0];
          } else {
            ++n_p[1];
          }
          tc_fence_after();
          const uint32_t d = tmem + 256 + D * g, a = tmem + 128 * g, vd = v0 + s * kSlot;
          umma_ts_lo(d, a, vd, hi, idesc_pv, i >= 2 ? 1u : 0u);
#pragma unroll
          for (int k = 1; k < 4; ++k) umma_ts_lo_acc(d, a + 8 * k, vd + k * 128, hi, idesc_pv);   // 16 keys = 2048 bytes
          if (Cfg::kHalves && i + 2 < n) {   // half of the next scores under the second half's exponentials
            alive = mbar_wait_lim(bar_e + 8 * g, par, abort_flag, p.status, 43, limit);
            if (alive) scores(i + 2, 1);
            if (!alive) break;
          }
          alive = mbar_wait_lim(bar_p + 8 * g, par, abort_flag, p.status, 56 + g, limit);
          if (!alive) break;
          tc_fence_after();
#pragma unroll
          for (int k = 4; k < 8; ++k) umma_ts_lo_acc(d, a + 8 * k, vd + k * 128, hi, idesc_pv);
          tc_commit(bar_empty + 8 * s);
          if (i + 2 >= n) tc_commit(bar_o + 8 * g);
          if (i + 2 < n) scores(i + 2, 0);
        }
        fill += 2 * n;
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {   // the same in all threads now: wait for what is in flight
    if (warp == 8) ring.drain(st);
    if (warp == 9 && elect_one()) {
      tc_commit(bar_end);
      mbar_wait_drain(bar_end, 0, kDrain);
    }
    __syncthreads();
  }
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (how.late_wait) grid_wait();
}

template <int D, bool BF16, bool SOFTCAP>
cudaError_t launch_wide_t(const CUtensorMap& tmK, const CUtensorMap& tmV, const CacheAttnParams& p, const CacheLaunch& how, int d_real,
                          cudaStream_t stream) {
  auto kern = omni_cache_wide_kernel<D, BF16, SOFTCAP>;
  static SmemAttrOnce attr_once[kMaxDevices];
  const cudaError_t e = ensure_smem_attr(kern, WideCfg<D>::kSmem, attr_once);
  if (e != cudaSuccess) return e;
  static const int regs = [kern] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (2 * kSoftmaxRegs + kOtherRegs > 3 * regs) return cudaErrorLaunchOutOfResources;
  return launch_chained(kern, how.ctas, kWideThreads, WideCfg<D>::kSmem, stream, tmK, tmV, p, how, d_real);
}

template <int D, bool BF16>
cudaError_t launch_wide_c(const CUtensorMap& tmK, const CUtensorMap& tmV, const CacheAttnParams& p, const CacheLaunch& how, int d_real,
                          cudaStream_t stream) {
  return p.softcap > 0.f ? launch_wide_t<D, BF16, true>(tmK, tmV, p, how, d_real, stream)
                         : launch_wide_t<D, BF16, false>(tmK, tmV, p, how, d_real, stream);
}

}  // namespace

// head_dim 32 is computed as 64: the TMA unit fills the missing columns with zeros.
cudaError_t launch_cache_wide(int head_dim, bool bf16, const CUtensorMap& tmK, const CUtensorMap& tmV, const CacheAttnParams& p,
                              const CacheLaunch& how, cudaStream_t stream) {
  if (head_dim == 128) {
    return bf16 ? launch_wide_c<128, true>(tmK, tmV, p, how, head_dim, stream) : launch_wide_c<128, false>(tmK, tmV, p, how, head_dim, stream);
  }
  return bf16 ? launch_wide_c<64, true>(tmK, tmV, p, how, head_dim, stream) : launch_wide_c<64, false>(tmK, tmV, p, how, head_dim, stream);
}

}  // namespace omni
