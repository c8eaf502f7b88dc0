// Attention of pieces of new tokens over a paged cache, in tiles of 128 queries and 128 keys: `tcgen05` products with TMEM accumulators,
// keys and values brought page by page by TMA.  The formula stands with the kernels for pieces of a few tokens (paged.cu).
//
// Three kernels.  A plan (one CTA; others clear the rows that get no result).  The attention itself, persistent: an item is a head's tile of
// queries against its visible tiles of keys.  Where these are fewer than two an SM, the CTAs share all key tiles equally instead, and what they have of a tile that is
// not theirs alone goes to memory.  A join of such parts, where there may be some.
#include "decode_common.cuh"
#include "paged.cuh"

namespace bones {

constexpr int PT = 128;                          // tile edge
constexpr uint32_t PATOM = PT * 64 * 2;          // one 128-byte-swizzled atom of [128 rows][64 columns]; a tile has D / 64

struct PiecesArgs {
  Paged p;
  float c1, c2;               // scale log2 e, |scale| D log2 e
  int window_tiles;
  const int* doc_start;       // [N] or null
  __nv_bfloat16* y;           // [N, H * D]
  int* err;
  int* next;                  // items drawn
  int* tiles;                 // [B + 1]: tiles of queries, heads' one after another, of the sequences before
  long long* before;          // [B + 1]: what the sequences before count for, in tiles of keys; behind that a CTA's share, 0 where items are drawn
  float* parts;               // [slots][D][128], and behind them [slots][128] sums of weights: two places a CTA, of the tile that its share begins in and of
                              // the one that it ends in
  int slots, sms, row_bytes;
};

// ---------------------------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------------------------
constexpr int PLAN_T = 256;

constexpr int PIECE_WAY = 2;                     // tiles of keys that a tile of queries' way in and out counts for
constexpr int PIECE_LEAST = 4;                   // tiles of keys that are worth a part
constexpr int PIECE_JOIN = 6;                    // tiles of keys that the join takes as long as

// Tiles of keys of a piece's tile of queries, documents apart, and of all in front of one, with their ways
__device__ __forceinline__ int plan_tiles(const PiecesArgs& a, const Piece& s, int qt) {
  const int last = (s.pos + min(s.live, (qt + 1) * PT) - 1) >> 7;
  return a.window_tiles > 0 ? min(last + 1, a.window_tiles + 1) : last + 1;
}
__device__ __forceinline__ long long plan_front(const PiecesArgs& a, const Piece& s, int qt) {
  long long n = 0;
  for (int i = 0; i < qt; ++i) n += plan_tiles(a, s, i) + PIECE_WAY;
  return n;
}
// Sums of `v` over the threads in front; the total in *all.
__device__ __forceinline__ long long plan_scan(long long v, long long* box, long long* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += x;
  }
  if (lane == 31) box[warp] = up;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < PLAN_T / 32; ++w) {
    const long long x = box[w];
    if (w < warp) before += x;
    total += x;
  }
  __syncthreads();
  *all = total;
  return before + up - v;
}

__global__ void __launch_bounds__(PLAN_T) paged_plan_kernel(const PiecesArgs a) {
  __shared__ long long box[PLAN_T / 32];
  __shared__ int longest;
  const Paged& p = a.p;
  pdl_wait();
  pdl_launch();
  if (blockIdx.x > 0) {                          // rows without a result: outside all pieces, or left out
    const int lane = threadIdx.x & 31;
    for (int row = (blockIdx.x - 1) * (PLAN_T / 32) + (threadIdx.x >> 5); row < p.N; row += (gridDim.x - 1) * (PLAN_T / 32)) {
      const int b = paged_owner(p.starts, p.B, row);
      if (b >= 0 && b < p.B) {
        const Piece s = paged_piece(p, b);
        if (row - s.row >= 0 && row - s.row < s.live) continue;
      }
      for (int i = lane * 16; i < a.row_bytes; i += 512) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(a.y) + (long long)row * a.row_bytes + i) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  long long tiles = 0, total = 0;
  if (threadIdx.x == 0) longest = 0;
  __syncthreads();
  for (int b0 = 0; b0 < p.B; b0 += PLAN_T) {
    const int b = b0 + threadIdx.x;
    long long rows = 0, n = 0;
    if (b < p.B) {
      const Piece x = paged_piece(p, b);
      if (x.live) {
        rows = (x.live + PT - 1) / PT;
        n = a.slots > 0 ? plan_front(a, x, (int)rows) * p.H : 0;
        if (a.slots > 0) atomicMax(&longest, plan_tiles(a, x, (int)rows - 1) + PIECE_WAY);
        rows *= p.H;
      }
    }
    long long more, all;
    const long long at = tiles + plan_scan(rows, box, &more), in_front = total + plan_scan(n, box, &all);
    if (b < p.B) {
      a.tiles[b] = (int)at;
      a.before[b] = in_front;
    }
    tiles += more;
    total += all;
  }
  if (threadIdx.x == 0) {
    *a.next = 0;
    a.tiles[p.B] = (int)tiles;
    a.before[p.B] = total;
    // drawn, the CTAs are done when the longest tile of queries is, or half of one behind the mean
    const long long mean = (total + a.sms - 1) / a.sms, drawn = max((long long)longest, mean + longest / 2), shared = max(mean, (long long)PIECE_WAY + PIECE_LEAST);
    a.before[p.B + 1] = a.slots > 0 && tiles < 2 * a.sms && shared + PIECE_JOIN < drawn ? shared : 0;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------------------------
// Roles as in the training forward (attention.cu): a warp each for Q and K loads, V loads, S = Q K^T, O += P V; sixteen softmax warps (four per
// 32-lane TMEM quadrant, 32 keys a thread); four drain warps.  Here a warp of its own draws the items and looks up what they are (the sequence, its
// rows, the first and last of their keys): three dependent reads that nobody waits for, since it runs ahead.  What is of this kernel:
//  - pages: a box of the tensor map is one page's P tokens of one head; a position without a page is loaded as zeros and masked.
//  - rows behind a piece's end (a step with a few drafts has 5 of 128) take no exponentials: a softmax warp without a live row passes its tiles on.
//  - values that a row does not see may be anything (other sequences' leftovers behind the end): tiles with a mask are looked through before V's
//    product by two warps, zeros are put for what is not finite, and it is added back to the rows that do see it at the end.  (By the drain warps they waited for an
//    item's output, by the loading warp for its loads: 31 us for 26 of the banded case of short pieces.)
//  - a stage of Q, three of K and of V: the next item's queries come while the softmax still has two or three tiles of this one's (two stages of Q and of K
//    99.4 and 50.2 us in the first two cases below).
// Measured, us of a whole call: 8 prompts of 2048 tokens, 10 heads of 128, 91.7 (86 GFLOP at 0.94 PFLOP/s); 512 tokens behind 15900, 10 heads of 128, 48.5 (0.87); 24 pieces
// of up to 700 tokens, 4 heads of 64, window 512, documents, 21.8.  A tile takes about 1850 clocks, at about 1.7 GHz: 1024 of
// exponentials by sixteen warps (16384 at 16 a clock and SM), some 400 between two tiles' (barriers, TMEM), an item's way in and out 3000 once.  The tensor pipe is
// active 0.56 of the time; shared memory moves 160 KB a tile (Q and K read for S, V for O, both written by TMA), 1280 clocks at 128 bytes each; L2 delivers half of what
// it can (half as many bytes again: 4 % longer).  CTA pairs with half of each tile of K and V apiece would take 96 KB.  Calls without a pause between them settle at a lower
// clock: 110 (0.78 PFLOP/s), 56 and 22 us.  Slower, us in the first case: two halves of the softmax warps on
// alternate tiles 93.8 (for 91.7), a sixth or a third of the exponentials by a polynomial 108 or 117 (of 104.6 then), two accumulators and two S buffers instead of one and
// three 108.6.  (The order in which items are drawn and how far ahead: 104.6 with a head's tiles in turn and an item ahead, 94.8 as it is; the
// mask as bits, 94.8 -> 92.9, and 24.0 -> 21.8 in the third, where most tiles have one; with the exponentials left out that no row sees 94.9, 50.9 and 21.4.)
constexpr int PP_SW = 16, PP_DW = 4;
constexpr int PP_PV = 2 + PP_SW + PP_DW, PP_VW = PP_PV + 1, PP_IW = PP_VW + 1, PP_LW = PP_IW + 1, PP_LOOK = 2;
constexpr int PP_THREADS = 32 * (PP_LW + PP_LOOK);
constexpr int PP_RING = 2;                      // items handed round: the one being computed and the next (three: the same times)
constexpr int PP_NEAR = 5;                      // tiles of keys from an item's end at which the next is drawn (whole prompts, us: 98.0 / 96.8 / 95.7 / 94.8 / 95.0 / 95.3 / 95.5
                                                // with 1 / 2 / 3 / 5 / 7 / 9 / 12; 97.5 an item ahead)
constexpr uint32_t PP_BARS = 512;               // barriers, TMEM address, abort flag, items

struct PieceItem {
  int row0, live, pos0, h;                      // first row, rows, position of the first
  int kt0, n, seq, place;                       // first key tile, tiles; place of its sums or -1
  int far, none;                                // the last of its rows' first keys; `none`: a part without a tile (its one tile is masked)
};

template <int D>
__global__ void __launch_bounds__(PP_THREADS, 1)
paged_pieces_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PiecesArgs a) {
  constexpr uint32_t TILE = (D / 64) * PATOM;
  const Paged& p = a.p;
  if (threadIdx.x == 32 * PP_VW) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  extern __shared__ __align__(1024) uint8_t gen[];
  const uint32_t base = smem_u32(gen);
  if (base & 1023u) {                           // the swizzled tiles want it
    pdl_wait();
    if (threadIdx.x == 0) atomicCAS(a.err, 0, ERR_WAIT_AUX);
    return;
  }
  const uint32_t sQ = base;
  auto sK = [&](int s) { return base + TILE * (1 + s); };
  auto sV = [&](int s) { return base + TILE * (4 + s); };
  constexpr uint32_t kBars = TILE * 7;
  const uint32_t bars = base + kBars;
  const uint32_t q_full = bars, q_free = bars + 8u;
  auto k_full = [&](int s) { return bars + 8u * (2 + s); };
  auto k_free = [&](int s) { return bars + 8u * (5 + s); };
  auto v_full = [&](int s) { return bars + 8u * (8 + s); };
  auto v_free = [&](int s) { return bars + 8u * (11 + s); };
  auto v_fine = [&](int s) { return bars + 8u * (14 + s); };
  auto s_full = [&](int s) { return bars + 8u * (17 + s); };
  auto s_free = [&](int s) { return bars + 8u * (20 + s); };
  auto p_full = [&](int s) { return bars + 8u * (23 + s); };
  auto i_full = [&](int s) { return bars + 8u * (26 + s); };
  auto i_free = [&](int s) { return bars + 8u * (29 + s); };
  const uint32_t o_full = bars + 8u * 32, o_free = bars + 8u * 33, l_full = bars + 8u * 34, l_free = bars + 8u * 35;
  const uint32_t near = bars + 8u * 36;         // an item's end is near
  const uint32_t tmem_slot = bars + 296u;
  volatile uint32_t* tmem_slot_g = reinterpret_cast<volatile uint32_t*>(gen + kBars + 296);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kBars + 300);
  int* taint = reinterpret_cast<int*>(gen + kBars + 304);                                    // [PP_RING]
  volatile int* holes = reinterpret_cast<volatile int*>(gen + kBars + 448);                  // [8], by tile: whether a page that it needs is missing
  PieceItem* ring = reinterpret_cast<PieceItem*>(gen + kBars + 320);                         // [PP_RING]
  static_assert(PP_RING <= 3 && 320 + PP_RING * sizeof(PieceItem) <= 448 && 448 + 8 * 4 <= PP_BARS, "room");
  float* lsum = reinterpret_cast<float*>(gen + kBars + PP_BARS);                             // [4 column parts][128 rows]

  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int A = p.H * D;
  if (warp == 0) {
    for (int i = lane; i < 37; i += 32) {
      const bool by_softmax = (i >= 23 && i < 26) || i == 34, by_drain = (i >= 29 && i < 32) || i == 33 || i == 35, by_look = i >= 14 && i < 17;
      mbar_init(bars + 8u * (uint32_t)i, by_softmax ? PP_SW : by_drain ? PP_DW : by_look ? PP_LOOK : 1);
    }
    if (lane == 0) *abort_flag = 0;
    fence_barrier_init();
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)warp_uniform((int)*tmem_slot_g);
  pdl_wait();                                   // the plan
  pdl_launch();                                 // (the join reads it ahead of its own wait)
  auto tS = [&](int s) { return tmem + (uint32_t)s * 128u; };
  const uint32_t tO = tmem + 384u;
  // the it-th item of this CTA; false behind the last one
  auto take = [&](int it, PieceItem* im) {
    if (!__all_sync(0xffffffffu, mbar_wait(i_full(it % PP_RING), (uint32_t)(it / PP_RING & 1), abort_flag, a.err, ERR_WAIT_AUX))) return false;
    *im = ring[it % PP_RING];
    return warp_uniform(im->n) > 0;
  };
  // whether some row of the item does not see some key of the tile
  auto masked = [&](const PieceItem& im, int kt) { return kt * PT + PT - 1 > im.pos0 || kt * PT < im.far || im.none; };
  const int per_tile = PT >> p.shift;           // pages of a tile
  // row of the tensor map of lane i's page of tile kt (lanes below per_tile); behind the map, which reads as zeros, where there is none
  const int none = (int)(((long long)p.pages * p.H) << p.shift);
  auto page_row = [&](const PieceItem& im, int kt) {
    const int i = kt * per_tile + lane;
    int row = none;
    if (lane < per_tile && i < p.M && (i << p.shift) < im.pos0 + im.live) {
      const long long at = paged_at(p, p.table[im.seq * p.ldt + i], im.h);
      if (at >= 0) row = (int)at;
    }
    return row;
  };
  const uint32_t page_bytes = 128u << p.shift;  // of a column half

  if (warp == PP_IW) {
    // The items, in sequence- and head-major order, so that CTAs at work at one time share keys and values through L2: drawn, or what a share of all
    // tiles of keys has of them.
    const long long share = a.before[p.B + 1], total = share ? a.before[p.B] : a.tiles[p.B];
    long long at = (long long)blockIdx.x * share;
    const long long stop = min(at + share, total);
    for (int it = 0;; ++it) {
      int b = -1, g = 0, from_v = 0, to_v = 0, all_v = 0;           // the sequence, its tile of queries, and which of the tiles of keys that it counts for
      if (share) {
        while (at < stop && to_v <= from_v) {
          b = min(max(paged_owner(a.before, p.B, at), 0), p.B - 1);
          const Piece s = paged_piece(p, b);
          const int rows = (s.live + PT - 1) / PT;
          const long long head = plan_front(a, s, rows), in_seq = at - a.before[b];
          long long off_v = in_seq % head;
          int qt = 0;
          all_v = plan_tiles(a, s, 0);
          while (off_v >= all_v + PIECE_WAY) {
            off_v -= all_v + PIECE_WAY;
            all_v = plan_tiles(a, s, ++qt);
          }
          const int off = (int)off_v;
          const int take = (int)min((long long)(all_v + PIECE_WAY - off), stop - at);
          at += take;
          g = (int)(in_seq / head) * rows + qt;
          from_v = max(off - PIECE_WAY, 0);
          to_v = off + take - PIECE_WAY;
        }
        if (to_v <= from_v) b = -1;
      } else {
        // (an item drawn a whole item ahead would be a CTA's own while others have nothing left)
        if (it >= 1 && !__all_sync(0xffffffffu, mbar_wait(near, (uint32_t)((it - 1) & 1), abort_flag, a.err, ERR_WAIT_AUX))) break;
        const int w = it == 0 ? (int)blockIdx.x : (int)gridDim.x + warp_uniform(lane == 0 ? atomicAdd(a.next, 1) : 0);
        if (w < total) {
          b = min(max(paged_owner(a.tiles, p.B, w), 0), p.B - 1);
          g = w - a.tiles[b];
          to_v = all_v = 1;
        }
      }
      PieceItem im = {};
      if (b >= 0) {
        const Piece s = paged_piece(p, b);
        const int rows = (s.live + PT - 1) / PT;
        im.seq = b;
        // shared: a head's tiles one after another; drawn: the heads' last tiles first, which see the most keys, so that what is drawn last is short
        im.h = share ? g / rows : g % p.H;
        const int qt = share ? g % rows : rows - 1 - g / p.H;
        im.row0 = s.row + qt * PT;
        im.live = min(PT, s.live - qt * PT);
        im.pos0 = s.pos + qt * PT;
        im.place = to_v - from_v < all_v ? 2 * (int)blockIdx.x + (from_v == 0) : -1;
        int lo = 0x7fffffff, hi = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = lane + 32 * i;
          if (row < im.live) {
            int x = a.doc_start ? max(a.doc_start[im.row0 + row], 0) : 0;
            if (a.window_tiles > 0) x = max(x, (((im.pos0 + row) >> 7) - (a.window_tiles - 1)) * 128);
            lo = min(lo, x);
            hi = max(hi, x);
          }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        im.far = __reduce_max_sync(0xffffffffu, hi);
        const int last = (im.pos0 + im.live - 1) >> 7, first = min(lo >> 7, last), n = last - first + 1;
        const int from = (int)((long long)from_v * n / all_v), to = (int)((long long)to_v * n / all_v);
        im.none = to <= from;
        im.kt0 = im.none ? last : first + from;
        im.n = im.none ? 1 : to - from;
      }
      const int slot = it % PP_RING;
      if (it >= PP_RING && !__all_sync(0xffffffffu, mbar_wait(i_free(slot), (uint32_t)((it / PP_RING - 1) & 1), abort_flag, a.err, ERR_WAIT_EMPTY))) break;
      if (lane == 0) {
        ring[slot] = im;
        taint[slot] = 0;
        mbar_arrive(i_full(slot));
      }
      __syncwarp();
      if (im.n == 0) break;
    }
  } else if (warp == 0) {
    // Q and K loads
    PieceItem im;
    int g = 0, ks = 0;
    uint32_t kph = 1;
    bool dead = false;
    for (int it = 0; !dead && take(it, &im); ++it) {
      if (it >= 1 && !dead) dead = !mbar_wait(q_free, (uint32_t)((it - 1) & 1), abort_flag, a.err, ERR_WAIT_EMPTY);
      const int h = warp_uniform(im.h), row0 = warp_uniform(im.row0);
      if (elect_one() && !dead) {
        mbar_arrive_expect_tx(q_full, TILE);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_load_2d(sQ + c * PATOM, &tm_q, q_full, h * D + c * 64, row0);
      }
      int row = page_row(im, im.kt0);
      for (int j = 0; j < im.n; ++j, ++g) {
        const int now = row;
        if (j + 1 < im.n) row = page_row(im, im.kt0 + j + 1);
        if (g >= 3 && !dead) dead = !mbar_wait(k_free(ks), kph, abort_flag, a.err, ERR_WAIT_EMPTY);
        // (at most six tiles are between this one and the oldest whose scores are still read)
        const uint32_t missing = __ballot_sync(0xffffffffu, lane < per_tile && now == none && ((im.kt0 + j) * per_tile + lane) << p.shift < im.pos0 + im.live);
        if (lane == 0) holes[g & 7] = (int)missing;
        if (elect_one() && !dead) mbar_arrive_expect_tx(k_full(ks), TILE);
        __syncwarp();
        for (int i = 0; i < per_tile; ++i) {
          const int at = __shfl_sync(0xffffffffu, now, i);
          if (elect_one() && !dead) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_2d(sK(ks) + c * PATOM + i * page_bytes, &tm_k, k_full(ks), c * 64, at);
          }
        }
        if (++ks == 3) { ks = 0; kph ^= 1u; }
        if (j == max(im.n - PP_NEAR, 0) && lane == 0) mbar_arrive(near);
      }
    }
  } else if (warp == PP_VW) {
    // V loads
    PieceItem im;
    int g = 0, vs = 0;
    uint32_t vph = 1;
    bool dead = false;
    for (int it = 0; !dead && take(it, &im); ++it) {
      int row = page_row(im, im.kt0);
      for (int j = 0; j < im.n; ++j, ++g) {
        const int now = row;
        if (j + 1 < im.n) row = page_row(im, im.kt0 + j + 1);
        if (g >= 3 && !dead) dead = !mbar_wait(v_free(vs), vph, abort_flag, a.err, ERR_WAIT_EMPTY);
        if (elect_one() && !dead) mbar_arrive_expect_tx(v_full(vs), TILE);
        __syncwarp();
        for (int i = 0; i < per_tile; ++i) {
          const int at = __shfl_sync(0xffffffffu, now, i);
          if (elect_one() && !dead) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_2d(sV(vs) + c * PATOM + i * page_bytes, &tm_v, v_full(vs), c * 64, at);
          }
        }
        if (++vs == 3) { vs = 0; vph ^= 1u; }
      }
    }
  } else if (warp >= PP_LW) {
    // Tiles of V in which some row sees only some of the keys are looked through, half by either warp.  Every tile is passed on from here, so that no
    // phase of a stage goes by unseen (a wait tells apart two phases, not three).
    const int half = warp - PP_LW;
    PieceItem im;
    int vs = 0;
    uint32_t vph = 0;
    bool ok = true;
    for (int it = 0; ok && take(it, &im); ++it) {
      for (int kt = im.kt0; kt < im.kt0 + im.n; ++kt) {
        if (!__all_sync(0xffffffffu, mbar_wait(v_full(vs), vph, abort_flag, a.err, ERR_WAIT_FULL))) { ok = false; break; }
        if (masked(im, kt)) {
          constexpr int ROUNDS = (int)(TILE / 512 / PP_LOOK);
          uint4* tile = reinterpret_cast<uint4*>(gen + TILE * (4 + vs)) + half * ROUNDS * 32 + lane;
          // the largest magnitude of each half: an infinity is larger than the finite, a NaN stays
          __nv_bfloat162 most[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) most[k] = __float2bfloat162_rn(0.f);
#pragma unroll 8
          for (int i = 0; i < ROUNDS; ++i) {
            const uint4 u = tile[i * 32];
            const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
            for (int k = 0; k < 4; ++k) most[k] = __hmax2_nan(most[k], __habs2(x[k]));
          }
#pragma unroll
          for (int k = 1; k < 4; ++k) most[0] = __hmax2_nan(most[0], most[k]);
          const uint32_t top = *reinterpret_cast<const uint32_t*>(&most[0]);
          if (__any_sync(0xffffffffu, (top & 0x7f80u) == 0x7f80u || (top & 0x7f800000u) == 0x7f800000u)) {
            bool seen = false;
            for (int i = 0; i < ROUNDS; ++i) {
              const uint4 u = tile[i * 32];
              uint32_t w[4] = {u.x, u.y, u.z, u.w};
              bool any = false;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const bool low = (w[k] & 0x7f80u) == 0x7f80u, high = (w[k] & 0x7f800000u) == 0x7f800000u;
                any = any || low || high;
                if (low) w[k] &= 0xffff0000u;
                if (high) w[k] &= 0xffffu;
              }
              if (any) {
                tile[i * 32] = make_uint4(w[0], w[1], w[2], w[3]);
                if (kt * PT + (((half * ROUNDS * 32 + lane + i * 32) * 16 >> 7) & (PT - 1)) < im.pos0 + im.live) seen = true;        // not a leftover behind the end
              }
            }
            if (__any_sync(0xffffffffu, seen) && lane == 0) atomicOr(&taint[it % PP_RING], 1);
            fence_proxy_async_smem();
            __threadfence_block();
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(v_fine(vs));
        if (++vs == 3) { vs = 0; vph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // S = Q K^T of each tile, into the buffer whose O += P V (three tiles before) is done
    constexpr uint32_t kHi = umma_desc_hi(1024, kLayoutSw128);
    const uint32_t idesc_s = umma_idesc_f16(128, 128, 1, 0, 0);   // Q (K-major) x K (K-major)
    const uint32_t q_lo = (uint32_t)warp_uniform((int)umma_desc_lo(sQ, 0)), k_lo = (uint32_t)warp_uniform((int)umma_desc_lo(sK(0), 0));
    PieceItem im;
    bool dead = false;
    int g = 0, gs = 0;                       // tile; S buffer and K stage
    uint32_t fph = 1, kph = 0;
    for (int it = 0; !dead && take(it, &im); ++it) {
      const int n = warp_uniform(im.n);
      if (!dead) dead = !mbar_wait(q_full, (uint32_t)(it & 1), abort_flag, a.err, ERR_WAIT_FULL);
      for (int j = 0; j < n; ++j, ++g) {
        if (!dead) dead = !mbar_wait(k_full(gs), kph, abort_flag, a.err, ERR_WAIT_FULL);
        if (g >= 3 && !dead) dead = !mbar_wait(s_free(gs), fph, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
        tc_fence_after();
        const uint32_t kd = k_lo + (uint32_t)gs * (TILE >> 4), sd = tS(gs);
        if (elect_one() && !dead) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = ((k >> 2) * PATOM + (k & 3) * 32) >> 4;
            umma_f16_lh(sd, q_lo + off, kHi, kd + off, kHi, idesc_s, k ? 1u : 0u);
          }
          tc_commit(s_full(gs));
          tc_commit(k_free(gs));
          if (j == n - 1) tc_commit(q_free);
        }
        if (++gs == 3) {
          gs = 0;
          fph ^= 1u;
          kph ^= 1u;
        }
      }
    }
  } else if (warp == PP_PV) {
    // O += P V; P(g) lies in TMEM as packed bf16 pairs over the S(g) columns that it was computed from
    constexpr uint32_t kHi = umma_desc_hi(1024, kLayoutSw128);
    const uint32_t idesc_o = umma_idesc_f16(128, D, 1, 0, 1);   // P (TMEM) x V (MN-major)
    const uint32_t v_lo = (uint32_t)warp_uniform((int)umma_desc_lo(sV(0), PATOM));
    PieceItem im;
    bool dead = false;
    int ps = 0;                              // P buffer and V stage
    uint32_t pph = 0;
    for (int it = 0; !dead && take(it, &im); ++it) {
      const int n = warp_uniform(im.n);
      for (int j = 0; j < n; ++j) {
        if (!dead) dead = !mbar_wait(v_fine(ps), pph, abort_flag, a.err, ERR_WAIT_FULL);
        if (j == 0 && it >= 1 && !dead) dead = !mbar_wait(o_free, (uint32_t)((it - 1) & 1), abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
        if (!dead) dead = !mbar_wait(p_full(ps), pph, abort_flag, a.err, ERR_WAIT_AUX);
        tc_fence_after();
        const uint32_t vd = v_lo + (uint32_t)ps * (TILE >> 4), pd = tS(ps);
        if (elect_one() && !dead) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts_lh(tO, pd + (uint32_t)((k >> 1) * 32 + (k & 1) * 8), vd + (uint32_t)((k * 2048) >> 4), kHi, idesc_o, (j == 0 && k == 0) ? 0u : 1u);
          tc_commit(s_free(ps));
          tc_commit(v_free(ps));
          if (j == n - 1) tc_commit(o_full);
        }
        if (++ps == 3) { ps = 0; pph ^= 1u; }
      }
    }
  } else if (warp < 2 + PP_SW) {
    // Softmax: a thread has one query row and 32 of the tile's 128 keys
    const int q = warp & 3, part = (warp - 2) >> 2;
    const int r = q * 32 + lane, c0 = part * 32;
    const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
    PieceItem im;
    int gs = 0, g = 0;
    uint32_t sph = 0;
    bool ok = true;
    for (int it = 0; ok && take(it, &im); ++it) {
      const bool idle = q * 32 >= im.live;       // none of this warp's rows is one
      // rows behind the piece's end are not stored: no mask either
      const int qpos = r >= im.live ? 0x3fffffff : im.none ? -1 : im.pos0 + r;
      int lo = 0;
      if (r < im.live) {
        if (a.doc_start) lo = max(a.doc_start[im.row0 + r], 0);
        if (a.window_tiles > 0) lo = max(lo, (((im.pos0 + r) >> 7) - (a.window_tiles - 1)) * 128);
      }
      float l = 0.f;
      for (int j = 0; j < im.n; ++j, ++g) {
        const int k0 = (im.kt0 + j) * PT + c0;
        const bool got = mbar_wait(s_full(gs), sph, abort_flag, a.err, ERR_WAIT_TMEM_FULL);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
        tc_fence_after();
        if (!idle) {
          uint32_t v0[32], pk[16];
          __syncwarp();
          BONES_TMEM_LD32(tS(gs) + lane_addr + (uint32_t)c0, v0);
          tmem_ld_wait();
          float e[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float x = fmaf(__uint_as_float(v0[i]), a.c1, -a.c2);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i]) : "f"(x));
          }
          const int missing = holes[g & 7];
          if (__any_sync(0xffffffffu, (k0 + 31 > qpos) || (k0 < lo) || missing)) {
            const int end = qpos - k0, from = lo - k0;
            // which of its keys the row sees
            uint32_t seen = end < 0 || from > 31 ? 0u : (0xffffffffu >> (31 - min(end, 31))) & (0xffffffffu << max(from, 0));
            // pages of the first and second sixteen keys
            if (missing >> (c0 >> p.shift) & 1) seen &= 0xffff0000u;
            if (missing >> ((c0 + 16) >> p.shift) & 1) seen &= 0xffffu;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(seen >> i & 1)) e[i] = 0.f;
          }
          float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 32; ++i) l4[i & 3] += e[i];
          l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack_bf16(e[2 * i], e[2 * i + 1]);
          BONES_TMEM_ST16(tS(gs) + lane_addr + (uint32_t)c0, pk);
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(gs));
        if (++gs == 3) { gs = 0; sph ^= 1u; }
      }
      if (!ok) break;
      if (it >= 1 && !__all_sync(0xffffffffu, mbar_wait(l_free, (uint32_t)((it - 1) & 1), abort_flag, a.err, ERR_WAIT_AUX))) break;
      lsum[part * PT + r] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(l_full);
    }
  } else {
    // Drain: a thread per query row
    const int q = warp & 3, r = q * 32 + lane;
    const uint32_t tOr = tO + ((uint32_t)(q * 32) << 16);
    PieceItem im;
    for (int it = 0; take(it, &im); ++it) {
      const bool real = r < im.live;
      bool got = mbar_wait(l_full, (uint32_t)(it & 1), abort_flag, a.err, ERR_WAIT_AUX);
      if (!__all_sync(0xffffffffu, got)) break;
      const float l = (lsum[r] + lsum[PT + r]) + (lsum[2 * PT + r] + lsum[3 * PT + r]);
      __syncwarp();
      if (lane == 0) mbar_arrive(l_free);
      const float inv = l == 0.f ? 0.f : 1.0f / l;        // a row that sees no key has zeros
      const long long col = (long long)im.h * D;
      __nv_bfloat16* y = a.y + (long long)(im.row0 + r) * A + col;
      float* part = a.parts + (long long)im.place * PT * D + r;              // columns of 128 rows: a warp's stores lie side by side
      if (im.place >= 0 && real) a.parts[(long long)a.slots * PT * D + (long long)im.place * PT + r] = l;
      got = mbar_wait(o_full, (uint32_t)(it & 1), abort_flag, a.err, ERR_WAIT_TMEM_FULL);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      const bool tainted = warp_uniform(*(volatile int*)&taint[it % PP_RING]) != 0;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t v[32];
        __syncwarp();
        BONES_TMEM_LD32(tOr + (uint32_t)c, v);
        tmem_ld_wait();
        if (c + 32 >= D) {                             // the next item's products may have the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(o_free);
        }
        if (tainted && real) {                         // rare: what the products left out
          const int* table = p.table + im.seq * p.ldt;
          const int qpos = im.pos0 + r;
          int lo = a.doc_start ? max(a.doc_start[im.row0 + r], 0) : 0;
          if (a.window_tiles > 0) lo = max(lo, ((qpos >> 7) - (a.window_tiles - 1)) * 128);
          const __nv_bfloat16* values = reinterpret_cast<const __nv_bfloat16*>(a.p.values);
          for (int j = 0; j < im.n && !im.none; ++j) {
            if (!masked(im, im.kt0 + j)) continue;
            for (int key = max((im.kt0 + j) * PT, lo); key < min((im.kt0 + j + 1) * PT, qpos + 1); ++key) {
              const long long at = paged_at(p, table[key >> p.shift], im.h);
              if (at < 0) continue;
              const __nv_bfloat16* val = values + (at + (key & ((1 << p.shift) - 1))) * D + c;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float x = __bfloat162float(val[i]);
                if (!isfinite(x)) v[i] = __float_as_uint(__uint_as_float(v[i]) + x);
              }
            }
          }
        }
        if (im.place >= 0) {
          if (real)
#pragma unroll
            for (int i = 0; i < 32; ++i) part[(c + i) * PT] = __uint_as_float(v[i]);
        } else {
          uint4 u[4];
#pragma unroll
          for (int gq = 0; gq < 4; ++gq) {
            u[gq].x = pack_bf16(__uint_as_float(v[gq * 8 + 0]) * inv, __uint_as_float(v[gq * 8 + 1]) * inv);
            u[gq].y = pack_bf16(__uint_as_float(v[gq * 8 + 2]) * inv, __uint_as_float(v[gq * 8 + 3]) * inv);
            u[gq].z = pack_bf16(__uint_as_float(v[gq * 8 + 4]) * inv, __uint_as_float(v[gq * 8 + 5]) * inv);
            u[gq].w = pack_bf16(__uint_as_float(v[gq * 8 + 6]) * inv, __uint_as_float(v[gq * 8 + 7]) * inv);
          }
          if (real) {
            st_global_v8(y + c, u[0], u[1]);
            st_global_v8(y + c + 16, u[2], u[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(i_free(it % PP_RING));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the parts of tiles of queries in their order: a CTA the four columns each of 128 rows, then the next that is its own.  (CTAs of 128 threads find room
// beside the attention's, and have looked up what they need when that ends; where nothing is shared they leave at once.)
template <int D>
__global__ void __launch_bounds__(PT) paged_pieces_join_kernel(const PiecesArgs a) {
  const Paged& p = a.p;
  const long long share = a.before[p.B + 1];
  const int items = share ? a.tiles[p.B] * (D / 4) : 0, r = threadIdx.x;
  bool waited = false;
  for (int item = blockIdx.x; item < items || !waited; item += gridDim.x) {
    int splits = 0, w0 = 0, h = 0, row = -1;
    const int tile = item / (D / 4), c = item % (D / 4) * 4;
    const int b = item < items ? paged_owner(a.tiles, p.B, tile) : -1;
    if (b >= 0 && b < p.B) {
      const Piece s = paged_piece(p, b);
      const int rows = (s.live + PT - 1) / PT, g = tile - a.tiles[b], qt = g % rows;
      const long long from = a.before[b] + (g / rows) * plan_front(a, s, rows) + plan_front(a, s, qt) + PIECE_WAY;
      h = g / rows;
      w0 = (int)(from / share);
      splits = (int)((from + plan_tiles(a, s, qt) - 1) / share) - w0 + 1;
      if (qt * PT + r < s.live) row = s.row + qt * PT + r;
    }
    if (!waited) {
      pdl_wait();                                 // (by every CTA: who comes behind this kernel waits for its end alone)
      pdl_launch();
      waited = true;
    }
    if (splits < 2 || row < 0) continue;
    // the first CTA's second place, the others' first
    const float* part = a.parts + (2ll * w0 * D + c) * PT + r;
    const float* sum = a.parts + (long long)a.slots * PT * D + 2ll * w0 * PT + r;
    float x[4] = {}, l = 0.f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += part[((2ll * k + (k == 0)) * D + i) * PT];
      l += sum[(2ll * k + (k == 0)) * PT];
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<uint2*>(a.y + ((long long)row * p.H + h) * D + c) = make_uint2(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv));
  }
}

static int tmap_rows_2d(CUtensorMap* out, const void* ptr, long long rows, long long cols, int box_rows) {
  uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  uint64_t strides[1] = {(uint64_t)cols * 2};
  uint32_t box[2] = {64, (uint32_t)box_rows};
  return make_tmap(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D>
static int launch_pieces(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PiecesArgs& a, cudaStream_t s) {
  constexpr size_t smem = (size_t)(D / 64) * PATOM * 7 + PP_BARS + 4 * PT * sizeof(float);
  static OncePerDevice limit;
  BONES_ONCE(limit, {
    BONES_CHECK(cudaFuncSetAttribute(paged_pieces_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  });
  const Paged& p = a.p;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3(1 + (unsigned)min((p.N + 31ll) / 32, (long long)a.sms));
  cfg.blockDim = dim3(PLAN_T);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  BONES_CHECK(cudaLaunchKernelEx(&cfg, paged_plan_kernel, a));
  // a CTA an SM, fewer where the items cannot be as many
  const long long tiles = (p.N / PT + (long long)min(p.B, p.N)) * p.H;
  cfg.gridDim = dim3((unsigned)(a.slots ? a.sms : min(tiles, (long long)a.sms)));
  cfg.blockDim = dim3(PP_THREADS);
  cfg.dynamicSmemBytes = smem;
  BONES_CHECK(cudaLaunchKernelEx(&cfg, paged_pieces_kernel<D>, tq, tk, tv, a));
  if (a.slots == 0) return 0;
  cfg.gridDim = dim3((unsigned)min(tiles * (D / 4), 12ll * a.sms));
  cfg.blockDim = dim3(PT);
  cfg.dynamicSmemBytes = 0;
  return (int)cudaLaunchKernelEx(&cfg, paged_pieces_join_kernel<D>, a);
}

// Places for parts, two a CTA; none where the tiles of queries alone are two an SM, or see a few tiles of keys at most.
static int pieces_slots(int N, int cap, int H, int window_tiles, int sms) {
  const long long seen = window_tiles > 0 ? min((long long)cap, window_tiles * 128ll + 128) : cap;
  return seen > PIECE_LEAST * PT && (long long)(N / PT) * H < 2ll * sms ? 2 * sms : 0;
}
static long long pieces_ints(int B) { return (3ll * B + 16 + 7) / 8 * 8; }

long long paged_pieces_room(int B, int N, int cap, int H, int D, int window_tiles, int sms) {
  return 4 * (pieces_ints(B) + (long long)pieces_slots(N, cap, H, window_tiles, sms) * PT * (D + 1));
}

int paged_pieces(const void* q, const void* k, const Paged& p, const int* doc_start, void* y, int D, float scale, int window_tiles, int sms, void* work, void* stream) {
  if ((p.N / PT + (long long)p.B) * p.H > 0x3fffffffll) return -2;
  const float log2e = 1.4426950408889634f;
  PiecesArgs a = {};
  a.p = p;
  a.c1 = scale * log2e;
  a.c2 = (scale < 0 ? -scale : scale) * D * log2e;
  a.window_tiles = window_tiles;
  a.doc_start = doc_start;
  a.y = (__nv_bfloat16*)y;
  a.err = error_word();
  a.next = (int*)work;
  a.before = (long long*)(a.next + 2);
  a.tiles = (int*)(a.before + p.B + 2);
  a.slots = pieces_slots(p.N, p.cap, p.H, window_tiles, sms);
  a.parts = (float*)work + pieces_ints(p.B);
  a.row_bytes = p.H * D * 2;
  a.sms = sms;
  CUtensorMap tq, tk, tv;
  const long long rows = ((long long)p.pages * p.H) << p.shift;
  int rc = tmap_rows_2d(&tq, q, p.N, (long long)p.H * D, PT);
  if (!rc) rc = tmap_rows_2d(&tk, k, rows, D, 1 << p.shift);
  if (!rc) rc = tmap_rows_2d(&tv, p.values, rows, D, 1 << p.shift);
  if (rc) return rc;
  return D == 128 ? launch_pieces<128>(tq, tk, tv, a, (cudaStream_t)stream) : launch_pieces<64>(tq, tk, tv, a, (cudaStream_t)stream);
}

}  // namespace bones
