// Attention of pieces of new tokens over a paged cache, in tiles of 128 queries and 128 keys: `tcgen05` products with TMEM accumulators,
// keys and values brought page by page by TMA.  The formula stands with the kernels for pieces of a few tokens (paged.cu).
//
// Three kernels.  A plan (one CTA; others clear the rows that get no result): how many items each sequence has.  An item is a head's tile of
// queries against its visible tiles of keys, or, where there are too few of those for all SMs, a part of these, whose sums go to memory.
// The attention itself, persistent.  A join of parts, where there may be some.
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
  int* prefix;                // [B + 1]: items of the sequences before
  int* splits;                // [B]: parts of a tile of queries
  int* places;                // [B]: the first of its parts' places, where there are parts
  float* parts;               // [slots][128][D], and behind them [slots][128] sums of weights
  int slots, sms, row_bytes;
};

// ---------------------------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------------------------
constexpr int PLAN_T = 256;

__device__ __forceinline__ int plan_tiles(const PiecesArgs& a, const Piece& s) {       // key tiles of the longest row of tiles
  const int last = (s.pos + s.live - 1) >> 7;
  return a.window_tiles > 0 ? min(last + 1, a.window_tiles + 1) : last + 1;
}
// Sums of `v` over the threads in front; the total in *all.
__device__ __forceinline__ int plan_scan(int v, int* box, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += x;
  }
  if (lane == 31) box[warp] = up;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < PLAN_T / 32; ++w) {
    const int x = box[w];
    if (w < warp) before += x;
    total += x;
  }
  __syncthreads();
  *all = total;
  return before + up - v;
}

__global__ void __launch_bounds__(PLAN_T) paged_plan_kernel(const PiecesArgs a) {
  __shared__ int box[PLAN_T / 32], rows_of[PLAN_T], tiles_of[PLAN_T], part;
  __shared__ float cost[2];
  __shared__ int cut[2];
  const Paged& p = a.p;
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
  if (threadIdx.x == 0) *a.next = 0;
  // Parts only where the tiles of queries alone leave SMs without work, and only of up to PLAN_T sequences
  part = 0x7fffffff;
  if (a.slots > 0 && p.B <= PLAN_T) {
    int rows = 0, tiles = 0, items;
    if ((int)threadIdx.x < p.B) {
      const Piece s = paged_piece(p, threadIdx.x);
      if (s.live) {
        rows = (s.live + PT - 1) / PT * p.H;
        tiles = plan_tiles(a, s);
      }
    }
    rows_of[threadIdx.x] = rows;
    tiles_of[threadIdx.x] = tiles;
    plan_scan(rows, box, &items);
    if (items < 2 * a.sms) {
      // parts of a 1st to 64th of the longest row of tiles: what the fullest SM has, an item's way in and out as one tile more
      int most = 0;
      for (int b = 0; b < p.B; ++b) most = max(most, tiles_of[b]);
      if (threadIdx.x < 64) {
        const int len = (most + threadIdx.x) / ((int)threadIdx.x + 1);
        float work = 0.f, n = 0.f, used = 0.f;
        if (len > 0) {
          const float inv = 1.0f / len;
          for (int b = 0; b < p.B; ++b) {
            const float rows_b = (float)rows_of[b], s = ceilf(tiles_of[b] * inv);          // (as estimates go)
            work += rows_b * tiles_of[b];
            n += rows_b * s;
            if (s > 1.f) used += rows_b * (s + 1.f);
          }
        }
        const float waves = ceilf(n / a.sms);
        float c = used > a.slots || (threadIdx.x > 0 && len < 3) ? 1e30f : fmaxf(fminf(waves * (len + 1.f), (work + n) / a.sms + 0.5f * len), len + 1.f);
        int best = threadIdx.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float x = __shfl_xor_sync(0xffffffffu, c, o);
          const int i = __shfl_xor_sync(0xffffffffu, best, o);
          if (x < c || (x == c && i < best)) {
            c = x;
            best = i;
          }
        }
        if ((threadIdx.x & 31) == 0) {
          cost[threadIdx.x >> 5] = c;
          cut[threadIdx.x >> 5] = best;
        }
      }
      __syncthreads();
      const int best = cost[1] < cost[0] ? cut[1] : cut[0];
      if (threadIdx.x == 0 && best) part = (most + best) / (best + 1);
    }
  }
  __syncthreads();
  int items = 0, places = 0;
  for (int b0 = 0; b0 < p.B; b0 += PLAN_T) {
    const int b = b0 + threadIdx.x;
    int rows = 0, s = 1;
    if (b < p.B) {
      const Piece x = paged_piece(p, b);
      if (x.live) {
        rows = (x.live + PT - 1) / PT * p.H;
        s = part == 0x7fffffff ? 1 : max(1, (plan_tiles(a, x) + part - 1) / part);
      }
    }
    int all, more;
    const int at = items + plan_scan(rows * s, box, &all), place = places + plan_scan(s > 1 ? rows * s : 0, box, &more);
    if (b < p.B) {
      a.prefix[b] = at;
      a.splits[b] = s;
      a.places[b] = place;
    }
    items += all;
    places += more;
  }
  if (threadIdx.x == 0) a.prefix[p.B] = items;
}

// ---------------------------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------------------------
// Roles as in the training forward (attention.cu): a warp each for Q and K loads, V loads, S = Q K^T, O += P V; sixteen softmax warps (four per
// 32-lane TMEM quadrant, 32 keys a thread); four drain warps.  Here a warp of its own draws the items and looks up what they are (the sequence, its
// rows, the first and last of their keys): three dependent reads that nobody waits for, since it runs one item ahead.  What is of this kernel:
//  - pages: a box of the tensor map is one page's P tokens of one head; a position without a page is loaded as zeros and masked.
//  - rows behind a piece's end (a step with a few drafts has 5 of 128) take no exponentials: a softmax warp without a live row passes its tiles on.
//  - values that a row does not see may be anything (other sequences' leftovers behind the end): in tiles with a mask the drain warps look
//    through V before its product, put zeros for what is not finite, and add it back to the rows that do see it at the end.
constexpr int PP_SW = 16, PP_DW = 4;
constexpr int PP_PV = 2 + PP_SW + PP_DW, PP_VW = PP_PV + 1, PP_IW = PP_VW + 1;
constexpr int PP_THREADS = 32 * (PP_IW + 1);
constexpr int PP_RING = 2;                      // items handed round: the one being computed and the next
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
    if (threadIdx.x == 0) atomicCAS(a.err, 0, ERR_WAIT_AUX);
    return;
  }
  auto sQ = [&](int s) { return base + TILE * s; };
  auto sK = [&](int s) { return base + TILE * (2 + s); };
  auto sV = [&](int s) { return base + TILE * (4 + s); };
  constexpr uint32_t kBars = TILE * 7;
  const uint32_t bars = base + kBars;
  auto q_full = [&](int s) { return bars + 8u * (0 + s); };
  auto q_free = [&](int s) { return bars + 8u * (2 + s); };
  auto k_full = [&](int s) { return bars + 8u * (4 + s); };
  auto k_free = [&](int s) { return bars + 8u * (6 + s); };
  auto v_full = [&](int s) { return bars + 8u * (8 + s); };
  auto v_free = [&](int s) { return bars + 8u * (11 + s); };
  auto v_fine = [&](int s) { return bars + 8u * (14 + s); };
  auto s_full = [&](int s) { return bars + 8u * (17 + s); };
  auto s_free = [&](int s) { return bars + 8u * (20 + s); };
  auto p_full = [&](int s) { return bars + 8u * (23 + s); };
  auto i_full = [&](int s) { return bars + 8u * (26 + s); };
  auto i_free = [&](int s) { return bars + 8u * (28 + s); };
  const uint32_t o_full = bars + 8u * 30, o_free = bars + 8u * 31, l_full = bars + 8u * 32, l_free = bars + 8u * 33;
  const uint32_t tmem_slot = bars + 288u;
  volatile uint32_t* tmem_slot_g = reinterpret_cast<volatile uint32_t*>(gen + kBars + 288);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kBars + 292);
  int* taint = reinterpret_cast<int*>(gen + kBars + 296);                                    // [PP_RING]
  PieceItem* ring = reinterpret_cast<PieceItem*>(gen + kBars + 320);                         // [PP_RING]
  static_assert(320 + PP_RING * sizeof(PieceItem) <= PP_BARS && PP_RING == 2, "room");
  float* lsum = reinterpret_cast<float*>(gen + kBars + PP_BARS);                             // [4 column parts][128 rows]

  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int A = p.H * D;
  if (warp == 0) {
    for (int i = lane; i < 34; i += 32) {
      const bool by_softmax = (i >= 23 && i < 26) || i == 32, by_drain = (i >= 14 && i < 17) || i == 28 || i == 29 || i == 31 || i == 33;
      mbar_init(bars + 8u * (uint32_t)i, by_softmax ? PP_SW : by_drain ? PP_DW : 1);
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
  pdl_launch();
  pdl_wait();                                   // the plan
  auto tS = [&](int s) { return tmem + (uint32_t)s * 128u; };
  const uint32_t tO = tmem + 384u;
  // the it-th item of this CTA; false behind the last one
  auto take = [&](int it, PieceItem* im) {
    if (!__all_sync(0xffffffffu, mbar_wait(i_full(it & 1), (uint32_t)((it >> 1) & 1), abort_flag, a.err, ERR_WAIT_AUX))) return false;
    *im = ring[it & 1];
    return warp_uniform(im->n) > 0;
  };
  // whether some row of the item does not see some key of the tile
  auto masked = [&](const PieceItem& im, int kt) { return kt * PT + PT - 1 > im.pos0 || kt * PT < im.far || im.none; };
  const int per_tile = PT >> p.shift;           // pages of a tile
  // row of the tensor map of lane i's page of tile kt (lanes below per_tile); behind the map, which reads as zeros, where there is none
  auto page_row = [&](const PieceItem& im, int kt) {
    const int i = kt * per_tile + lane;
    int row = (int)(((long long)p.pages * p.H) << p.shift);
    if (lane < per_tile && i < p.M && (i << p.shift) < im.pos0 + im.live) {
      const long long at = paged_at(p, p.table[im.seq * p.ldt + i], im.h);
      if (at >= 0) row = (int)at;
    }
    return row;
  };
  const uint32_t page_bytes = 128u << p.shift;  // of a column half

  if (warp == PP_IW) {
    // The items, in sequence- and head-major order, so that CTAs at work at one time share keys and values through L2.
    const int total = p.B > 0 ? a.prefix[p.B] : 0;
    for (int it = 0;; ++it) {
      int w = (int)blockIdx.x;
      if (it > 0) w = (int)gridDim.x + warp_uniform(lane == 0 ? atomicAdd(a.next, 1) : 0);
      PieceItem im = {};
      if (w < total) {
        const int b = min(max(paged_owner(a.prefix, p.B, w), 0), p.B - 1);
        const Piece s = paged_piece(p, b);
        const int splits = a.splits[b], r = w - a.prefix[b], part = r % splits, g = r / splits, rows = (s.live + PT - 1) / PT;
        im.seq = b;
        im.h = g / rows;
        const int qt = rows - 1 - (g % rows + im.h) % rows;
        im.row0 = s.row + qt * PT;
        im.live = min(PT, s.live - qt * PT);
        im.pos0 = s.pos + qt * PT;
        im.place = splits > 1 ? a.places[b] + r : -1;
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
        const int from = (int)((long long)part * n / splits), to = (int)((long long)(part + 1) * n / splits);
        im.none = to <= from;
        im.kt0 = im.none ? last : first + from;
        im.n = im.none ? 1 : to - from;
      }
      const int slot = it & 1;
      if (it >= PP_RING && !__all_sync(0xffffffffu, mbar_wait(i_free(slot), (uint32_t)(((it - PP_RING) >> 1) & 1), abort_flag, a.err, ERR_WAIT_EMPTY))) break;
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
    int g = 0;
    bool dead = false;
    for (int it = 0; !dead && take(it, &im); ++it) {
      const int qb = it & 1;
      if (it >= 2 && !dead) dead = !mbar_wait(q_free(qb), (uint32_t)(((it - 2) >> 1) & 1), abort_flag, a.err, ERR_WAIT_EMPTY);
      const int h = warp_uniform(im.h), row0 = warp_uniform(im.row0);
      if (elect_one() && !dead) {
        mbar_arrive_expect_tx(q_full(qb), TILE);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_load_2d(sQ(qb) + c * PATOM, &tm_q, q_full(qb), h * D + c * 64, row0);
      }
      int row = page_row(im, im.kt0);
      for (int j = 0; j < im.n; ++j, ++g) {
        const int ks = g & 1, now = row;
        if (j + 1 < im.n) row = page_row(im, im.kt0 + j + 1);
        if (g >= 2 && !dead) dead = !mbar_wait(k_free(ks), (uint32_t)(((g - 2) >> 1) & 1), abort_flag, a.err, ERR_WAIT_EMPTY);
        if (elect_one() && !dead) mbar_arrive_expect_tx(k_full(ks), TILE);
        __syncwarp();
        for (int i = 0; i < per_tile; ++i) {
          const int at = __shfl_sync(0xffffffffu, now, i);
          if (elect_one() && !dead) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_2d(sK(ks) + c * PATOM + i * page_bytes, &tm_k, k_full(ks), c * 64, at);
          }
        }
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
  } else if (warp == 1) {
    // S = Q K^T of each tile, into the buffer whose O += P V (three tiles before) is done
    constexpr uint32_t kHi = umma_desc_hi(1024, kLayoutSw128);
    const uint32_t idesc_s = umma_idesc_f16(128, 128, 1, 0, 0);   // Q (K-major) x K (K-major)
    const uint32_t q_lo = (uint32_t)warp_uniform((int)umma_desc_lo(sQ(0), 0)), k_lo = (uint32_t)warp_uniform((int)umma_desc_lo(sK(0), 0));
    PieceItem im;
    bool dead = false;
    int g = 0, gs = 0;
    uint32_t fph = 1;
    for (int it = 0; !dead && take(it, &im); ++it) {
      const int n = warp_uniform(im.n), qb = it & 1;
      if (!dead) dead = !mbar_wait(q_full(qb), (uint32_t)((it >> 1) & 1), abort_flag, a.err, ERR_WAIT_FULL);
      for (int j = 0; j < n; ++j, ++g) {
        const int kb = g & 1;
        if (!dead) dead = !mbar_wait(k_full(kb), (uint32_t)((g >> 1) & 1), abort_flag, a.err, ERR_WAIT_FULL);
        if (g >= 3 && !dead) dead = !mbar_wait(s_free(gs), fph, abort_flag, a.err, ERR_WAIT_TMEM_EMPTY);
        tc_fence_after();
        const uint32_t qd = q_lo + (uint32_t)qb * (TILE >> 4), kd = k_lo + (uint32_t)kb * (TILE >> 4), sd = tS(gs);
        if (elect_one() && !dead) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = ((k >> 2) * PATOM + (k & 3) * 32) >> 4;
            umma_f16_lh(sd, qd + off, kHi, kd + off, kHi, idesc_s, k ? 1u : 0u);
          }
          tc_commit(s_full(gs));
          tc_commit(k_free(kb));
          if (j == n - 1) tc_commit(q_free(qb));
        }
        if (++gs == 3) { gs = 0; fph ^= 1u; }
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
    int gs = 0;
    uint32_t sph = 0;
    bool ok = true;
    for (int it = 0; ok && take(it, &im); ++it) {
      const bool idle = q * 32 >= im.live;       // none of this warp's rows is one
      // rows behind the piece's end are not stored: no mask either
      const int qpos = r >= im.live ? 0x3fffffff : im.none ? -1 : im.pos0 + r;
      int lo = 0;
      if (r < im.live) {
        if (a.doc_start) lo = a.doc_start[im.row0 + r];
        if (a.window_tiles > 0) lo = max(lo, (((im.pos0 + r) >> 7) - (a.window_tiles - 1)) * 128);
      }
      const int* table = p.table + im.seq * p.ldt;
      float l = 0.f;
      for (int j = 0; j < im.n; ++j) {
        const int k0 = (im.kt0 + j) * PT + c0;
        bool there_a = true, there_b = true;     // pages of the first and second sixteen keys
        if (!idle) {
          const int ia = k0 >> p.shift, ib = (k0 + 16) >> p.shift;
          there_a = ia < p.M && (uint32_t)table[ia] < (uint32_t)p.pages;
          there_b = ib < p.M && (uint32_t)table[ib] < (uint32_t)p.pages;
        }
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
          if (__any_sync(0xffffffffu, (k0 + 31 > qpos) || (k0 < lo) || !there_a || !there_b)) {
            const int end = qpos - k0, from = lo - k0;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i > end || i < from || !(i < 16 ? there_a : there_b)) e[i] = 0.f;
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
    // Drain: a thread per query row; before, the tiles of V in which some row sees only some keys
    const int q = warp & 3, r = q * 32 + lane;
    const uint32_t tOr = tO + ((uint32_t)(q * 32) << 16);
    PieceItem im;
    int vs = 0;
    uint32_t vph = 0;
    bool ok = true;
    for (int it = 0; ok && take(it, &im); ++it) {
      const int end = im.pos0 + im.live;
      for (int j = 0; j < im.n; ++j) {
        // Every tile is passed on from here, so that no phase of a stage goes by unseen (a wait tells apart two phases, not three)
        if (!__all_sync(0xffffffffu, mbar_wait(v_full(vs), vph, abort_flag, a.err, ERR_WAIT_FULL))) { ok = false; break; }
        if (masked(im, im.kt0 + j)) {
          uint4* tile = reinterpret_cast<uint4*>(gen + TILE * (4 + vs)) + q * (TILE / 64) + lane;        // a quarter; TILE / 16 pieces of 16 bytes
          uint32_t odd = 0;
#pragma unroll 8
          for (int i = 0; i < (int)(TILE / 64 / 32); ++i) {
            const uint4 u = tile[i * 32];
            // an exponent of all ones carries into the sign's place
            odd |= ((u.x & 0x7f807f80u) + 0x00800080u) | ((u.y & 0x7f807f80u) + 0x00800080u) | ((u.z & 0x7f807f80u) + 0x00800080u) | ((u.w & 0x7f807f80u) + 0x00800080u);
          }
          if (__any_sync(0xffffffffu, odd & 0x80008000u)) {
            bool seen = false;
            for (int i = 0; i < (int)(TILE / 64 / 32); ++i) {
              uint4 u = tile[i * 32];
              uint32_t w[4] = {u.x, u.y, u.z, u.w};
              bool any = false;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t t = ((w[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                if (t) any = true;
                if (t & 0x8000u) w[k] &= 0xffff0000u;
                if (t & 0x80000000u) w[k] &= 0xffffu;
              }
              if (any) {
                tile[i * 32] = make_uint4(w[0], w[1], w[2], w[3]);
                const int key = (im.kt0 + j) * PT + (((q * (int)(TILE / 64) + lane + i * 32) * 16 >> 7) & (PT - 1));
                if (key < end) seen = true;         // not a leftover behind the end
              }
            }
            if (__any_sync(0xffffffffu, seen) && lane == 0) atomicOr(&taint[it & 1], 1);
            fence_proxy_async_smem();
            __threadfence_block();
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(v_fine(vs));
        if (++vs == 3) { vs = 0; vph ^= 1u; }
      }
      if (!ok) break;
      const bool real = r < im.live;
      bool got = mbar_wait(l_full, (uint32_t)(it & 1), abort_flag, a.err, ERR_WAIT_AUX);
      if (!__all_sync(0xffffffffu, got)) break;
      const float l = (lsum[r] + lsum[PT + r]) + (lsum[2 * PT + r] + lsum[3 * PT + r]);
      __syncwarp();
      if (lane == 0) mbar_arrive(l_free);
      const float inv = l == 0.f ? 0.f : 1.0f / l;        // a row that sees no key has zeros
      const long long col = (long long)im.h * D;
      __nv_bfloat16* y = a.y + (long long)(im.row0 + r) * A + col;
      float* part = a.parts + ((long long)im.place * PT + r) * D;
      if (im.place >= 0 && real) a.parts[(long long)a.slots * PT * D + (long long)im.place * PT + r] = l;
      got = mbar_wait(o_full, (uint32_t)(it & 1), abort_flag, a.err, ERR_WAIT_TMEM_FULL);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      const bool tainted = warp_uniform(*(volatile int*)&taint[it & 1]) != 0;
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
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(part + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
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
      if (lane == 0) mbar_arrive(i_free(it & 1));
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

// Adds the parts of a row and head in their order.  D / 4 threads a row and head.
template <int D>
__global__ void __launch_bounds__(256) paged_pieces_join_kernel(const PiecesArgs a) {
  constexpr int T = D / 4, PAIRS = 256 / T;
  const Paged& p = a.p;
  const long long item = (long long)blockIdx.x * PAIRS + threadIdx.x / T;
  const int d = threadIdx.x % T;
  const bool on = item < (long long)p.N * p.H;
  const int row = on ? (int)(item / p.H) : -1, h = on ? (int)(item % p.H) : 0;
  int b = -1;
#pragma unroll
  for (int i = 0; i < 32; i += T) {
    const int x = paged_owner(p.starts, p.B, __shfl_sync(0xffffffffu, row, i));
    if ((int)(threadIdx.x & 31) >= i) b = x;
  }
  Piece s = {};
  if (on && b >= 0 && b < p.B) s = paged_piece(p, b);
  pdl_wait();
  const int i = row - s.row;
  if (!on || !s.live || i < 0 || i >= s.live) return;
  const int splits = a.splits[b], place0 = a.places[b];
  if (splits == 1) return;
  const int rows = (s.live + PT - 1) / PT, qt = i / PT, g = h * rows + ((rows - 1 - qt - h) % rows + rows) % rows;
  const long long place = place0 + (long long)g * splits;
  const float* parts = a.parts + (place * PT + i % PT) * D + 4 * d;
  const float* sums = a.parts + (long long)a.slots * PT * D + place * PT + i % PT;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    const float4 z = *reinterpret_cast<const float4*>(parts + (long long)k * PT * D);
    x.x += z.x;
    x.y += z.y;
    x.z += z.z;
    x.w += z.w;
    l += sums[(long long)k * PT];
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<uint2*>(a.y + ((long long)row * p.H + h) * D + 4 * d) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
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
  BONES_ONCE(limit, { BONES_CHECK(cudaFuncSetAttribute(paged_pieces_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)); });
  const Paged& p = a.p;
  paged_plan_kernel<<<1 + (unsigned)min((p.N + 31ll) / 32, (long long)a.sms), PLAN_T, 0, s>>>(a);
  BONES_CHECK(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  // a CTA an SM, fewer where the items cannot be as many
  const long long most = (p.N / PT + (long long)min(p.B, p.N)) * p.H + a.slots;
  cfg.gridDim = dim3((unsigned)min(most, (long long)a.sms));
  cfg.blockDim = dim3(PP_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  BONES_CHECK(cudaLaunchKernelEx(&cfg, paged_pieces_kernel<D>, tq, tk, tv, a));
  if (a.slots == 0) return 0;
  const long long pairs = (long long)p.N * p.H;
  cfg.gridDim = dim3((unsigned)((pairs + 1024 / D - 1) / (1024 / D)));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return (int)cudaLaunchKernelEx(&cfg, paged_pieces_join_kernel<D>, a);
}

}  // namespace bones

extern "C" {
using namespace bones;

// As bones_paged_rows.  ints: room for 3 B + 16 ints; parts: room for slots * 128 * (D + 1) floats on 16 bytes, or null with slots 0; both of this
// call alone until it ends.
int bones_paged_pieces(const void* q, const void* k, const void* v, int pages, const int* table, long long ldt, const int* starts, const int* pos,
                       const int* doc_start, void* y, int B, int N, int M, int H, int D, int shift, float scale, int window_tiles, int* ints, float* parts,
                       int slots, void* stream) {
  if (paged_refused(B, N, M, H, D, shift, pages, ldt, k, v, starts, pos, table) || !q || !y || (((uintptr_t)q | (uintptr_t)y) & 31) || window_tiles < 0 || !ints ||
      slots < 0 || (slots && !parts) || misaligned16(parts) || (N / PT + (long long)B) * H > 0x3fffffffll)
    return -2;
  if (N == 0) return 0;
  const float log2e = 1.4426950408889634f;
  PiecesArgs a = {};
  a.p = Paged{starts, pos, table, ldt, B, N, M, H, shift, pages, (int)min((long long)M << shift, 0x7fffff00ll), v};
  a.c1 = scale * log2e;
  a.c2 = (scale < 0 ? -scale : scale) * D * log2e;
  a.window_tiles = window_tiles;
  a.doc_start = doc_start;
  a.y = (__nv_bfloat16*)y;
  a.err = error_word();
  a.next = ints;
  a.prefix = ints + 4;
  a.splits = a.prefix + B + 1;
  a.places = a.splits + B;
  a.parts = parts;
  a.slots = slots;
  a.row_bytes = H * D * 2;
  int dev = 0;
  BONES_CHECK(cudaGetDevice(&dev));
  BONES_CHECK(cudaDeviceGetAttribute(&a.sms, cudaDevAttrMultiProcessorCount, dev));
  CUtensorMap tq, tk, tv;
  const long long rows = ((long long)pages * H) << shift;
  int rc = tmap_rows_2d(&tq, q, N, (long long)H * D, PT);
  if (!rc) rc = tmap_rows_2d(&tk, k, rows, D, 1 << shift);
  if (!rc) rc = tmap_rows_2d(&tv, v, rows, D, 1 << shift);
  if (rc) return rc;
  return D == 128 ? launch_pieces<128>(tq, tk, tv, a, (cudaStream_t)stream) : launch_pieces<64>(tq, tk, tv, a, (cudaStream_t)stream);
}
}  // extern "C"
