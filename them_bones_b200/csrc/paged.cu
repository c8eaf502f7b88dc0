// A paged key/value cache in bf16: append with RoPE and QK-norm on the way, and attention of pieces of new tokens in tiles of 16 rows.
//
//   append:     u = rope(x, p), x^ = u / sqrt(mean u^2 + 2^-23) for the query and the key;  k^, v -> page table[b, p / P], slot p % P;  q^ out
//   attention:  y_i = sum_j softmax_j(scale q_i . k_j) v_j  over the positions j of the sequence with first_i <= j <= pos_i
//
// Queries and keys are normalised, so |q . k| <= D and the soft-max takes the fixed shift |scale| D instead of a running maximum: the
// parts that warps and CTAs make of a row are plain sums, and joining them is adding.
#include "decode_common.cuh"
#include "paged.cuh"

namespace bones {

constexpr float kPagedEps = 1.1920928955078125e-07f;   // 2^-23

__device__ __forceinline__ void paged_st8(__nv_bfloat16* p, const float* f) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ void paged_ld8f(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// ---------------------------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------------------------
// A head vector by D / 16 lanes: eight values of the first half and their partners of the second each.  All lanes of the warp come here.
template <int D>
__device__ __forceinline__ void paged_turn(const float* a, const float* b, const float* cs, const float* sn, float* y1, float* y2) {
  auto turn = [&](float by) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x1 = a[e] * by, x2 = b[e] * by;
      y1[e] = x1 * cs[e] + x2 * sn[e];
      y2[e] = -x1 * sn[e] + x2 * cs[e];
      ss += y1[e] * y1[e] + y2[e] * y2[e];
    }
#pragma unroll
    for (int o = 1; o < D / 16; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return ss;
  };
  float ss = turn(1.0f), eps = kPagedEps;
  if (__any_sync(0xffffffffu, !(ss < 1e36f))) {      // values whose squares leave fp32: the norm of 2^-70 of them is the same
    const bool large = !(ss < 1e36f);
    ss = turn(large ? 0x1p-70f : 1.0f);
    if (large) eps = 0.f;                            // beside a mean square of 1e34 and more it was nothing
  }
  const float r = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y1[e] *= r;
    y2[e] *= r;
  }
}

__device__ __forceinline__ void paged_unpack(const uint4* raw, float* a, float* b) {
  unpack8(raw[0], a);
  unpack8(raw[1], b);
}

// A CTA takes up to AR rows with all their heads, D / 16 lanes a head: a row's sequence, page and angles are looked up once a CTA, and no lane is left
// over whatever the number of heads.  What a lane takes stays packed until it is worked on: 96 bytes on their way in 24 registers.  Bound by memory: 8 prompts of 2048
// tokens, 10 heads of 128, 46.6 us (5.6 TB/s, 0.85 of the copy rate); a warp a row with unpacked values 57; this with 256 threads a CTA 48.4, with 8 / 16 rows of 128 / 256 threads
// 50.4 / 52.2.
constexpr int AT = 128, AR = 4;
template <int D>
__global__ void __launch_bounds__(AT, 6) paged_append_kernel(const __nv_bfloat16* __restrict__ qkv, long long ldq, const float* __restrict__ cosT,
                                                             const float* __restrict__ sinT, int rope_rows, int rows, const Paged p, __nv_bfloat16* __restrict__ k,
                                                             __nv_bfloat16* __restrict__ v, __nv_bfloat16* __restrict__ q) {
  constexpr int LANES = D / 16, HALF = D / 2;
  __shared__ int pos_of[AR];                 // -1: no new token, or one that is left out
  __shared__ long long place_of[AR];         // of head 0, in rows of D; -1 without a page
  const int row0 = blockIdx.x * rows, items = min(rows, p.N - row0) * p.H;
  const int l8 = threadIdx.x % LANES, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long A = (long long)p.H * D;
  uint4 raw[3][2];
  auto load = [&](int item) {
    if (item >= items) return;
    const int r = item / p.H;
    const __nv_bfloat16* src = qkv + (row0 + r) * ldq + (long long)(item - r * p.H) * D + l8 * 8;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      raw[i][0] = *reinterpret_cast<const uint4*>(src + i * A);
      raw[i][1] = *reinterpret_cast<const uint4*>(src + i * A + HALF);
    }
  };
  int item = threadIdx.x / LANES;
  pdl_wait();
  pdl_launch();
  load(item);                                // on its way while the rows are looked up
  for (int r = warp; r < rows && row0 + r < p.N; r += AT / 32) {
    const int b = paged_owner(p.starts, p.B, row0 + r);
    int t = -1;
    long long at = -1;
    if (b >= 0 && b < p.B) {
      const Piece s = paged_piece(p, b);
      const int i = row0 + r - s.row;
      if (i >= 0 && i < s.live && s.pos + i < rope_rows) {
        t = s.pos + i;
        at = paged_at(p, p.table[b * p.ldt + (t >> p.shift)], 0);
        if (at >= 0) at += t & ((1 << p.shift) - 1);
      }
    }
    if (lane == 0) {
      pos_of[r] = t;
      place_of[r] = at;
    }
  }
  __syncthreads();
  // all lanes of a warp make the same rounds
  for (int first = (int)(threadIdx.x & ~31u) / LANES; first < items; first += AT / LANES, item += AT / LANES) {
    const bool on = item < items;
    const int r = on ? item / p.H : 0, h = on ? item - r * p.H : 0, t = on ? pos_of[r] : -1;
    const long long at = on ? place_of[r] : -1;
    __nv_bfloat16* out = q + (row0 + r) * A + (long long)h * D + l8 * 8;
    float cs[8], sn[8], y1[8], y2[8], a[8], b[8];
    const long long angle = (long long)max(t, 0) * HALF + l8 * 8;
    if (rope_rows > 0) {
      paged_ld8f(cosT + angle, cs);
      paged_ld8f(sinT + angle, sn);
    }
    paged_unpack(raw[0], a, b);
    paged_turn<D>(a, b, cs, sn, y1, y2);
    if (on && t >= 0) {
      paged_st8(out, y1);
      paged_st8(out + HALF, y2);
    } else if (on) {
      *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(out + HALF) = make_uint4(0, 0, 0, 0);
    }
    paged_unpack(raw[1], a, b);
    paged_turn<D>(a, b, cs, sn, y1, y2);
    if (on && at >= 0) {
      const long long o = (at + ((long long)h << p.shift)) * D + l8 * 8;
      paged_st8(k + o, y1);
      paged_st8(k + o + HALF, y2);
      *reinterpret_cast<uint4*>(v + o) = raw[2][0];
      *reinterpret_cast<uint4*>(v + o + HALF) = raw[2][1];
    }
    load(item + AT / LANES);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// attention in tiles of 16 rows
// ---------------------------------------------------------------------------------------------------------------
// A step of one to sixteen tokens a sequence is bound by the bytes of its keys and values, each read once.  A warp takes 16 keys a turn,
// straight from their page into the registers that the legacy matrix instruction wants them in: `tcgen05` would leave 112 and more of its 128
// rows to waste and have everything go through shared memory.  The contraction's order is free, so lane (g, c) = (lane / 4, lane % 4) takes
// 16 consecutive dimensions of key g as its share of four steps (32 bytes a load), with the queries laid out alike; of the values it takes
// D / 8 consecutive dimensions of keys 2c, 2c + 1, 2c + 8, 2c + 9, whose pairs two byte permutations make into operands.
// Probabilities enter the second product in bf16, the type of the values: each is off by 2^-8 of itself at most.
//
// The turns of all tiles of all heads, one after another, are shared equally by as many warps as the SMs hold: a step's sequences have any lengths,
// and with a CTA or a cluster a head the way in and out of each was longer than its turns.  A warp that has all turns of a tile writes its
// rows; of the at most two tiles that it shares with others it leaves sums, which a second kernel adds in order.  A tile counts as RC turns more than it
// has, the way to its first keys: without them a warp got as many tiles of a turn or two as others got turns of one (64 sequences: 33.4 us; with one, two or three 26).
//
// Measured, us of a whole call, 10 heads of 128: 4 sequences of 32768 to 131072 tokens 253 (the copy rate); 64 of up to 2048 tokens 26.0 (4.1 TB/s), 32 of 1500 with up to
// five new tokens each the same; one of 300 7.6.  In the second the first keys are there 10000 clocks behind the launch (the shares 2800, where in them 1900, tables, and 19 MB that
// all warps ask for at once), the warps end between 36000 and 41600, and the join takes 2 us.  Stretches drawn from a common counter instead of equal shares: 39 and 301 us.
constexpr int RW = 4;                       // warps of a CTA
constexpr int RT = 16;                      // rows of a tile, keys of a turn
constexpr int RB = 512;                     // sequences of a call: what is known of each lies in shared memory.  More go by tiles of 128 rows: one token each of 512 / 513 / 1024
                                            // sequences of up to 256, 10 heads of 128, 68 / 139 / 270 us
constexpr int RC = 1;                       // turns that getting to a tile counts for

__device__ __forceinline__ void mma_bf16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool pair_not_finite(uint32_t u) { return (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u; }

struct RowsArgs {
  const __nv_bfloat16* q;     // [N, H * D]
  const __nv_bfloat16 *k, *v;
  Paged p;
  __nv_bfloat16* y;           // [N, H * D]
  const int* doc_start;       // [N] or null
  int window_tiles;
  float c1, c2;               // scale log2 e, |scale| D log2 e
  long long* before;          // [B + 1]: turns of the sequences before
  int* first;                 // [B]: the first key that one of the sequence's rows sees, a multiple of 16
  float* parts;               // [warps][2][RT][D + 4]: sums of the tile that a warp's turns begin in and of the one that they end in
  int warps;
};

__device__ __forceinline__ int paged_first_key(const RowsArgs& p, int row, int pos) {
  int lo = p.doc_start ? max(p.doc_start[row], 0) : 0;
  if (p.window_tiles > 0) lo = max(lo, ((pos >> 7) - (p.window_tiles - 1)) * 128);
  return lo;
}
// What tile t of a piece whose first row is `ahead` keys behind the first key counts for: RC and its turns, to the end of its last row; 0 without keys.
__device__ __forceinline__ int tile_turns(int ahead, int live, int t) {
  const int n = max(ahead + min(live, (t + 1) * RT) + RT - 1, 0) / RT;
  return n ? n + RC : 0;
}
// and of all tiles in front of t
__device__ __forceinline__ int turns_before(int ahead, int live, int t) {
  int n = 0;
  for (int i = 0; i < t; ++i) n += tile_turns(ahead, live, i);
  return n;
}
// A warp's turns: from w * share to below (w + 1) * share
__device__ __forceinline__ long long turn_share(long long total, int warps) { return max((total + warps - 1) / warps, 1ll); }

// Keys and values are read once a step: past the first-level cache, and first to go from the second.  us with plain loads / past the first / so:
// 4 sequences of 32768 to 131072 tokens 297 / 253 / 253 (6.6 TB/s), 64 of up to 2048 32.8 / 29.2 / 26.0.
__device__ __forceinline__ void ld_32(uint32_t* r, const __nv_bfloat16* p) {
  asm volatile("ld.global.nc.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
template <int D>
__device__ __forceinline__ void ld_value(uint32_t* r, const __nv_bfloat16* p) {          // D / 8 consecutive values (loads of 16 bytes have no say in the second)
  if (D == 128) ld_32(r, p);
  else asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
}

// What the CTAs' threads agree on: turns before each sequence.  At most RB sequences.
__device__ __forceinline__ long long rows_plan(const RowsArgs& p, long long* before, int* first, int* heads, Piece* pieces, long long* box) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long total = 0;
  for (int b0 = 0; b0 < p.p.B; b0 += 32 * RW) {
    const int b = b0 + threadIdx.x;
    long long n = 0;
    int f = 0, head = 0;
    if (b < p.p.B) {
      const Piece s = paged_piece(p.p, b);
      pieces[b] = s;
      if (s.live) {
        int lo = 0x7fffffff;
        if (p.doc_start) {
#pragma unroll 4
          for (int i = 0; i < s.live; ++i) lo = min(lo, paged_first_key(p, s.row + i, s.pos + i));
        } else {
          lo = paged_first_key(p, s.row, s.pos);
        }
        f = lo & ~(RT - 1);
        head = turns_before(s.pos - f, s.live, (s.live + RT - 1) / RT);
        n = (long long)p.p.H * head;
      }
    }
    long long up = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    if (lane == 31) box[warp] = up;
    __syncthreads();
    long long front = total;
    for (int w = 0; w < RW; ++w) {
      if (w < warp) front += box[w];
      total += box[w];
    }
    if (b < p.p.B) {
      before[b] = front + up - n;
      first[b] = f;
      heads[b] = head;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) before[p.p.B] = total;
  __syncthreads();
  return total;
}

template <int D>
__global__ void __launch_bounds__(32 * RW, D == 128 ? 3 : 4) paged_rows_kernel(const RowsArgs p) {
  constexpr int KC = D / 64;                // 32-byte pieces of a key that a lane has
  constexpr int NV = D / 8;                 // dimensions of a value that a lane has: tiles of eight output columns
  __shared__ long long before[RB + 1], box[RW];
  __shared__ int first_of[RB], head_of[RB];         // (turns of a head)
  __shared__ Piece piece_of[RB];
  __shared__ uint4 qs_all[RW][KC * 4 * 32];        // a warp's queries: the A operand's registers, lane by lane
  pdl_wait();
  pdl_launch();                              // (the join reads the pieces ahead of its own wait: they are there behind this one's)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const long long A = (long long)p.p.H * D;
  const int mask = (1 << p.p.shift) - 1;
  const long long total = rows_plan(p, before, first_of, head_of, piece_of, box);
  if (blockIdx.x == 0) {                     // for the join
    for (int b = threadIdx.x; b <= p.p.B; b += 32 * RW) {
      p.before[b] = before[b];
      if (b < p.p.B) p.first[b] = first_of[b];
    }
  }
  const int me = blockIdx.x * RW + warp;
  const long long share = turn_share(total, p.warps);
  long long at_turn = me * share;
  const long long end_turn = min(at_turn + share, total);
  uint4* qs = qs_all[warp];
  const uint32_t qs_at = smem_u32(qs + lane);
  while (at_turn < end_turn) {
    // the sequence, head and tile of the turn
    int b = 0;
    for (int n = p.p.B; n > 1;) {
      const int half = n >> 1;
      if (before[b + half] <= at_turn) b += half;
      n -= half;
    }
    const Piece s = piece_of[b];
    const int key0 = first_of[b], ahead = s.pos - key0, a_head = head_of[b];
    const long long in_seq = at_turn - before[b];
    int h, from, t = 0, turns = tile_turns(ahead, s.live, 0);
    if (in_seq >> 31) {                                  // (a division of 64 bits takes ten times one of 32)
      h = (int)(in_seq / a_head);
      from = (int)(in_seq % a_head);
    } else {
      h = (int)((uint32_t)in_seq / (uint32_t)a_head);
      from = (int)((uint32_t)in_seq - (uint32_t)h * (uint32_t)a_head);
    }
    while (from >= turns) {
      from -= turns;
      turns = tile_turns(ahead, s.live, ++t);
    }
    int to = (int)min((long long)turns, from + end_turn - at_turn);
    at_turn += to - from;
    // without what getting there counts for
    from = max(from - RC, 0);
    to -= RC;
    turns -= RC;
    if (to <= from) continue;
    const int live = min(RT, s.live - t * RT), row0 = s.row + t * RT, pos0 = s.pos + t * RT;
    const int* table = p.p.table + b * p.p.ldt;
    uint32_t kr[2][KC][8], vr[4][NV / 2];
    auto page_of = [&](int turn) { return turn < to ? table[(key0 + turn * RT) >> p.p.shift] : -1; };
    auto place = [&](int turn, int id) {
      const long long at = paged_at(p.p, id, h);
      return at < 0 ? at : (at + ((key0 + turn * RT) & mask)) * D;
    };
    auto load_k = [&](long long at) {
      if (at < 0) return;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < KC; ++j) ld_32(kr[i][j], p.k + at + (long long)(8 * i + g) * D + (4 * j + c) * 16);
    };
    auto load_v = [&](long long at) {
      if (at < 0) return;
#pragma unroll
      for (int i = 0; i < 4; ++i) ld_value<D>(vr[i], p.v + at + (long long)(2 * c + (i & 1) + 8 * (i >> 1)) * D + g * NV);
    };
    // All that comes from memory is asked for before any of it is waited for, but for the keys and values, which wait for their page.
    const int id_first = page_of(from);
    int id_next = page_of(from + 1);
    // rows g and g + 8: their positions and first keys
    const int pos_a = g < live ? pos0 + g : -1, pos_b = g + 8 < live ? pos0 + g + 8 : -1;
    const int lo_a = g < live ? paged_first_key(p, row0 + g, pos_a) : 0x7fffffff, lo_b = g + 8 < live ? paged_first_key(p, row0 + g + 8, pos_b) : 0x7fffffff;
    // queries: step (j, i) takes rows g, g + 8 at dimensions 16 (4 j + c) + 4 i + {0, 1} and + {2, 3}; the registers of all steps would leave no room
    // for the keys and values on their way
    uint4 qr[KC * 4];
#pragma unroll
    for (int i = 0; i < KC * 4; ++i) {
      const int r = g + (i & 1) * 8;
      qr[i] = r < live ? *reinterpret_cast<const uint4*>(p.q + (long long)(row0 + r) * A + (long long)h * D + (i >> 2) * 64 + c * 16 + ((i >> 1) & 1) * 8)
                       : make_uint4(0, 0, 0, 0);
    }
    long long at = place(from, id_first);
    load_k(at);
    load_v(at);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < KC * 4; ++i) qs[i * 32 + lane] = qr[i];
    __syncwarp();
    const int far = __reduce_max_sync(0xffffffffu, max(g < live ? lo_a : 0, g + 8 < live ? lo_b : 0));
    float o[NV][4], l_a = 0.f, l_b = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    for (int turn = from; turn < to; ++turn) {
      const int k0 = key0 + turn * RT;
      const long long at_next = place(turn + 1, id_next), now = at;
      id_next = page_of(turn + 2);
      at = at_next;
      if (now < 0) {                              // no such page: its positions are not seen
        load_k(at);
        load_v(at);
        continue;
      }
      float sc[2][4] = {};
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          uint32_t x[2][4];                        // rows g and g + 8
#pragma unroll
          for (int r = 0; r < 2; ++r)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[r][0]), "=r"(x[r][1]), "=r"(x[r][2]), "=r"(x[r][3]) : "r"(qs_at + (j * 4 + i + r) * 512));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {x[0][2 * e], x[1][2 * e], x[0][2 * e + 1], x[1][2 * e + 1]};
            mma_bf16_16816(sc[0], a, kr[0][j][2 * (i + e)], kr[0][j][2 * (i + e) + 1]);
            mma_bf16_16816(sc[1], a, kr[1][j][2 * (i + e)], kr[1][j][2 * (i + e) + 1]);
          }
        }
      load_k(at);
      // columns 2 c, 2 c + 1 of both halves
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = fmaf(sc[i][e], p.c1, -p.c2);
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(sc[i][e]) : "f"(x));
        }
      const bool masked = k0 + RT - 1 > pos0 || k0 < far;      // some row does not see some key
      if (masked) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = k0 + 8 * i + 2 * c + (e & 1);
            if (key > (e < 2 ? pos_a : pos_b) || key < (e < 2 ? lo_a : lo_b)) sc[i][e] = 0.f;
          }
      }
      l_a += (sc[0][0] + sc[0][1]) + (sc[1][0] + sc[1][1]);
      l_b += (sc[0][2] + sc[0][3]) + (sc[1][2] + sc[1][3]);
      const uint32_t pr[4] = {pack_bf16(sc[0][0], sc[0][1]), pack_bf16(sc[0][2], sc[0][3]), pack_bf16(sc[1][0], sc[1][1]), pack_bf16(sc[1][2], sc[1][3])};
      if (masked) {
        // a value that is not finite would make NaN of the zeros of rows that do not see it (behind the sequence's end lies what the page held before)
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < NV / 2; ++i) odd |= pair_not_finite(vr[j][i]);
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) {
              uint32_t u = vr[j][i];
              if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
              if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
              vr[j][i] = u;
            }
          for (int j = 0; j < RT; ++j) {          // and goes to those that do
            const int key = k0 + j;
            const bool in_a = key <= pos_a && key >= lo_a, in_b = key <= pos_b && key >= lo_b;
            const __nv_bfloat16* val = p.v + now + (long long)j * D;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float x = __bfloat162float(val[(2 * c + e) * NV + i]);
                if (!isfinite(x)) {
                  if (in_a) o[i][e] += x;
                  if (in_b) o[i][2 + e] += x;
                }
              }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        // dimensions 2 i and 2 i + 1 of this lane's: pairs of keys
        mma_bf16_16816(o[2 * i], pr, __byte_perm(vr[0][i], vr[1][i], 0x5410), __byte_perm(vr[2][i], vr[3][i], 0x5410));
        mma_bf16_16816(o[2 * i + 1], pr, __byte_perm(vr[0][i], vr[1][i], 0x7632), __byte_perm(vr[2][i], vr[3][i], 0x7632));
      }
      load_v(at);
    }
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    // a lane has dimensions 2 c NV .. 2 (c + 1) NV of rows g and g + 8
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = g + 8 * half;
      const float l = half ? l_b : l_a;
      if (r >= live) continue;
      if (from == 0 && to == turns) {                // all of the tile's
        const float inv = l == 0.f ? 0.f : 1.0f / l;       // a row that sees no key has zeros
        __nv_bfloat16* y = p.y + (long long)(row0 + r) * A + (long long)h * D + 2 * c * NV;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < NV; i += 8) {
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = pack_bf16(o[i + 2 * k][2 * half + e] * inv, o[i + 2 * k + 1][2 * half + e] * inv);
            *reinterpret_cast<uint4*>(y + e * NV + i) = make_uint4(u[0], u[1], u[2], u[3]);
          }
      } else {
        float* part = p.parts + (((long long)me * 2 + (from > 0 ? 0 : 1)) * RT + r) * (D + 4);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < NV; i += 4)
            *reinterpret_cast<float4*>(part + (2 * c + e) * NV + i) =
                make_float4(o[i][2 * half + e], o[i + 1][2 * half + e], o[i + 2][2 * half + e], o[i + 3][2 * half + e]);
        if (c == 0) part[D] = l;
      }
    }
  }
}

// Adds a row's sums where several warps have some, in their order; zeros for rows without a result.  256 threads take D / 4 threads' worth of rows and
// heads, G groups of threads for each: eight where there are few (44 warps share a head of a long cache).
template <int D, int G>
__global__ void __launch_bounds__(256) paged_rows_join_kernel(const RowsArgs p) {
  constexpr int T = D / 4, PAIRS = 256 / (T * G);
  __shared__ float4 box[G > 1 ? G : 1][PAIRS][T];
  __shared__ float box_l[G > 1 ? G : 1][PAIRS];
  const int pair = threadIdx.x / (T * G), group = threadIdx.x / T % G, d = threadIdx.x % T;
  const long long item = (long long)blockIdx.x * PAIRS + pair;
  const bool on = item < (long long)p.p.N * p.p.H;
  // (a warp's two rows are looked up one after the other where a row has less than a warp's threads)
  const int row = on ? (int)(item / p.p.H) : -1, h = on ? (int)(item % p.p.H) : 0;
  int b = -1;
#pragma unroll
  for (int i = 0; i < 32; i += min(T * G, 32)) {
    const int x = paged_owner(p.p.starts, p.p.B, __shfl_sync(0xffffffffu, row, i));
    if ((int)(threadIdx.x & 31) >= i) b = x;
  }
  Piece s = {};
  if (on && b >= 0 && b < p.p.B) s = paged_piece(p.p, b);
  const int i = row - s.row, tile = i / RT;
  const bool live = on && s.live && i >= 0 && i < s.live;
  pdl_wait();
  pdl_launch();
  bool written = !on;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (live) {
    const long long in_front = p.before[b], total = p.before[p.p.B];
    const int ahead = s.pos - p.first[b], turns = tile_turns(ahead, s.live, tile);
    if (turns > 0) {
      const long long from = in_front + (long long)h * turns_before(ahead, s.live, (s.live + RT - 1) / RT) + turns_before(ahead, s.live, tile);
      const long long share = turn_share(total, p.warps);
      const int w0 = (int)((from + RC) / share), w1 = (int)((from + turns - 1) / share);
      written = w0 == w1;
      if (!written) {
        // the first warp's second place, the others' first
        const float* at = p.parts + (long long)(i % RT) * (D + 4);
        constexpr int STEP = RT * (D + 4);
#pragma unroll 4
        for (int w = w0 + group; w <= w1; w += G) {
          const float* y = at + (long long)(2 * w + (w == w0)) * STEP;
          const float4 z = *reinterpret_cast<const float4*>(y + 4 * d);
          x.x += z.x;
          x.y += z.y;
          x.z += z.z;
          x.w += z.w;
          l += y[D];
        }
      }
    }
  }
  if (G > 1) {
    box[group][pair][d] = x;
    if (d == 0) box_l[group][pair] = l;
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int k = 1; k < G; ++k) {
      const float4 z = box[k][pair][d];
      x.x += z.x;
      x.y += z.y;
      x.z += z.z;
      x.w += z.w;
      l += box_l[k][pair];
    }
  }
  if (written) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<uint2*>(p.y + ((long long)row * p.p.H + h) * D + 4 * d) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
}

// Whether a call goes by tiles of 16 rows: one of few tokens, whose turns of a head keep to 32 bits whatever lies in the pieces
static bool by_rows(int B, int N, int cap, int tall) { return !tall && B <= RB && (N / RT + 1ll) * (cap / RT + 1 + RC) < 1ll << 31; }

// CTAs that share a step's turns: what the SMs hold
static int rows_ctas(int D, int sms) { return (D == 128 ? 3 : 4) * sms; }

template <int D>
static int launch_rows(RowsArgs& p, int ctas, cudaStream_t s) {
  p.warps = ctas * RW;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(32 * RW);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  BONES_CHECK(cudaLaunchKernelEx(&cfg, paged_rows_kernel<D>, (const RowsArgs&)p));
  const long long pairs = (long long)p.p.N * p.p.H;
  const bool few = pairs <= 8 * ctas;
  const int a_cta = 256 / (D / 4 * (few ? 8 : 1));
  cfg.gridDim = dim3((unsigned)((pairs + a_cta - 1) / a_cta));
  cfg.blockDim = dim3(256);
  return (int)(few ? cudaLaunchKernelEx(&cfg, paged_rows_join_kernel<D, 8>, p) : cudaLaunchKernelEx(&cfg, paged_rows_join_kernel<D, 1>, p));
}

}  // namespace bones

extern "C" {
using namespace bones;

long long bones_paged_room(int B, int N, int cap, int H, int D, int window_tiles, int tall, int sms);

// qkv: bf16 rows of 3 * H * D, ldq apart; cosT, sinT: fp32 [rope_rows, D / 2]; k, v: bf16 [pages, H, 1 << shift, D] on 32 bytes; table: int32 [B, M],
// rows ldt apart; starts: int32 [B + 1]; pos: int32 [B]; q: bf16 [N, H * D].
int bones_paged_append(const void* qkv, long long ldq, const float* cosT, const float* sinT, int rope_rows, void* k, void* v, int pages, const int* table,
                       long long ldt, const int* starts, const int* pos, int B, int N, int M, int H, int D, int shift, void* q, void* stream) {
  const Paged p{starts, pos, table, ldt, B, N, M, H, shift, pages, (int)min((long long)M << shift, 0x7fffff80ll), v};
  if (paged_refused(B, N, M, H, D, shift, pages, ldt, k, v, starts, pos, table) || !qkv || !q || !cosT || !sinT || rope_rows < 0 || misaligned16(qkv, q, cosT, sinT) || (N > 1 && ldq % 8)) return -2;
  if (N == 0) return 0;
  int dev = 0, sms = 0;
  BONES_CHECK(cudaGetDevice(&dev));
  BONES_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int rows = (int)max(1ll, min((long long)AR, N / (4ll * sms)));
  const unsigned grid = (unsigned)((N + rows - 1) / rows);
  const auto* x = (const __nv_bfloat16*)qkv;
  auto *kc = (__nv_bfloat16*)k, *vc = (__nv_bfloat16*)v, *out = (__nv_bfloat16*)q;
  cudaStream_t s = (cudaStream_t)stream;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(AT);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  return (int)(D == 128 ? cudaLaunchKernelEx(&cfg, paged_append_kernel<128>, x, ldq, cosT, sinT, rope_rows, rows, p, kc, vc, out)
                        : cudaLaunchKernelEx(&cfg, paged_append_kernel<64>, x, ldq, cosT, sinT, rope_rows, rows, p, kc, vc, out));
}

// q, y: bf16 [N, H * D]; doc_start: int32 [N] or null; window_tiles: of 128 tokens, 0 for all; tall: by tiles of 128 rows (pieces of more than a few tokens),
// which calls of more than 512 sequences take in any case, and those of some thousand tokens or more over the longest caches; work: of this call alone until it ends, on 32 bytes, as many as bones_paged_room says.
int bones_paged_attention(const void* q, const void* k, const void* v, int pages, const int* table, long long ldt, const int* starts, const int* pos,
                          const int* doc_start, void* y, int B, int N, int M, int H, int D, int shift, float scale, int window_tiles, int tall, void* work,
                          long long room, void* stream) {
  if (paged_refused(B, N, M, H, D, shift, pages, ldt, k, v, starts, pos, table) || !q || !y || (((uintptr_t)q | (uintptr_t)y | (uintptr_t)work) & 31) ||
      window_tiles < 0 || !work)
    return -2;
  if (N == 0) return 0;
  int dev = 0, sms = 0;
  BONES_CHECK(cudaGetDevice(&dev));
  BONES_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const Paged p{starts, pos, table, ldt, B, N, M, H, shift, pages, (int)min((long long)M << shift, 0x7fffff80ll), v};
  window_tiles = min(window_tiles, MOST_WINDOW);
  if (room < bones_paged_room(B, N, p.cap, H, D, window_tiles, tall, sms)) return -2;
  if (!by_rows(B, N, p.cap, tall)) return paged_pieces(q, k, p, doc_start, y, D, scale, window_tiles, sms, work, stream);
  const float log2e = 1.4426950408889634f;
  const int ctas = rows_ctas(D, sms);
  float* parts = (float*)work;
  long long* before = (long long*)(parts + (long long)ctas * RW * 2 * RT * (D + 4));
  RowsArgs a{(const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, p, (__nv_bfloat16*)y, doc_start, window_tiles,
             scale * log2e, (scale < 0 ? -scale : scale) * D * log2e, before, (int*)(before + B + 1), parts, 0};
  return D == 128 ? launch_rows<128>(a, ctas, (cudaStream_t)stream) : launch_rows<64>(a, ctas, (cudaStream_t)stream);
}

// Bytes of bones_paged_attention's `work` on a device of `sms` SMs (0: the current one; below 0: an error), for caches of `cap` tokens a sequence.
long long bones_paged_room(int B, int N, int cap, int H, int D, int window_tiles, int tall, int sms) {
  int dev = 0;
  if (sms <= 0 && (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)) return -1;
  if (!by_rows(B, N, cap, tall)) return paged_pieces_room(B, N, cap, H, D, min(window_tiles, MOST_WINDOW), sms);
  return (long long)rows_ctas(D, sms) * RW * 2 * RT * (D + 4) * 4 + 12ll * B + 16;
}
}  // extern "C"
