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

__device__ __forceinline__ void paged_ld8(const __nv_bfloat16* p, float* f) { unpack8(*reinterpret_cast<const uint4*>(p), f); }
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

// A warp takes 512 / D heads of one row, so the row's sequence, page and angles are looked up once a warp.
template <int D>
__global__ void __launch_bounds__(256) paged_append_kernel(const __nv_bfloat16* __restrict__ qkv, long long ldq, const float* __restrict__ cosT,
                                                           const float* __restrict__ sinT, int rope_rows, const Paged p, __nv_bfloat16* __restrict__ k,
                                                           __nv_bfloat16* __restrict__ v, __nv_bfloat16* __restrict__ q) {
  constexpr int LANES = D / 16, HEADS = 32 / LANES, HALF = D / 2;
  const int parts = (p.H + HEADS - 1) / HEADS;
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, l8 = lane % LANES;
  if (w >= (long long)p.N * parts) return;
  const int row = (int)(w / parts), h = (int)(w % parts) * HEADS + lane / LANES;
  const bool on = h < p.H;
  const long long A = (long long)p.H * D, col = (long long)(on ? h : 0) * D + l8 * 8;
  // the row itself is on its way while its place is looked up
  const __nv_bfloat16* src = qkv + row * ldq + col;
  float a[3][8], b[3][8];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    paged_ld8(src + i * A, a[i]);
    paged_ld8(src + i * A + HALF, b[i]);
  }
  const int seq = paged_owner(p.starts, p.B, row);
  long long at = -1;
  int t = -1;
  if (seq >= 0 && seq < p.B) {
    const Piece s = paged_piece(p, seq);
    const int i = row - s.row;
    if (i >= 0 && i < s.live && s.pos + i < rope_rows) {
      t = s.pos + i;
      at = paged_at(p, p.table[seq * p.ldt + (t >> p.shift)], on ? h : 0);
    }
  }
  __nv_bfloat16* out = q + row * A + col;
  if (t < 0) {                                       // not a new token, or left out
    if (on) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(out + HALF) = make_uint4(0, 0, 0, 0);
    return;
  }
  float cs[8], sn[8], y1[8], y2[8];
  paged_ld8f(cosT + (long long)t * HALF + l8 * 8, cs);
  paged_ld8f(sinT + (long long)t * HALF + l8 * 8, sn);
  paged_turn<D>(a[0], b[0], cs, sn, y1, y2);
  if (on) {
    paged_st8(out, y1);
    paged_st8(out + HALF, y2);
  }
  paged_turn<D>(a[1], b[1], cs, sn, y1, y2);
  if (on && at >= 0) {
    const long long o = (at + (t & ((1 << p.shift) - 1))) * D + l8 * 8;
    paged_st8(k + o, y1);
    paged_st8(k + o + HALF, y2);
    paged_st8(v + o, a[2]);
    paged_st8(v + o + HALF, b[2]);
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
constexpr int RW = 4;                       // warps of a CTA
constexpr int RT = 16;                      // rows of a tile, keys of a turn

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
  float* parts;               // PARTS: [N, H, gridDim.x, D + 4]
  int turns;                  // PARTS: turns of a part
};

__device__ __forceinline__ int paged_first_key(const RowsArgs& p, int row, int pos) {
  int lo = p.doc_start ? max(p.doc_start[row], 0) : 0;
  if (p.window_tiles > 0) lo = max(lo, ((pos >> 7) - (p.window_tiles - 1)) * 128);
  return lo;
}

// Where a tile's keys lie: `first` (a multiple of 16) and `turns` of 16 keys.
struct TileKeys {
  int first, turns;
};

template <int D>
__device__ __forceinline__ void ld_row(uint32_t* r, const __nv_bfloat16* p) {          // D / 8 consecutive values, 32 bytes (16 of heads of 64)
  if (D == 128) {
    uint4 a, b;
    ld_global_v8(p, a, b);
    r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w; r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
  }
}

// grid: (CTAs of a head, H, B + 1): the last layer clears the rows that belong to no sequence.  PARTS: each CTA of a head takes `turns` turns of
// its keys and leaves sums; else the CTAs are a cluster that shares the turns equally and joins its sums through distributed shared memory.
template <int D, bool PARTS>
__global__ void __launch_bounds__(32 * RW, 3) paged_rows_kernel(const RowsArgs p) {
  constexpr int KC = D / 64;                // 32-byte pieces of a key a lane has
  constexpr int NV = D / 8;                 // dimensions of a value a lane has: tiles of eight output columns
  constexpr int LD = D + 4;                 // a row of sums: column d at d + d / 32, so that a warp's stores meet no bank twice
  extern __shared__ __align__(16) float red[];   // [RW][RT][LD] sums, [RW][RT] sums of weights, the CTA's own [RT][LD] and [RT], the queries
  float* red_l = red + RW * RT * LD;
  float* own = red_l + RW * RT;
  float* own_l = own + RT * LD;
  uint4* qs = reinterpret_cast<uint4*>(own_l + RT);        // [KC][4][32]: the A operand's registers, lane by lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, seq = blockIdx.z;
  const long long A = (long long)p.p.H * D;
  const int S = gridDim.x, rank = blockIdx.x;
  if (seq == p.p.B) {                       // (the whole cluster is here)
    const int head = min(max(p.p.starts[0], 0), p.p.N), tail = min(max(p.p.starts[p.p.B], head), p.p.N);
    for (int r = rank; r < head + p.p.N - tail; r += S) {
      const int row = r < head ? r : tail + r - head;
      for (int d = threadIdx.x; d < D; d += 32 * RW) p.y[row * A + (long long)h * D + d] = __float2bfloat16(0.f);
    }
    return;
  }
  const Piece s = paged_piece(p.p, seq);
  const int* table = p.p.table + seq * p.p.ldt;
  const int mask = (1 << p.p.shift) - 1;
  for (int t0 = 0; t0 < s.len; t0 += RT) {
    const int n = min(RT, s.len - t0), live = min(max(s.live - t0, 0), n), row0 = s.row + t0, pos0 = s.pos + t0;
    // rows g and g + 8 of the tile: their positions and first keys
    const int pos_a = g < live ? pos0 + g : -1, pos_b = g + 8 < live ? pos0 + g + 8 : -1;
    const int lo_a = g < live ? paged_first_key(p, row0 + g, pos_a) : 0x7fffffff, lo_b = g + 8 < live ? paged_first_key(p, row0 + g + 8, pos_b) : 0x7fffffff;
    const int lo = __reduce_min_sync(0xffffffffu, min(lo_a, lo_b)), hi_lo = __reduce_max_sync(0xffffffffu, max(g < live ? lo_a : 0, g + 8 < live ? lo_b : 0));
    const int first = lo & ~(RT - 1), end = live ? pos0 + live : 0;       // keys first .. end
    const int turns = end > first ? (end - first + RT - 1) / RT : 0;
    // this warp's turns: `from`, from + step, ... below `to`
    const int from = PARTS ? rank * p.turns + warp : rank * RW + warp, step = PARTS ? RW : S * RW, to = PARTS ? min(turns, (rank + 1) * p.turns) : turns;
    // queries: step (j, i) takes rows g, g + 8 at dimensions 16 (4 j + c) + 4 i + {0, 1} and + {2, 3}; the registers of all steps would leave no room
    // for the keys and values on their way
    for (int i = warp; i < KC * 4; i += RW) {
      const int r = g + (i & 1) * 8;
      qs[i * 32 + lane] = r < live ? *reinterpret_cast<const uint4*>(p.q + (long long)(row0 + r) * A + (long long)h * D + (i >> 2) * 64 + c * 16 + ((i >> 1) & 1) * 8)
                                   : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    float o[NV][4], l_a = 0.f, l_b = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    if (from < to) {
      uint32_t kr[2][KC][8], vr[4][NV / 2];
      auto page_of = [&](int turn) { return turn < to ? table[(first + turn * RT) >> p.p.shift] : -1; };
      auto place = [&](int turn, int id) {
        const long long at = paged_at(p.p, id, h);
        return at < 0 ? at : (at + ((first + turn * RT) & mask)) * D;
      };
      auto load_k = [&](long long at) {
        if (at < 0) return;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < KC; ++j) ld_row<128>(kr[t][j], p.k + at + (long long)(8 * t + g) * D + (4 * j + c) * 16);
      };
      auto load_v = [&](long long at) {
        if (at < 0) return;
#pragma unroll
        for (int t = 0; t < 4; ++t) ld_row<D>(vr[t], p.v + at + (long long)(2 * c + (t & 1) + 8 * (t >> 1)) * D + g * NV);
      };
      const uint32_t qs_at = smem_u32(qs + lane);
      long long at = place(from, page_of(from));
      load_k(at);
      load_v(at);
      int id_next = page_of(from + step);
      for (int turn = from; turn < to; turn += step) {
        const int k0 = first + turn * RT;
        const long long at_next = place(turn + step, id_next), now = at;
        id_next = page_of(turn + 2 * step);
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
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = fmaf(sc[t][e], p.c1, -p.c2);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(sc[t][e]) : "f"(x));
          }
        const bool masked = k0 + RT - 1 > pos0 || k0 < hi_lo;      // some row does not see some key
        if (masked) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = k0 + 8 * t + 2 * c + (e & 1);
              if (key > (e < 2 ? pos_a : pos_b) || key < (e < 2 ? lo_a : lo_b)) sc[t][e] = 0.f;
            }
        }
        l_a += (sc[0][0] + sc[0][1]) + (sc[1][0] + sc[1][1]);
        l_b += (sc[0][2] + sc[0][3]) + (sc[1][2] + sc[1][3]);
        const uint32_t pr[4] = {pack_bf16(sc[0][0], sc[0][1]), pack_bf16(sc[0][2], sc[0][3]), pack_bf16(sc[1][0], sc[1][1]), pack_bf16(sc[1][2], sc[1][3])};
        if (masked) {
          // a value that is not finite would make NaN of the zeros of rows that do not see it (behind the sequence's end lies what the page held before)
          uint32_t odd = 0;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) odd |= pair_not_finite(vr[t][i]);
          if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int i = 0; i < NV / 2; ++i) {
                uint32_t u = vr[t][i];
                if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
                if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
                vr[t][i] = u;
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
    }
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    // warps of the CTA, in their order
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = (2 * c + e) * NV + i;
        if (g < live) red[(warp * RT + g) * LD + d + (d >> 5)] = o[i][e];
        if (g + 8 < live) red[(warp * RT + g + 8) * LD + d + (d >> 5)] = o[i][2 + e];
      }
    if (c == 0) {
      red_l[warp * RT + g] = l_a;
      red_l[warp * RT + g + 8] = l_b;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < live * D; i += 32 * RW) {
      const int d = i % D, at = i / D * LD + d + (d >> 5);
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < RW; ++w) x += red[w * RT * LD + at];
      if (PARTS) {
        if (rank * p.turns < turns) p.parts[(((long long)(row0 + i / D) * p.p.H + h) * S + rank) * (D + 4) + d] = x;
      } else {
        own[at] = x;
      }
    }
    if (threadIdx.x < live) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < RW; ++w) x += red_l[w * RT + threadIdx.x];
      if (PARTS) {
        if (rank * p.turns < turns) p.parts[(((long long)(row0 + threadIdx.x) * p.p.H + h) * S + rank) * (D + 4) + D] = x;
      } else {
        own_l[threadIdx.x] = x;
      }
    }
    if (!PARTS) {
      __syncthreads();
      if (S > 1) cluster_barrier();
      // the cluster's CTAs each finish some of the values
      for (int i = rank * 32 * RW + threadIdx.x; i < n * D; i += S * 32 * RW) {
        const int d = i % D;
        float x = 0.f, l = 0.f;
        if (i < live * D) {
          if (S > 1) {
            const uint32_t at_x = smem_u32(own + i / D * LD + d + (d >> 5)), at_l = smem_u32(own_l + i / D);
            for (int r = 0; r < S; ++r) {
              float a, b;
              asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a) : "r"(map_to_rank(at_x, r)));
              asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b) : "r"(map_to_rank(at_l, r)));
              x += a;
              l += b;
            }
          } else {
            x = own[i / D * LD + d + (d >> 5)];
            l = own_l[i / D];
          }
        }
        // a row that sees no key has zeros
        p.y[(long long)(row0 + i / D) * A + (long long)h * D + d] = __float2bfloat16(l == 0.f ? 0.f : x / l);
      }
      __syncwarp();
      if (S > 1) cluster_barrier();             // nobody's sums change or go before all have read them
    }
    __syncthreads();
  }
}

// Joins the parts of a row and head in their order.  grid: (N, H), D threads.
template <int D>
__global__ void __launch_bounds__(D) paged_join_kernel(const RowsArgs p, int S) {
  pdl_wait();
  const int row = blockIdx.x, h = blockIdx.y, d = threadIdx.x;
  const int seq = paged_owner(p.p.starts, p.p.B, row);
  if (seq < 0 || seq >= p.p.B) return;              // cleared already
  const Piece s = paged_piece(p.p, seq);
  const int i = row - s.row;
  if (i < 0 || i >= s.len) return;
  // the turns of the tile that the row was in
  const int t0 = i / RT * RT, live = min(max(s.live - t0, 0), RT), lane = d & 31;
  int lo = 0x7fffffff;
  if (lane < live) lo = paged_first_key(p, s.row + t0 + lane, s.pos + t0 + lane);
  lo = __reduce_min_sync(0xffffffffu, lo);
  const int first = lo & ~(RT - 1), end = live ? s.pos + t0 + live : 0;
  const int turns = end > first ? (end - first + RT - 1) / RT : 0, parts = min((turns + p.turns - 1) / p.turns, S);
  float x = 0.f, l = 0.f;
  if (i < s.live) {
    const float* at = p.parts + ((long long)row * p.p.H + h) * S * (D + 4);
#pragma unroll 8
    for (int r = 0; r < parts; ++r) {
      x += at[r * (D + 4) + d];
      l += at[r * (D + 4) + D];
    }
  }
  p.y[(long long)row * p.p.H * D + (long long)h * D + d] = __float2bfloat16(l == 0.f ? 0.f : x / l);
}

template <int D>
static int launch_rows(const RowsArgs& p, int S, bool parts, cudaStream_t s) {
  constexpr size_t smem = sizeof(float) * (RW * RT * (D + 4) + RW * RT + RT * (D + 4) + RT) + D / 64 * 4 * 32 * 16;
  static OncePerDevice limit;
  BONES_ONCE(limit, {
    BONES_CHECK(cudaFuncSetAttribute(paged_rows_kernel<D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    BONES_CHECK(cudaFuncSetAttribute(paged_rows_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  });
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)S, (unsigned)p.p.H, (unsigned)p.p.B + 1);
  cfg.blockDim = dim3(32 * RW);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, parts ? 1 : S, 0);
  if (!parts) return (int)cudaLaunchKernelEx(&cfg, paged_rows_kernel<D, false>, p);
  BONES_CHECK(cudaLaunchKernelEx(&cfg, paged_rows_kernel<D, true>, p));
  cfg.gridDim = dim3((unsigned)p.p.N, (unsigned)p.p.H);
  cfg.blockDim = dim3(D);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  return (int)cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, p, S);
}

}  // namespace bones

extern "C" {
using namespace bones;

// qkv: bf16 rows of 3 * H * D, ldq apart; cosT, sinT: fp32 [rope_rows, D / 2]; k, v: bf16 [pages, H, 1 << shift, D] on 32 bytes; table: int32 [B, M],
// rows ldt apart; starts: int32 [B + 1]; pos: int32 [B]; q: bf16 [N, H * D].
int bones_paged_append(const void* qkv, long long ldq, const float* cosT, const float* sinT, int rope_rows, void* k, void* v, int pages, const int* table,
                       long long ldt, const int* starts, const int* pos, int B, int N, int M, int H, int D, int shift, void* q, void* stream) {
  const Paged p{starts, pos, table, ldt, B, N, M, H, shift, pages, (int)min((long long)M << shift, 0x7fffff00ll), v};
  if (paged_refused(B, N, M, H, D, shift, pages, ldt, k, v, starts, pos, table) || !qkv || !q || !cosT || !sinT || rope_rows < 0 || misaligned16(qkv, q, cosT, sinT) || (N > 1 && ldq % 8)) return -2;
  if (N == 0) return 0;
  const long long warps = (long long)N * ((H + 512 / D - 1) / (512 / D));
  if (warps > 0x3fffffffll) return -2;
  const unsigned grid = (unsigned)((warps + 7) / 8);
  const auto* x = (const __nv_bfloat16*)qkv;
  auto *kc = (__nv_bfloat16*)k, *vc = (__nv_bfloat16*)v, *out = (__nv_bfloat16*)q;
  cudaStream_t s = (cudaStream_t)stream;
  if (D == 128) paged_append_kernel<128><<<grid, 256, 0, s>>>(x, ldq, cosT, sinT, rope_rows, p, kc, vc, out);
  else paged_append_kernel<64><<<grid, 256, 0, s>>>(x, ldq, cosT, sinT, rope_rows, p, kc, vc, out);
  return (int)cudaGetLastError();
}

// q, y: bf16 [N, H * D]; doc_start: int32 [N] or null; parts: room for part_floats floats on 16 bytes, of this call alone until it ends, or null.
int bones_paged_rows(const void* q, const void* k, const void* v, int pages, const int* table, long long ldt, const int* starts, const int* pos,
                     const int* doc_start, void* y, int B, int N, int M, int H, int D, int shift, float scale, int window_tiles, float* parts,
                     long long part_floats, void* stream) {
  const Paged p{starts, pos, table, ldt, B, N, M, H, shift, pages, (int)min((long long)M << shift, 0x7fffff00ll), v};
  if (paged_refused(B, N, M, H, D, shift, pages, ldt, k, v, starts, pos, table) || !q || !y || (((uintptr_t)q | (uintptr_t)y) & 31) || window_tiles < 0 || misaligned16(parts)) return -2;
  if (N == 0) return 0;
  const float log2e = 1.4426950408889634f;
  RowsArgs a{(const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, p, (__nv_bfloat16*)y, doc_start, window_tiles, scale * log2e,
             (scale < 0 ? -scale : scale) * D * log2e, parts, 0};
  int dev = 0, sms = 0;
  BONES_CHECK(cudaGetDevice(&dev));
  BONES_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const long long heads = (long long)B * H, seen = window_tiles > 0 ? min((long long)p.cap, (window_tiles + 1) * 128ll) : p.cap;
  const long long turns = (seen + RT - 1) / RT;
  // few heads and long caches: parts of their own, ten rounds of CTAs so that unequal lengths even out
  long long S = min(30ll * sms / heads, turns / 64);
  if (parts && S > 8 && (long long)N * H * S * (D + 4) <= part_floats && N <= 65535) {
    a.turns = (int)((turns + S - 1) / S);
    return D == 128 ? launch_rows<128>(a, (int)S, true, (cudaStream_t)stream) : launch_rows<64>(a, (int)S, true, (cudaStream_t)stream);
  }
  int C = 1;
  while (C < 8 && heads * C < 6ll * sms && turns >= 2 * RW * C) C *= 2;
  return D == 128 ? launch_rows<128>(a, C, false, (cudaStream_t)stream) : launch_rows<64>(a, C, false, (cudaStream_t)stream);
}
}  // extern "C"
