// A key/value cache in 8 bits: append, read-back and single-token attention.  Layout (one layer): blocks of 64 tokens; key codes
// [B, H, T, D] and value codes [B, H, T / 64, D, 64] (int8), scales [B, H, T / 64] (fp32), the open block's tokens [B, H, 64, D] (bf16).
//
//   code = rint(x * (127 / most)),  scale = most / 127,  most = the block's largest finite |x|
//
// A value that is not finite gets the code -128, which stands for NaN, and its block a scale with a minus sign, so that blocks
// without one need not look for it.  A block is quantised once, from its 64 bf16 tokens, when it is full.
#include "decode_common.cuh"

#include <cuda_fp16.h>

namespace bones {

constexpr int KB = 64;                          // tokens of a block
constexpr float kKv8Tiny = 7.888609052210118e-31f;   // 2^-100: a block below it is stored as zeros

struct Kv8 {
  int8_t *k, *v;
  float *ks, *vs;
  __nv_bfloat16 *kt, *vt;
};
// a value for each sequence, or one for all
struct PerSeq {
  const int* at;
  int step, value;
  __device__ __forceinline__ int operator[](int b) const { return at ? at[(long long)b * step] : value; }
};

__device__ __forceinline__ float kv8_inverse(float most) { return most >= kKv8Tiny ? 127.0f / most : 0.f; }
// the scale as it is stored; `bad`: the block holds a value that is not finite
__device__ __forceinline__ float kv8_scale(float most, bool bad) { return copysignf(most >= kKv8Tiny ? most / 127.0f : 0.f, bad ? -1.f : 1.f); }
// rint(x * inv) in the low byte: 1.5 * 2^23 is added, which rounds to whole numbers, ties to even
__device__ __forceinline__ uint32_t kv8_code(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f)); }
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ bool is_bad(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }         // a bf16 that is not finite
// byte i of four codes as a number: with its sign bit turned, byte u is the end of 2^23 + u
__device__ __forceinline__ float kv8_number(uint32_t turned, int i) {
  return __uint_as_float(__byte_perm(turned, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
}

constexpr int kTurnRow = KB + 4;                // bytes of a row on its way from [64][D] to [D][64] or back: banks 8 dimensions apart are 8 apart
struct __align__(16) QuantShared {
  float most[8];
  int bad[8];
  uint8_t turn[128 * kTurnRow];
};

// A block is taken in units of four tokens by eight dimensions; 32 lanes are eight by four of them, so that rows are read and written in
// 64-byte pieces and the words of four tokens go to shared memory without conflicts.
template <int D>
__device__ __forceinline__ void kv8_unit(int i, int& token, int& dim) {
  const int lane = i & 31, w = i >> 5;
  token = 4 * (lane >> 2) + 32 * (w & 1);
  dim = 8 * (lane & 3) + 32 * (w >> 1);
}

// A whole block by a CTA of QT threads (256 at most); `piece(token, dim)` is the address of 16 bytes of it.  Key codes go out as they lie,
// value codes through shared memory to be transposed.
template <int QT, int D, bool VALUES, class Piece>
__device__ __forceinline__ void kv8_quantise_block(Piece piece, int8_t* __restrict__ out, float* __restrict__ scale, QuantShared& sm) {
  constexpr int UNITS = 2 * D, N = (UNITS + QT - 1) / QT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint4 u[N][4];
  __nv_bfloat162 top = __nv_bfloat162{__ushort_as_bfloat16(0), __ushort_as_bfloat16(0)};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int t, d;
    kv8_unit<D>(tid + n * QT, t, d);
#pragma unroll
    for (int r = 0; r < 4; ++r) u[n][r] = tid + n * QT < UNITS ? *reinterpret_cast<const uint4*>(piece(t + r, d)) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t w[4] = {u[n][r].x, u[n][r].y, u[n][r].z, u[n][r].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = w[i] & 0x7fff7fffu;
        top = __hmax2_nan(top, *reinterpret_cast<const __nv_bfloat162*>(&a));
      }
    }
  float most = fmaxf(__bfloat162float(top.x), __bfloat162float(top.y));
  const uint32_t tops = *reinterpret_cast<const uint32_t*>(&top);
  bool bad = is_bad(tops) || is_bad(tops >> 16);
  if (bad) {                                    // those that are not finite do not count
    most = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float f[8];
        unpack8(u[n][r], f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (fabsf(f[i]) <= 3.402823466e38f) most = fmaxf(most, fabsf(f[i]));
      }
  }
  most = warp_max(most);
  const bool any = __any_sync(0xffffffffu, bad);
  if (lane == 0) { sm.most[warp] = most; sm.bad[warp] = any; }
  __syncthreads();
  bool marked = false;
#pragma unroll
  for (int w = 0; w < QT / 32; ++w) { most = fmaxf(most, sm.most[w]); marked |= sm.bad[w] != 0; }
  const float inv = kv8_inverse(most);
  if (tid == 0) *scale = kv8_scale(most, marked);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (tid + n * QT >= UNITS) break;
    int t, d;
    kv8_unit<D>(tid + n * QT, t, d);
    uint32_t c[4][8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float f[8];
      unpack8(u[n][r], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[r][i] = kv8_code(f[i], inv);
      if (bad) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(fabsf(f[i]) <= 3.402823466e38f)) c[r][i] = 0x80u;
      }
    }
    if (VALUES) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(sm.turn + (d + i) * kTurnRow + t) = low_bytes(c[0][i], c[1][i], c[2][i], c[3][i]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<uint2*>(out + (t + r) * D + d) =
            make_uint2(low_bytes(c[r][0], c[r][1], c[r][2], c[r][3]), low_bytes(c[r][4], c[r][5], c[r][6], c[r][7]));
    }
  }
  __syncthreads();
  if (VALUES) {
    for (int i = tid; i < D * 4; i += QT) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(sm.turn + (i >> 2) * kTurnRow + (i & 3) * 16);
      *reinterpret_cast<uint4*>(out + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();
  }
}

constexpr int kAppendThreads = 128;
// Bound by bytes: 2 read and 1 written for each value.  4 x 16384 tokens of 10 heads of 128, keys and values, 84 us (6.0 TB/s, 0.91 of the copy
// rate); CTAs of 256 threads, which wait for their slowest load twice as often, 95 to 107.  64 registers a thread, 8 bytes spilled with heads of 128.
// Tokens pos .. pos + len of a sequence.  A CTA takes one block that the run touches, of the keys or of the values of one head; the first
// one also stores what is left over for the open block, after it has read the tokens that were in it before.
template <int D, bool VALUES>
__device__ __forceinline__ void kv8_append_block(const __nv_bfloat16* __restrict__ src, long long st, int8_t* __restrict__ codes, float* __restrict__ scales,
                                                 __nv_bfloat16* __restrict__ tail, int pos, int len, int i, QuantShared& sm) {
  const int first = pos / KB, end = pos + len, blk = first + i;
  if ((long long)(blk + 1) * KB <= end)
    kv8_quantise_block<kAppendThreads, D, VALUES>(
        [&](int t, int d) -> const __nv_bfloat16* {
          const int j = blk * KB + t;
          return j < pos ? tail + t * D + d : src + (long long)(j - pos) * st + d;
        },
        codes + (long long)blk * KB * D, scales + blk, sm);
  if (i == 0) {
    const int open = end / KB * KB, from = max(pos, open);
    for (int p = threadIdx.x; p < (end - from) * (D / 8); p += kAppendThreads) {
      const int j = from + p / (D / 8), d = p % (D / 8) * 8;
      *reinterpret_cast<uint4*>(tail + (j - open) * D + d) = *reinterpret_cast<const uint4*>(src + (long long)(j - pos) * st + d);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kAppendThreads, 8) kv8_append_kernel(Kv8 c, const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, long long kb,
                                                        long long kt, long long kh, long long vb, long long vt, long long vh, PerSeq pos_, PerSeq len_, int t,
                                                        int H, int cap) {
  __shared__ QuantShared sm;
  const int b = blockIdx.z, h = blockIdx.y, i = blockIdx.x >> 1;
  const int pos = pos_[b], len = min(len_[b], t);
  if (pos < 0 || len <= 0 || pos > cap - len || pos / KB + i > (pos + len - 1) / KB) return;
  const long long bh = (long long)b * H + h, nb = cap / KB;
  if (blockIdx.x & 1)
    kv8_append_block<D, true>(v + b * vb + h * vh, vt, c.v + bh * cap * D, c.vs + bh * nb, c.vt + bh * KB * D, pos, len, i, sm);
  else
    kv8_append_block<D, false>(k + b * kb + h * kh, kt, c.k + bh * cap * D, c.ks + bh * nb, c.kt + bh * KB * D, pos, len, i, sm);
}

// One block of one head back to bf16 rows [B, length, H, D]; zeros behind the tokens held.  Bound by bytes, two thirds of them written:
// 4 x 16384 tokens of 10 heads of 128 in 95 us (0.80 of the copy rate; filling the outputs alone takes PyTorch 86).  Heads of 64 are further from
// it (24 x up to 1357 tokens of 4 heads, 13.5 us for 7.6): half of the 256 threads only bring codes to shared memory, and a row is one line.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v, PerSeq held_, int length, int H, int cap) {
  __shared__ __align__(16) uint8_t turn[D * kTurnRow];
  const int b = blockIdx.z, h = blockIdx.y, blk = blockIdx.x >> 1, tid = threadIdx.x;
  const bool values = blockIdx.x & 1;
  const int held = max(held_[b], 0), j0 = blk * KB;
  const long long bh = (long long)b * H + h;
  __nv_bfloat16* out = (values ? v : k) + ((long long)b * length * H + h) * D;
  const bool open = blk == held / KB, some = j0 < held && j0 < cap;
  const int8_t* codes = (values ? c.v : c.k) + (bh * cap + j0) * D;
  const __nv_bfloat16* tail = (values ? c.vt : c.kt) + bh * KB * D;
  const float scale = some && !open ? (values ? c.vs : c.ks)[bh * (cap / KB) + blk] : 0.f, by = fabsf(scale);
  if (values && some && !open) {
    for (int i = tid; i < D * 4; i += 256) {
      const uint4 u = *reinterpret_cast<const uint4*>(codes + i * 16);
      uint32_t* w = reinterpret_cast<uint32_t*>(turn + (i >> 2) * kTurnRow + (i & 3) * 16);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    }
    __syncthreads();
  }
  if (tid >= 2 * D) return;
  // four tokens by eight dimensions a thread, whole rows a warp: what is written counts for more than the conflicts (four ways) of what is read
  const int d = tid % (D / 8) * 8, t = tid / (D / 8) * 4;
  uint32_t w[4][2];                             // codes of four tokens by eight dimensions: by token, or four tokens to a word
  uint32_t x[8];
  if (some && !open) {
    if (values) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint32_t*>(turn + (d + i) * kTurnRow + t) ^ 0x80808080u;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint2 u = *reinterpret_cast<const uint2*>(codes + (t + r) * D + d);
        w[r][0] = u.x ^ 0x80808080u;
        w[r][1] = u.y ^ 0x80808080u;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = j0 + t + r;
    if (j >= length) break;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (some && j < held) {
      if (open) {
        o = *reinterpret_cast<const uint4*>(tail + (t + r) * D + d);
      } else {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = values ? kv8_number(x[i], r) : kv8_number(w[r][i >> 2], i & 3);
          f[i] = n * by;
          if (signbit(scale) && n == -128.0f) f[i] = __int_as_float(0x7fc00000);
        }
        o = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
      }
    }
    *reinterpret_cast<uint4*>(out + (long long)j * H * D + d) = o;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Attention.  Per (head, sequence) a cluster of up to 16 CTAs; a warp takes 4 KB of keys and of values, half a block of 128
// dimensions or a block of 64, at a time,
//
//   s_t = scale ks sum_d q_d k_td,   m' = max(m, s),   p_t = 2^(s_t - m'),   o = o 2^(m - m') + vs sum_t p_t v_td,
//
// and keeps its own maximum, sum and output; the warps', then the CTAs' (through distributed shared memory, no workspace) are
// joined at the end.  Both sums are matrix products (mma.sync m16n8k16: codes as fp16, which holds them exactly, times one column;
// tcgen05 would want its operands in shared memory and 64 rows of queries, and there is one): the codes' rows are the MMA's rows,
// and a lane's consecutive bytes of a row are its columns of several MMAs, so that codes go from memory to the operands with
// two byte permutations and two subtractions for four of them.  The query is two fp16 numbers, hi and lo, in alternate columns of
// B: the scores lose nothing to it.  Probabilities go into the second product as fp16, times 2^15, so that the largest is in
// its top range: rounded by half of 2^-10 of each at most, in both directions, far below the rounding of the result to bf16, down to 2^-29
// of the largest, and gone below 2^-40 (unscaled 2^-25: with one key far above 2000 others a quarter of what they weigh was lost); the
// sum that the result is divided by is of the unrounded ones in fp32.
//
// Bound by the bytes of the codes where there are enough turns for every warp: 4 sequences of 131000 tokens, 10 heads, 213 us (6.3
// TB/s, 0.96 of the copy rate; before the CTAs shared all of it equally 240), 64 of 8192 224 (0.91).  A turn is about 2000 clocks of a warp
// that is alone on its scheduler (one CTA takes 21 us for 2040 tokens, 5.8 for 300) and 600 instructions, the two loads' latencies between
// them; three to a scheduler hide that.  Few or short sequences are bound by one turn after the other and by the way in and out (4.9 us for 300 tokens).
// The token that fills a block costs 4 us more (32 sequences of up to 1536 tokens, 10 heads: 26.7 for 22.6): its codes are made last, those of the
// keys before those of the values, by one CTA a head.  Heads of 128 take 161 or 163 of 168 registers; two of the three forms for heads of 64 spill
// 8 and 16 bytes at 128.  Taken before it: a block of 64 tokens a turn and two CTAs an SM (4 x 131000 273 us, 64 sequences of 64 tokens
// 17.4 for 10.3); the codes through shared memory, by each warp's own cp.async (250) or by bulk copies for the CTA (259), which cost the walk more instructions than the deeper prefetch saved; four CTAs an SM, whose 128 registers spill (248); equal
// runs of turns for one CTA after the other over the ends of heads, for many heads (64 sequences up to 2048 tokens, 10 heads: 48 for 40, all of
// 2048 72 for 75: each CTA's heads wait for one another's way in and out, where CTAs of one head overlap).
// ---------------------------------------------------------------------------------------------------------------
constexpr int kMaxSplit = 16;                   // CTAs of a cluster
constexpr int kFlatFrom = 16384;                // tokens
constexpr int kFlatTurns = 2;                   // turns of each warp of a CTA of equal shares, at least
constexpr float kLift = 15.f, kDrop = 1.f / 32768.f;       // of probabilities while they are fp16, and back

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four codes as two pairs of fp16: with the sign bit turned, byte u below 0x64 is 1024 + u, and u = code + 128
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));          // 1152
  uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
  lo = *reinterpret_cast<uint32_t*>(&x);
  hi = *reinterpret_cast<uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The other half of a line is the neighbouring warp's: the whole line comes to L2.
__device__ __forceinline__ void ld_stream(uint32_t (&w)[4], const void* p) {
  asm volatile("ld.global.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}
__device__ __forceinline__ void ld_stream(uint32_t (&w)[2], const void* p) {
  asm volatile("ld.global.L1::no_allocate.L2::128B.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
}
// bytes of `w` that are -128, as the top bits of theirs
__device__ __forceinline__ uint32_t bad_codes(uint32_t w) { return __vcmpeq4(w, 0x80808080u) & 0x80808080u; }

// 1 / sqrt(x), by Newton's steps to the rounding of the type (two where it is 64 bits), of what fits fp32 or is brought there by an even power of 2
__device__ __forceinline__ float inverse_root(float x) {
  const float r = rsqrtf(x);
  return r * (1.5f - 0.5f * x * r * r);
}
__device__ __forceinline__ double inverse_root(double x) {
  const bool far = x > 1e30;
  const double y = far ? x * 7.174648137343064e-43 : x;
  double r = (double)rsqrtf((float)y);
#pragma unroll
  for (int i = 0; i < 2; ++i) r *= 1.5 - 0.5 * y * r * r;
  return y > 3.4e38 ? 0.0 : far ? r * 8.470329472543003e-22 : r;           // of an infinite value: a step of Newton's would make it NaN
}
// RoPE of a row by a warp, and what norm multiplies it by: dimensions lane + 32 i of the first half in `a`, their partners in `e`.
template <int D, class T>
__device__ __forceinline__ T turn_and_norm(const __nv_bfloat16* __restrict__ x, const float* __restrict__ cs, const float* __restrict__ sn, T (&a)[D / 64],
                                           T (&e)[D / 64]) {
  const int lane = threadIdx.x & 31;
  auto turn = [&](T by) {                                          // the mean of the squares of `by` times the row
    T ss = 0;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int d = lane + 32 * i;
      const T x0 = (T)__bfloat162float(x[d]) * by, x1 = (T)__bfloat162float(x[d + D / 2]) * by, c = (T)cs[d], s = (T)sn[d];
      a[i] = x0 * c + x1 * s;
      e[i] = x1 * c - x0 * s;
      ss += a[i] * a[i] + e[i] * e[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return ss * (T)(1.0 / D);
  };
  T ss = turn((T)1) + (T)1.1920928955078125e-07;
  // squares beyond fp32 (values from 1e18 on): 2^-70 of the row, beside which the epsilon counts for nothing; 64 bits hold them
  if (sizeof(T) == 4 && !(ss <= (T)3.402823466e38f)) ss = turn((T)8.470329472543003e-22);
  return inverse_root(ss);
}

// The sequence with the n-th largest number of tokens to see, of 64 at most: CTAs begin in the order of their numbers, and the longest ones
// are not to begin last (64 sequences of 1 to 2048 tokens in documents, 10 heads: 30 us for 35; where all
// are alike it costs the look, 12.3 for 11.3 at 64 tokens each).  Every warp works it out for itself, from what nothing writes meanwhile:
// not where the kernel before this one may still run.
__device__ __forceinline__ int longest_first(int B, int n, PerSeq pos, const int* __restrict__ doc_start) {
  const int lane = threadIdx.x & 31;
  uint32_t key[2], most = 0, least = ~0u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = lane + 32 * i;
    const int p = b < B ? pos[b] : -1, lo = b < B && doc_start ? doc_start[b] : 0;
    const uint32_t len = (uint32_t)min(max(p - max(lo, 0) + 1, 0), 1 << 25);
    if (b < B) { most = max(most, len); least = min(least, len); }
    key[i] = b < B ? len << 6 | (uint32_t)(63 - b) : 0u;             // no two are equal
  }
  if (__reduce_max_sync(0xffffffffu, most) - __reduce_min_sync(0xffffffffu, least) < 2 * KB) return n;         // much the same length
  int r0 = 0, r1 = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const uint32_t k = __shfl_sync(0xffffffffu, key[0], j);
    r0 += k > key[0];
    r1 += k > key[1];
  }
  if (B > 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const uint32_t k = __shfl_sync(0xffffffffu, key[1], j);
      r0 += k > key[0];
      r1 += k > key[1];
    }
  }
  const unsigned a = __ballot_sync(0xffffffffu, lane < B && r0 == n), c = __ballot_sync(0xffffffffu, lane + 32 < B && r1 == n);
  return a ? __ffs(a) - 1 : 31 + __ffs(c);
}

template <int D, int AW>
struct __align__(16) AttnShared {
  float acc[2 * AW][D];                         // full blocks of each warp, then the open block's part of each
  float part[kMaxSplit][D + 4];                 // every CTA's output, sum and maximum, in the first CTA
  float q[D];
  __nv_bfloat16 fresh[2][D];                    // the new token's key and value
  float m[2 * AW], l[2 * AW];
};

// Long caches (`FLAT`): as many CTAs as the SMs hold share all turns of all heads and sequences, and a second kernel joins what they have,
// instead of a cluster for each.  CTAs of each head that sequence `lane` gets (32 sequences at most); 0 for a sequence outside, and
// `places` in all at most: a head gets one CTA more than its part of places - B H.  Warps of both kernels work it out alike.  us by
// clusters / shares, 10 heads: 131000 tokens 93 / 59 (0.87 of the copy rate), 32700 27 / 22, 3000 in a cache of 32768 8.0 / 10.1; 4 sequences of
// 131000 248 / 213 (0.96), of 32768 to 131072 157 / 148; 16 of 16300 128 / 129, of 1000 to 16000 90 / 68; 4 heads of 64, 131000 tokens 44 / 20.
// A CTA takes every n-th turn: a stretch for each is 3 to 7 % slower.  Two turns of each warp at least: four, 12.7 us for 10.1 of those 3000.
template <int TT, int AW>
__device__ __forceinline__ int flat_ctas(int B, int H, int places, PerSeq pos_, const int* __restrict__ doc_start, int limit, int window_tiles) {
  const int b = threadIdx.x & 31, p = b < B ? pos_[b] : -1;
  int turns = -1;
  if (p >= 0 && p < limit) {
    const int lo = max(doc_start ? ld_relaxed(doc_start + b) : 0, window_tiles > 0 ? max((p / 128 - (window_tiles - 1)) * 128, 0) : 0);
    turns = max(p / KB * (KB / TT) - lo / TT, 0);
  }
  long long all = max(turns, 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  const long long room = (long long)(places - B * H) * AW;
  const int share = (int)max((all * H + room - 1) / room, (long long)kFlatTurns) * AW;
  return turns < 0 ? 0 : max((turns + share - 1) / share, 1);
}
// CTA `n` of all: its sequence in `b` (none: B), its number among that sequence's CTAs in `n`, their number for each head in `ctas`.
__device__ __forceinline__ void flat_place(int mine, int H, int B, int& n, int& b, int& ctas) {
  const int lane = threadIdx.x & 31;
  int upto = mine * H;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  const unsigned who = __ballot_sync(0xffffffffu, upto > n);
  b = who ? __ffs(who) - 1 : B;
  ctas = __shfl_sync(0xffffffffu, mine, b & 31);
  n -= __shfl_sync(0xffffffffu, upto, b & 31) - ctas * H;
}

template <int D, int AW, bool FLAT>
__global__ void __launch_bounds__(32 * AW, (D == 128 ? 12 : 16) / AW) kv8_attn_kernel(const __nv_bfloat16* __restrict__ qkv, long long ldq, const float* __restrict__ cosT,
                                                              const float* __restrict__ sinT, int rope_rows, Kv8 c, PerSeq pos_, const int* doc_start,
                                                              __nv_bfloat16* __restrict__ y, int H, int cap, float scale2, int window_tiles, int least, int by_length,
                                                              float* __restrict__ flat, int B) {
  constexpr int TT = 4096 / D, PER = TT / 8, VW = TT / 16;                // tokens of a turn, of a lane; words of a lane's piece of V
  constexpr int KL = D / 64, NT = D / 16, LPT = D / 8, TPI = 32 / LPT, RP = 4, PASS = KB / (AW * TPI * RP);
  __shared__ union {
    AttnShared<D, AW> at;
    QuantShared quant;
  } sm_;
  AttnShared<D, AW>& sm = sm_.at;
  pdl_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int S, rank, h, b, ctas = 0;
  if (FLAT) {
    pdl_wait();
    S = 1;
    rank = (int)blockIdx.x;
    flat_place(flat_ctas<TT, AW>(B, H, (int)gridDim.x, pos_, doc_start, min(cap, rope_rows), window_tiles), H, B, rank, b, ctas);
    if (b == B) return;
    h = rank / ctas;
    rank -= h * ctas;
  } else {
    S = (int)cluster_size();
    rank = (int)cluster_rank();
    h = blockIdx.x / S;
    b = by_length ? longest_first((int)gridDim.y, (int)blockIdx.y, pos_, doc_start) : (int)blockIdx.y;
  }
  const int g = lane >> 2, c4 = lane & 3;
  // the first kernel of a decode step may be storing a new document start: looked at again behind the wait
  int lo = doc_start ? ld_relaxed(doc_start + b) : 0;
  const int pos = pos_[b];
  __nv_bfloat16* out = y + ((long long)b * H + h) * D;
  if (pos < 0 || pos >= min(cap, rope_rows)) {
    pdl_wait();
    if (rank == 0)
      for (int i = tid; i < D / 2; i += 32 * AW) reinterpret_cast<uint32_t*>(out)[i] = 0u;
    return;
  }
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // waited for before the first store to another CTA
  const long long bh = (long long)b * H + h, nb = cap / KB;
  const int slot = pos % KB, last = pos / KB;
  const int band = window_tiles > 0 ? max((pos / 128 - (window_tiles - 1)) * 128, 0) : 0;
  lo = max(lo, band);
  const int8_t *kp = c.k + bh * cap * D + PER * g * D + 16 * c4, *vp = c.v + bh * cap * D + g * KB + 4 * VW * c4;
  uint32_t kr[VW][2][KL][4], vr[NT][2][VW];
  auto load_k = [&](int u) {
    const int8_t* p = kp + (long long)u * (TT * D);
#pragma unroll
    for (int i = 0; i < VW; ++i)
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int l = 0; l < KL; ++l) ld_stream(kr[i][f][l], p + (2 * i + f) * D + 64 * l);
  };
  auto load_v = [&](int u) {
    const int8_t* p = vp + (long long)(u * TT / KB) * (KB * D) + u * TT % KB;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int f = 0; f < 2; ++f) ld_stream(vr[t][f], p + (16 * t + 8 * f) * KB);
  };
  // the open block over the lanes in 16-byte pieces: a warp's pass is RP * TPI of its tokens
  const int sub = lane / LPT, piece = lane % LPT * 8;
  uint4 tk[RP], tv[RP];
  auto tail_slot = [&](int pass, int r) { return ((pass * RP + r) * AW + warp) * TPI + sub; };
  auto load_tail = [&](int pass) {
    const __nv_bfloat16 *kt = c.kt + bh * KB * D + piece, *vt = c.vt + bh * KB * D + piece;
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const int t = tail_slot(pass, r);
      tk[r] = tv[r] = make_uint4(0u, 0u, 0u, 0u);
      if (t < slot) {
        tk[r] = *reinterpret_cast<const uint4*>(kt + t * D);
        tv[r] = *reinterpret_cast<const uint4*>(vt + t * D);
      }
    }
  };
  // Of the cluster as many CTAs take part as get `least` turns each, and one for the open block; the others leave.  The last one has the open
  // block (and, where there is no further CTA, its share of the full ones).
  const int end = last * (KB / TT);
  auto taking_part = [&](int from) { return FLAT ? ctas : min(S, max(0, (end - from / TT + least - 1) / least) + 1); };
  int active = taking_part(lo), u = lo / TT + rank * AW + warp;
  if (rank >= active) return;
  bool tail_cta = rank == active - 1;
  if (u < end) load_k(u);
  if (tail_cta) load_tail(0);
  if (!FLAT) pdl_wait();
  if (!FLAT && doc_start) {
    const int now = max(ld_relaxed(doc_start + b), lo);             // a document that begins with this token; none begins earlier than was seen
    if (now != lo) {
      lo = now;
      active = taking_part(lo);
      if (rank >= active) return;
      u = lo / TT + rank * AW + warp;
      if (u < end) load_k(u);
      if (!tail_cta && rank == active - 1) load_tail(0);
      tail_cta = rank == active - 1;
    }
  }
  const int step = active * AW;
  for (int role = warp; role < (tail_cta ? 3 : 1); role += AW) {      // query, new key, new value
    const __nv_bfloat16* x = qkv + b * ldq + ((long long)role * H + h) * D;
    const float *cs = cosT + (long long)pos * (D / 2), *sn = sinT + (long long)pos * (D / 2);
    if (role == 0) {
      float a[D / 64], e[D / 64];
      const float r = turn_and_norm<D, float>(x, cs, sn, a, e);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        sm.q[lane + 32 * i] = a[i] * r;
        sm.q[lane + 32 * i + D / 2] = e[i] * r;
      }
    } else {
      __nv_bfloat16 *tail = (role == 1 ? c.kt : c.vt) + (bh * KB + slot) * D, v0[D / 64], v1[D / 64];
      if (role == 1) {                          // in 64 bits: the key's rounding to bf16 is the only one, and it stays
        double a[D / 64], e[D / 64];
        const double r = turn_and_norm<D, double>(x, cs, sn, a, e);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          v0[i] = __double2bfloat16(a[i] * r);
          v1[i] = __double2bfloat16(e[i] * r);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          v0[i] = x[lane + 32 * i];
          v1[i] = x[lane + 32 * i + D / 2];
        }
      }
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int d = lane + 32 * i;
        sm.fresh[role - 1][d] = v0[i];
        sm.fresh[role - 1][d + D / 2] = v1[i];
        tail[d] = v0[i];
        tail[d + D / 2] = v1[i];
      }
    }
  }
  if (u < end) load_v(u);
  __syncthreads();

  // The open block, in plain fp32.
  if (tail_cta) {
    const int from = lo - last * KB;                                // slots from .. slot are seen
    float q[8], m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { q[i] = sm.q[piece + i]; acc[i] = 0.f; }
#pragma unroll 1
    for (int pass = 0; pass < PASS && pass * RP * AW * TPI <= slot; ++pass) {
      if (pass) load_tail(pass);
      float s[RP], mn = m;
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const int t = tail_slot(pass, r);
        if (t == slot) {
          tk[r] = *reinterpret_cast<const uint4*>(&sm.fresh[0][piece]);
          tv[r] = *reinterpret_cast<const uint4*>(&sm.fresh[1][piece]);
        }
        float f[8], s0 = 0.f, s1 = 0.f;
        unpack8(tk[r], f);
#pragma unroll
        for (int i = 0; i < 8; i += 2) { s0 += q[i] * f[i]; s1 += q[i + 1] * f[i + 1]; }
        s[r] = s0 + s1;
      }
#pragma unroll
      for (int r = 0; r < RP; ++r) {
#pragma unroll
        for (int o = LPT / 2; o > 0; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
        s[r] *= scale2;
        const int t = tail_slot(pass, r);
        if (t >= from && t <= slot) mn = fmaxf(mn, s[r]);
      }
#pragma unroll
      for (int o = LPT; o < 32; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      const float base = mn == -INFINITY ? 0.f : mn, corr = exp2_fast(m - base);
      m = mn;
      l *= corr;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= corr;
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const int t = tail_slot(pass, r);
        if (t >= from && t <= slot) {
          const float p = exp2_fast(s[r] - base);
          float f[8];
          unpack8(tv[r], f);
          l += p;
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += p * f[i];
        }
      }
    }
#pragma unroll
    for (int o = LPT; o < 32; o <<= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    }
    if (sub == 0) {
      float4* to = reinterpret_cast<float4*>(&sm.acc[AW + warp][piece]);
      to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
    if (lane == 0) { sm.m[AW + warp] = m; sm.l[AW + warp] = l; }
  }

  // The full blocks.  Token PER g + 2 i + f of a turn is row g + 8 f of MMA i, so a lane ends up with the scores of the PER tokens from
  // PER g on.
  {
    float m = -INFINITY, l = 0.f, acc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = 0.f;
    if (u < end) {
      uint32_t qf[4 * KL][2];
#pragma unroll
      for (int l2 = 0; l2 < KL; ++l2)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 f = *reinterpret_cast<const float4*>(&sm.q[64 * l2 + 16 * c4 + 4 * w]);
          uint32_t u0 = pack_f16(f.x, f.y), u1 = pack_f16(f.z, f.w);
          if (g & 1) {
            const float2 h0 = __half22float2(*reinterpret_cast<__half2*>(&u0)), h1 = __half22float2(*reinterpret_cast<__half2*>(&u1));
            u0 = pack_f16(f.x - h0.x, f.y - h0.y);
            u1 = pack_f16(f.z - h1.x, f.w - h1.y);
          }
          qf[4 * l2 + w][0] = u0;
          qf[4 * l2 + w][1] = u1;
        }
      const float *ksp = c.ks + bh * nb, *vsp = c.vs + bh * nb;
      float ks_n = ksp[u * TT / KB], vs_n = vsp[u * TT / KB];
#pragma unroll 1
      while (true) {
        const int next = u + step, j = u * TT + PER * g;
        const float ks = ks_n, vs = vs_n;
        if (next < end) { ks_n = ksp[next * TT / KB]; vs_n = vsp[next * TT / KB]; }
        float s[PER];
        {
          float d[VW][KL][4];                   // chains of four MMAs
#pragma unroll
          for (int i = 0; i < VW; ++i)
#pragma unroll
            for (int l2 = 0; l2 < KL; ++l2) d[i][l2][0] = d[i][l2][1] = d[i][l2][2] = d[i][l2][3] = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int l2 = 0; l2 < KL; ++l2)
#pragma unroll
              for (int i = 0; i < VW; ++i) {
                uint32_t a0, a1, a2, a3;
                codes_f16(kr[i][0][l2][w], a0, a2);
                codes_f16(kr[i][1][l2][w], a1, a3);
                mma_f16(d[i][l2], a0, a1, a2, a3, qf[4 * l2 + w][0], qf[4 * l2 + w][1]);
              }
#pragma unroll
          for (int i = 0; i < VW; ++i) {
            s[2 * i] = d[i][0][0] + d[i][0][1];
            s[2 * i + 1] = d[i][0][2] + d[i][0][3];
            if (KL == 2) {
              s[2 * i] += d[i][KL - 1][0] + d[i][KL - 1][1];
              s[2 * i + 1] += d[i][KL - 1][2] + d[i][KL - 1][3];
            }
          }
        }
        if (signbit(ks)) {                      // a key with a value that is not finite
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            uint32_t bad = 0;
#pragma unroll
            for (int l2 = 0; l2 < KL; ++l2)
#pragma unroll
              for (int w = 0; w < 4; ++w) bad |= bad_codes(kr[i >> 1][i & 1][l2][w]);
            bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
            bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
            if (bad) s[i] = __int_as_float(0x7fc00000);
          }
        }
        if (next < end) load_k(next);
        const float f = fabsf(ks) * scale2;
        float mn = m;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          s[i] = j + i >= lo ? s[i] * f : -INFINITY;
          mn = fmaxf(mn, s[i]);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        const float top = mn == -INFINITY ? 0.f : mn, corr = exp2_fast(m - top), base = top - kLift;
        m = mn;
        l *= corr;
        uint32_t pr[VW], pf[VW][2];
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const float p0 = exp2_fast(s[2 * i] - base), p1 = exp2_fast(s[2 * i + 1] - base);
          l += p0 + p1;
          pr[i] = pack_f16(p0, p1);
        }
        // B's rows of MMA w are tokens 4 VW c + 4 w ..: with the lanes of g = 2 c, and 2 c + 1 from the middle on
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < VW; ++i) pf[(k * VW + i) >> 1][(k * VW + i) & 1] = __shfl_sync(0xffffffffu, pr[i], 4 * (2 * c4 + k));
        const float fv = fabsf(vs) * kDrop;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t a0, a1, a2, a3;
            codes_f16(vr[t][0][w], a0, a2);
            codes_f16(vr[t][1][w], a1, a3);
            mma_f16(d, a0, a1, a2, a3, pf[w][0], pf[w][1]);
          }
          acc[t][0] = acc[t][0] * corr + fv * d[0];
          acc[t][1] = acc[t][1] * corr + fv * d[2];
        }
        if (signbit(vs)) {                      // values that are not finite, of tokens that are seen
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              bool bad = false;
#pragma unroll
              for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int i = 0; i < 4; ++i) bad |= ((bad_codes(vr[t][e][w]) >> (8 * i)) & 0x80u) && u * TT + 4 * (VW * c4 + w) + i >= lo;
              bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1) != 0;
              bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 2) != 0;
              if (bad) acc[t][e] = __int_as_float(0x7fc00000);
            }
        }
        u = next;
        if (u >= end) break;
        load_v(u);
      }
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    l *= kDrop;
    if (c4 == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        sm.acc[warp][16 * t + g] = acc[t][0];
        sm.acc[warp][16 * t + 8 + g] = acc[t][1];
      }
    }
    if (lane == 0) { sm.m[warp] = m; sm.l[warp] = l; }
  }
  __syncthreads();

  // The CTA's own parts, then the cluster's.  A part without a token has -inf and 0.
  constexpr int OUT = (D + 32 * AW - 1) / (32 * AW);                      // dimensions of a thread
  const int parts = tail_cta ? 2 * AW : AW;
  float M = -INFINITY, L = 0.f, o[OUT] = {};
  auto sum_up = [&](int n, auto maximum, auto sum, auto values) {
    M = -INFINITY;
    for (int e = 0; e < n; ++e) M = fmaxf(M, maximum(e));
    const float base = M == -INFINITY ? 0.f : M;
    L = 0.f;
#pragma unroll
    for (int i = 0; i < OUT; ++i) o[i] = 0.f;
    for (int e = 0; e < n; ++e) {
      const float w = exp2_fast(maximum(e) - base);
      L += w * sum(e);
#pragma unroll
      for (int i = 0; i < OUT; ++i)
        if (tid + 32 * AW * i < D) o[i] += w * values(e)[tid + 32 * AW * i];
    }
  };
  sum_up(parts, [&](int e) { return sm.m[e]; }, [&](int e) { return sm.l[e]; }, [&](int e) { return sm.acc[e]; });
  if (FLAT) {
    float* to = flat + (long long)blockIdx.x * (D + 4);
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      const int d = tid + 32 * AW * i;
      if (d < D) to[d] = o[i];
    }
    if (tid == 0) *reinterpret_cast<float2*>(to + D) = make_float2(L, M);
  } else if (active > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t to = map_to_rank(smem_u32(&sm.part[rank][0]), 0);
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      const int d = tid + 32 * AW * i;
      if (d < D) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4u * (uint32_t)d), "f"(o[i]) : "memory");
    }
    if (tid == 0) {
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4u * D), "f"(L) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4u * D + 4u), "f"(M) : "memory");
    }
    cluster_barrier();
    if (rank == 0) sum_up(active, [&](int r) { return sm.part[r][D + 1]; }, [&](int r) { return sm.part[r][D]; }, [&](int r) { return sm.part[r]; });
  }
  if (!FLAT && rank == 0) {
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      const int d = tid + 32 * AW * i;
      if (d < D) out[d] = __float2bfloat16(L != 0.f ? o[i] / L : 0.f);
    }
  }
  if (tail_cta && slot == KB - 1) {
    // the block is full: its last token is in memory since the first barrier of the CTA
    __syncthreads();
    auto tail_of = [&](const __nv_bfloat16* t0) { return [=](int t, int d) { return t0 + t * D + d; }; };
    kv8_quantise_block<32 * AW, D, false>(tail_of(c.kt + bh * KB * D), c.k + (bh * cap + (long long)last * KB) * D, c.ks + bh * nb + last, sm_.quant);
    kv8_quantise_block<32 * AW, D, true>(tail_of(c.vt + bh * KB * D), c.v + (bh * cap + (long long)last * KB) * D, c.vs + bh * nb + last, sm_.quant);
  }
}

// What the CTAs of a head and sequence have, together: eight groups of threads, each some of the CTAs.  It is launched before they end, so that
// its CTAs come to the SMs as those leave; its 8 D threads find no room beside three of them.
template <int D, int AW>
__global__ void __launch_bounds__(8 * D) kv8_join_kernel(const float* parts, PerSeq pos_, const int* doc_start, __nv_bfloat16* __restrict__ y, int B, int H,
                                                        int places, int limit, int window_tiles) {
  __shared__ float acc[8][D], ml[8][2];
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x % D, group = threadIdx.x / D, lane = threadIdx.x & 31;
  pdl_launch();
  pdl_wait();
  const int mine = flat_ctas<4096 / D, AW>(B, H, places, pos_, doc_start, limit, window_tiles), n = __shfl_sync(0xffffffffu, mine, b);
  int before = lane < b ? mine * H : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const float* p = parts + (long long)(before + h * n) * (D + 4);
  float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll 8
  for (int e = group; e < n; e += 8) {
    const float2 lm = __ldcg(reinterpret_cast<const float2*>(p + e * (D + 4) + D));
    const float v = __ldcg(p + e * (D + 4) + d), top = fmaxf(M, lm.y), base = top == -INFINITY ? 0.f : top;
    const float f = exp2_fast(M - base), w = exp2_fast(lm.y - base);
    L = L * f + w * lm.x;
    o = o * f + w * v;
    M = top;
  }
  acc[group][d] = o;
  if (d == 0) { ml[group][0] = L; ml[group][1] = M; }
  __syncthreads();
  if (group) return;
  M = ml[0][1];
#pragma unroll
  for (int e = 1; e < 8; ++e) M = fmaxf(M, ml[e][1]);
  const float base = M == -INFINITY ? 0.f : M;
  L = o = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float w = exp2_fast(ml[e][1] - base);
    L += w * ml[e][0];
    o += w * acc[e][d];
  }
  y[((long long)b * H + h) * D + d] = __float2bfloat16(L != 0.f ? o / L : 0.f);
}

// CTAs of a cluster: doubled until there are one and a half for each SM, as long as the cache's length (the band's, if there is one) can give
// every warp a turn; where sequences have positions of their own until there are three, as long as each gets 2048 tokens.  us by 1 / 2 / 4 / 8 / 16 CTAs, heads of 128: 10 heads, 300 tokens
// 5.8 / 6.1 / 5.0 / 5.0 / 5.4, 2040 tokens 21 / 14 / 9.8 / 7.8 / 6.9; 40 heads, 2040 tokens 22 / 15 / 12 / 10 / 14, 131000 tokens 1113 / 571 / 354 / 240 / 245;
// 160 heads, 2040 tokens 27 / 20 / 25 / 33 / 52; 320 heads, 16000 tokens 234 / 247 / 245 / 244 / 274; 640 heads, 64 tokens 11 / 16 / 22 / 30 / 62, 2040 tokens
// 67 / 63 / 81 / 111 / 196.  192 heads, 32700 tokens 357 / 282 / 267 / 276.  16 sequences of 10 heads, random lengths up to 2048 22 / 15.6 / 17.5,
// up to 8192 74 / 46 / 34 (all of 8192: 92 / 62 / 68); 40 sequences up to 8192 87 / 58 / 69 (140 / 147 / 148); 4 sequences up to 8192 by 8 / 16 15.6 / 20.9.
inline int kv8_splits(int B, int H, int D, int AW, int cap, int window_tiles, bool own, int sms) {
  const long long tokens = window_tiles > 0 && window_tiles < cap / 128 ? window_tiles * 128ll : cap;
  const long long heads = (long long)B * H;
  int s = 1;
  while (s < kMaxSplit && heads * s < 3ll * sms / 2 && tokens >= (long long)s * AW * (4096 / D)) s *= 2;
  while (own && s < kMaxSplit && heads * s < 3ll * sms && tokens >= s * 4096ll) s *= 2;
  return s;
}

struct AttnArgs {
  const __nv_bfloat16* qkv;
  long long ldq;
  const float *cosT, *sinT;
  int rope_rows;
  Kv8 c;
  PerSeq pos;
  const int* doc_start;
  __nv_bfloat16* y;
  int H, cap;
  float scale2;
  int window_tiles, by_length;
  float* parts;
};
template <int D, int AW>
int launch_kv8_attn(const AttnArgs& p, int B, int split, int pdl, cudaStream_t s) {
  static OncePerDevice once;
  BONES_ONCE(once, {
    BONES_CHECK(cudaFuncSetAttribute(kv8_attn_kernel<D, AW, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  });
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)(p.H * split), (unsigned)B);
  cfg.blockDim = dim3(32 * AW);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, split, pdl);
  return (int)cudaLaunchKernelEx(&cfg, kv8_attn_kernel<D, AW, false>, p.qkv, p.ldq, p.cosT, p.sinT, p.rope_rows, p.c, p.pos, p.doc_start, p.y, p.H, p.cap, p.scale2,
                                 p.window_tiles, AW, p.by_length, (float*)nullptr, B);
}
template <int D>
int launch_kv8_flat(const AttnArgs& p, int B, int places, int pdl, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)places);
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, pdl);
  BONES_CHECK(cudaLaunchKernelEx(&cfg, kv8_attn_kernel<D, 4, true>, p.qkv, p.ldq, p.cosT, p.sinT, p.rope_rows, p.c, p.pos, p.doc_start, p.y, p.H, p.cap, p.scale2,
                                 p.window_tiles, 4, 0, p.parts, B));
  cfg.gridDim = dim3((unsigned)p.H, (unsigned)B);
  cfg.blockDim = dim3(8 * D);
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  return (int)cudaLaunchKernelEx(&cfg, kv8_join_kernel<D, 4>, (const float*)p.parts, p.pos, p.doc_start, p.y, B, p.H, places, min(p.cap, p.rope_rows), p.window_tiles);
}

inline bool kv8_refused(const Kv8& c, int B, int H, int D, int cap) {
  return B < 1 || H < 1 || B > 65535 || H > 65535 || (D != 64 && D != 128) || cap < KB || (cap % KB) || misaligned16(c.k, c.v, c.ks, c.vs, c.kt, c.vt) ||
         !c.k || !c.v || !c.ks || !c.vs || !c.kt || !c.vt;
}

}  // namespace bones

extern "C" {
using namespace bones;

// k, v: bf16, distances of sequences, tokens and heads in values (multiples of 8 where there are two or more); pos, len: an address and the distance between two
// sequences' values, or a value for all.  A sequence at a negative position, without tokens or with more than fit is left as it was.
int bones_kv8_append(void* k8, void* v8, float* ks, float* vs, void* kt, void* vt, const void* k, const void* v, long long kb, long long kst, long long kh,
                     long long vb, long long vst, long long vh, int B, int H, int D, int cap, int t, const int* pos, int pos_step, int pos0, const int* len,
                     int len_step, int len0, void* stream) {
  const Kv8 c{(int8_t*)k8, (int8_t*)v8, ks, vs, (__nv_bfloat16*)kt, (__nv_bfloat16*)vt};
  if (kv8_refused(c, B, H, D, cap) || t < 0 || !k || !v || misaligned16(k, v) ||
      (((t > 1 ? kst | vst : 0) | (B > 1 ? kb | vb : 0) | (H > 1 ? kh | vh : 0)) % 8))
    return -2;
  if (t == 0) return 0;
  // t tokens touch this many blocks at most; none lies past the capacity
  const long long blocks = min(((long long)t + KB - 2) / KB + 1, (long long)cap / KB);
  const dim3 grid((unsigned)(2 * blocks), (unsigned)H, (unsigned)B);
  (D == 128 ? kv8_append_kernel<128> : kv8_append_kernel<64>)<<<grid, kAppendThreads, 0, (cudaStream_t)stream>>>(
      c, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, kb, kst, kh, vb, vst, vh, PerSeq{pos, pos_step, pos0}, PerSeq{len, len_step, len0}, t, H, cap);
  return (int)cudaGetLastError();
}

// k, v: bf16 [B, length, H, D]
int bones_kv8_read(void* k8, void* v8, float* ks, float* vs, void* kt, void* vt, void* k, void* v, int B, int H, int D, int cap, int length, const int* held,
                   int held_step, int held0, void* stream) {
  const Kv8 c{(int8_t*)k8, (int8_t*)v8, ks, vs, (__nv_bfloat16*)kt, (__nv_bfloat16*)vt};
  if (kv8_refused(c, B, H, D, cap) || length < 0 || !k || !v || misaligned16(k, v)) return -2;
  if (length == 0) return 0;
  const dim3 grid((unsigned)(2 * (((long long)length + KB - 1) / KB)), (unsigned)H, (unsigned)B);
  (D == 128 ? kv8_read_kernel<128> : kv8_read_kernel<64>)<<<grid, 256, 0, (cudaStream_t)stream>>>(c, (__nv_bfloat16*)k, (__nv_bfloat16*)v,
                                                                                                 PerSeq{held, held_step, held0}, length, H, cap);
  return (int)cudaGetLastError();
}

// qkv: bf16 rows of 3 * H * D, ldq apart; cosT, sinT: fp32 [rope_rows, D / 2]; y: bf16 [B, H * D]; window_tiles: of 128 tokens, 0 for all;
// parts: room for part_places * (D + 4) floats on 16 bytes, of this call alone until it ends, or null; no more CTAs than it has places share a
// long cache (where no more than 16383 tokens are seen none is used).
int bones_kv8_attention(const void* qkv, long long ldq, const float* cosT, const float* sinT, int rope_rows, void* k8, void* v8, float* ks, float* vs, void* kt,
                        void* vt, const int* pos, int pos_step, int pos0, const int* doc_start, void* y, int B, int H, int D, int cap, float scale,
                        int window_tiles, int pdl, float* parts, int part_places, void* stream) {
  const Kv8 c{(int8_t*)k8, (int8_t*)v8, ks, vs, (__nv_bfloat16*)kt, (__nv_bfloat16*)vt};
  if (kv8_refused(c, B, H, D, cap) || !qkv || !cosT || !sinT || !y || misaligned16(qkv, y, parts) || (B > 1 && ldq % 8) || window_tiles < 0 || part_places < 0) return -2;
  const AttnArgs p{(const __nv_bfloat16*)qkv, ldq, cosT, sinT, rope_rows, c, PerSeq{pos, pos_step, pos0}, doc_start, (__nv_bfloat16*)y, H, cap,
                   scale * 1.4426950408889634f, window_tiles, B > 1 && B <= 64 && pos && pos_step && !pdl, parts};
  int dev = 0, sms = 0;
  BONES_CHECK(cudaGetDevice(&dev));
  BONES_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  // Two warps a CTA where sequences of one length make more CTAs of four than the SMs hold (three each) and the cache is short: twice as many,
  // smaller ones fit at once, but the longest take twice the time.  640 heads, us by four / two: alone, 64 tokens 11.8 / 8.2, lengths from 1 to
  // 2048 37 / 53; a step of 20 layers at 64 tokens 715 / 645, at 500 948 / 944, at 1900 1730 / 1866.
  const int aw = (long long)B * H > 3ll * sms && !(pos && pos_step) && cap <= 1024 ? 2 : 4;
  const int split = kv8_splits(B, H, D, aw, cap, window_tiles, B > 1 && pos && pos_step, sms);
  cudaStream_t s = (cudaStream_t)stream;
  // Equal shares for long caches where they pay for the second kernel (3 us of latencies): a cluster leaves SMs idle where heads are few, or where
  // lengths differ.  With many heads a share is most of one's turns, and the parts come out unequal: 4 sequences of 7000 to 28000 tokens, 32 heads,
  // 104 / 114, 6 of 5000 to 30000 150 / 165.  One position for all is known here where it comes as a number.
  const int places = parts ? min((D == 128 ? 3 : 4) * sms, part_places) : 0;
  const long long seen = pos ? cap : min((long long)cap, pos0 + 1ll), tokens = window_tiles > 0 ? min(seen, window_tiles * 128ll) : seen;
  if (B <= 32 && 8ll * B * H <= 3ll * places && tokens >= (B > 1 ? kFlatFrom : 2 * kFlatFrom))
    return D == 128 ? launch_kv8_flat<128>(p, B, places, pdl, s) : launch_kv8_flat<64>(p, B, places, pdl, s);
  if (aw == 2) return D == 128 ? launch_kv8_attn<128, 2>(p, B, split, pdl, s) : launch_kv8_attn<64, 2>(p, B, split, pdl, s);
  return D == 128 ? launch_kv8_attn<128, 4>(p, B, split, pdl, s) : launch_kv8_attn<64, 4>(p, B, split, pdl, s);
}
}  // extern "C"
