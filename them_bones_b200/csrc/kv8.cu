// A key/value cache in 8 bits: append, read-back and single-token attention.  Layout (one layer): blocks of 64 tokens; key codes
// [B, H, T, D] and value codes [B, H, T / 64, D, 64] (int8), scales [B, H, T / 64] (fp32), the open block's tokens [B, H, 64, D] (bf16).
//
//   code = rint(x * (127 / most)),  scale = most / 127,  most = the block's largest finite |x|
//
// A value that is not finite gets the code -128, which stands for NaN, and its block a scale with a minus sign, so that blocks
// without one need not look for it.  A block is quantised once, from its 64 bf16 tokens, when it is full.
#include "common.cuh"

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
__device__ __forceinline__ int kv8_code(float x, float inv) {
  if (!(fabsf(x) <= 3.402823466e38f)) return -128;
  return max(-127, min(127, __float2int_rn(x * inv)));
}
__device__ __forceinline__ float kv8_value(int code, float scale) { return code == -128 ? __int_as_float(0x7fc00000) : (float)code * fabsf(scale); }

__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = unpack_bf16(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

constexpr int QT = 256;                         // threads that quantise a block
struct __align__(16) QuantShared {
  float most[QT / 32];
  int bad[QT / 32];
  int8_t turn[128][KB + 16];                    // value codes on their way to [D][64]; rows stay 16-byte aligned
};

// A whole block by a CTA of QT threads: 16-byte piece i of the block is token i / (D / 8), dimensions 8 (i % (D / 8)) ..; `piece(token, dim)`
// is its address.  Key codes go out as they lie, value codes through shared memory to be transposed.
template <int D, bool VALUES, class Piece>
__device__ __forceinline__ void kv8_quantise_block(Piece piece, int8_t* __restrict__ out, float* __restrict__ scale, QuantShared& sm) {
  constexpr int PER = KB * D / 8 / QT, ROW = D / 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint4 u[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = tid + i * QT;
    u[i] = *reinterpret_cast<const uint4*>(piece(p / ROW, p % ROW * 8));
  }
  float most = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    float f[8];
    unpack8(u[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(f[j]);
      if (a <= 3.402823466e38f) most = fmaxf(most, a);
      else bad = true;
    }
  }
  most = warp_max(most);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) { sm.most[warp] = most; sm.bad[warp] = bad; }
  __syncthreads();
  bad = false;
#pragma unroll
  for (int w = 0; w < QT / 32; ++w) { most = fmaxf(most, sm.most[w]); bad |= sm.bad[w] != 0; }
  const float inv = kv8_inverse(most);
  if (tid == 0) *scale = kv8_scale(most, bad);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = tid + i * QT, t = p / ROW, d = p % ROW * 8;
    float f[8];
    unpack8(u[i], f);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = kv8_code(f[j], inv);
      if (VALUES) sm.turn[d + j][t] = (int8_t)c;
      else w[j >> 2] |= (uint32_t)(c & 255) << (8 * (j & 3));
    }
    if (!VALUES) *reinterpret_cast<uint2*>(out + t * D + d) = make_uint2(w[0], w[1]);
  }
  __syncthreads();
  if (VALUES) {
    for (int i = tid; i < D * (KB / 16); i += QT)
      *reinterpret_cast<uint4*>(out + i * 16) = *reinterpret_cast<const uint4*>(&sm.turn[i / (KB / 16)][i % (KB / 16) * 16]);
    __syncthreads();
  }
}

// Tokens pos .. pos + len of a sequence.  A CTA takes one block that the run touches, of the keys or of the values of one head; the first
// one also stores what is left over for the open block, after it has read the tokens that were in it before.
template <int D, bool VALUES>
__device__ __forceinline__ void kv8_append_block(const __nv_bfloat16* __restrict__ src, long long st, int8_t* __restrict__ codes, float* __restrict__ scales,
                                                 __nv_bfloat16* __restrict__ tail, int pos, int len, int i, QuantShared& sm) {
  const int first = pos / KB, end = pos + len, blk = first + i;
  if ((long long)(blk + 1) * KB <= end)
    kv8_quantise_block<D, VALUES>(
        [&](int t, int d) -> const __nv_bfloat16* {
          const int j = blk * KB + t;
          return j < pos ? tail + t * D + d : src + (long long)(j - pos) * st + d;
        },
        codes + (long long)blk * KB * D, scales + blk, sm);
  if (i == 0) {
    const int open = end / KB * KB, from = max(pos, open);
    for (int p = threadIdx.x; p < (end - from) * (D / 8); p += QT) {
      const int j = from + p / (D / 8), d = p % (D / 8) * 8;
      *reinterpret_cast<uint4*>(tail + (j - open) * D + d) = *reinterpret_cast<const uint4*>(src + (long long)(j - pos) * st + d);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(QT) kv8_append_kernel(Kv8 c, const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, long long kb,
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

// One block of one head back to bf16 rows [B, length, H, D]; zeros behind the tokens held.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v, PerSeq held_, int length, int H, int cap) {
  __shared__ __align__(16) int8_t turn[128][KB + 16];
  const int b = blockIdx.z, h = blockIdx.y, blk = blockIdx.x >> 1;
  const bool values = blockIdx.x & 1;
  const int held = max(held_[b], 0), j0 = blk * KB;
  const long long bh = (long long)b * H + h;
  __nv_bfloat16* out = (values ? v : k) + ((long long)b * length * H + h) * D;
  const bool open = blk == held / KB, some = j0 < held && j0 < cap;
  const int8_t* codes = (values ? c.v : c.k) + (bh * cap + j0) * D;
  const float scale = some && !open ? (values ? c.vs : c.ks)[bh * (cap / KB) + blk] : 0.f;
  const __nv_bfloat16* tail = (values ? c.vt : c.kt) + bh * KB * D;
  if (values && some && !open) {
    for (int i = threadIdx.x; i < D * 4; i += 256) *reinterpret_cast<uint4*>(&turn[i / 4][i % 4 * 16]) = *reinterpret_cast<const uint4*>(codes + i * 16);
  }
  __syncthreads();
  for (int p = threadIdx.x; p < KB * D / 8; p += 256) {
    const int t = p / (D / 8), d = p % (D / 8) * 8, j = j0 + t;
    if (j >= length) continue;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (some && j < held) {
      if (open) {
        o = *reinterpret_cast<const uint4*>(tail + t * D + d);
      } else {
        float f[8];
        if (values) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = kv8_value(turn[d + e][t], scale);
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(codes + t * D + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = kv8_value((int)(int8_t)((e < 4 ? u.x : u.y) >> (8 * (e & 3))), scale);
        }
        o = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
      }
    }
    *reinterpret_cast<uint4*>(out + (long long)j * H * D + d) = o;
  }
}

// One CTA per (head, sequence): a block at a time, four threads a key for the scores, two threads a dimension for the output, a running
// maximum.
template <int D>
__global__ void __launch_bounds__(256) kv8_attn_kernel(const __nv_bfloat16* __restrict__ qkv, long long ldq, const float* __restrict__ cosT,
                                                       const float* __restrict__ sinT, int rope_rows, Kv8 c, PerSeq pos_, const int* __restrict__ doc_start,
                                                       __nv_bfloat16* __restrict__ y, int H, int cap, float scale, int window_tiles) {
  __shared__ QuantShared sm;
  __shared__ __align__(16) float s_q[D];
  __shared__ __align__(16) __nv_bfloat16 s_new[2][D];
  __shared__ float s_p[KB], s_red[8], s_out[2][D];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pos = pos_[b];
  __nv_bfloat16* out = y + ((long long)b * H + h) * D;
  if (pos < 0 || pos >= min(cap, rope_rows)) {
    if (tid < D) out[tid] = __float2bfloat16(0.f);
    return;
  }
  const long long bh = (long long)b * H + h, nb = cap / KB;
  const int slot = pos % KB, blk_new = pos / KB;
  if (warp < 3) {
    constexpr int HALF = D / 2, N = HALF / 32;
    const __nv_bfloat16* x = qkv + b * ldq + ((long long)warp * H + h) * D;
    float a[N], e[N], ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 32 * i;
      a[i] = __bfloat162float(x[d]);
      e[i] = __bfloat162float(x[d + HALF]);
      if (warp < 2) {
        const float cs = cosT[(long long)pos * HALF + d], sn = sinT[(long long)pos * HALF + d], a0 = a[i], e0 = e[i];
        a[i] = a0 * cs + e0 * sn;
        e[i] = e0 * cs - a0 * sn;
        ss += a[i] * a[i] + e[i] * e[i];
      }
    }
    const float r = warp < 2 ? rsqrtf(warp_sum(ss) / D + 1.1920928955078125e-07f) : 1.f;
    __nv_bfloat16* tail = (warp == 1 ? c.kt : c.vt) + (bh * KB + slot) * D;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 32 * i;
      if (warp == 0) {
        s_q[d] = a[i] * r;
        s_q[d + HALF] = e[i] * r;
      } else {
        const __nv_bfloat16 u = __float2bfloat16(a[i] * r), w = __float2bfloat16(e[i] * r);
        s_new[warp - 1][d] = u;
        s_new[warp - 1][d + HALF] = w;
        tail[d] = u;
        tail[d + HALF] = w;
      }
    }
  }
  __syncthreads();
  int lo = doc_start ? doc_start[b] : 0;
  if (window_tiles > 0) lo = max(lo, (pos / 128 - (window_tiles - 1)) * 128);
  lo = max(lo, 0);
  float m = -INFINITY, l = 0.f, acc = 0.f;
  const int od = tid % D, oh = tid / D;                  // thread's dimension and half of the block's tokens (D = 64: a quarter)
  constexpr int PARTS = 256 / D, PT = KB / PARTS;
  for (int blk = lo / KB; blk <= blk_new; ++blk) {
    const bool open = blk == blk_new;
    const int t = tid >> 2, j = blk * KB + t, d0 = (tid & 3) * (D / 4);
    float s = 0.f;
    const bool seen = j >= lo && j <= pos;
    if (seen) {
      if (open) {
        const __nv_bfloat16* kr = t == slot ? s_new[0] : c.kt + (bh * KB + t) * D;
#pragma unroll 8
        for (int i = 0; i < D / 4; ++i) s += s_q[d0 + i] * __bfloat162float(kr[d0 + i]);
      } else {
        const float sc = c.ks[bh * nb + blk];
        const int8_t* kr = c.k + (bh * cap + j) * D;
#pragma unroll 8
        for (int i = 0; i < D / 4; ++i) s += s_q[d0 + i] * kv8_value(kr[d0 + i], sc);
      }
    }
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    s = seen ? s * scale : -INFINITY;
    const float wm = warp_max(s);
    if (lane == 0) s_red[warp] = wm;
    __syncthreads();
    float mn = m;
#pragma unroll
    for (int w = 0; w < 8; ++w) mn = fmaxf(mn, s_red[w]);
    // a score that is not a number has no part in the maximum but makes its probability, and with it the row, not a number
    const float base = mn == -INFINITY ? 0.f : mn;
    if ((tid & 3) == 0) s_p[t] = seen ? expf(s - base) : 0.f;
    __syncthreads();
    const float corr = m == -INFINITY ? 0.f : expf(m - base);
    m = mn;
    l *= corr;
    acc *= corr;
    const float vsc = open ? 0.f : c.vs[bh * nb + blk];
#pragma unroll 4
    for (int i = 0; i < KB; ++i) l += s_p[i];
    for (int i = 0; i < PT; ++i) {
      const int tt = oh * PT + i, jj = blk * KB + tt;
      if (jj < lo || jj > pos) continue;
      float vv;
      if (open) vv = __bfloat162float(tt == slot ? s_new[1][od] : c.vt[(bh * KB + tt) * D + od]);
      else vv = kv8_value(c.v[(bh * nb + blk) * KB * D + od * KB + tt], vsc);
      acc += s_p[tt] * vv;
    }
    __syncthreads();
  }
  if (PARTS == 2) {
    s_out[oh][od] = acc;
    __syncthreads();
    if (tid < D) out[tid] = __float2bfloat16(l != 0.f ? (s_out[0][tid] + s_out[1][tid]) / l : 0.f);
  } else {
    float* four = reinterpret_cast<float*>(sm.turn);
    four[tid] = acc;
    __syncthreads();
    if (tid < D) out[tid] = __float2bfloat16(l != 0.f ? ((four[tid] + four[tid + D]) + (four[tid + 2 * D] + four[tid + 3 * D])) / l : 0.f);
  }
  if (slot == KB - 1) {
    __syncthreads();
    kv8_quantise_block<D, false>([&](int t, int d) -> const __nv_bfloat16* { return t == slot ? s_new[0] + d : c.kt + (bh * KB + t) * D + d; },
                                 c.k + (bh * cap + (long long)blk_new * KB) * D, c.ks + bh * nb + blk_new, sm);
    kv8_quantise_block<D, true>([&](int t, int d) -> const __nv_bfloat16* { return t == slot ? s_new[1] + d : c.vt + (bh * KB + t) * D + d; },
                                c.v + (bh * cap + (long long)blk_new * KB) * D, c.vs + bh * nb + blk_new, sm);
  }
}

inline bool kv8_refused(const Kv8& c, int B, int H, int D, int cap) {
  return B < 1 || H < 1 || B > 65535 || H > 65535 || (D != 64 && D != 128) || cap < KB || (cap % KB) || misaligned16(c.k, c.v, c.ks, c.vs, c.kt, c.vt) ||
         !c.k || !c.v || !c.ks || !c.vs || !c.kt || !c.vt;
}

}  // namespace bones

extern "C" {
using namespace bones;

// k, v: bf16, distances of sequences, tokens and heads in values (multiples of 8); pos, len: an address and the distance between two
// sequences' values, or a value for all.  A sequence at a negative position, without tokens or with more than fit is left as it was.
int bones_kv8_append(void* k8, void* v8, float* ks, float* vs, void* kt, void* vt, const void* k, const void* v, long long kb, long long kst, long long kh,
                     long long vb, long long vst, long long vh, int B, int H, int D, int cap, int t, const int* pos, int pos_step, int pos0, const int* len,
                     int len_step, int len0, void* stream) {
  const Kv8 c{(int8_t*)k8, (int8_t*)v8, ks, vs, (__nv_bfloat16*)kt, (__nv_bfloat16*)vt};
  if (kv8_refused(c, B, H, D, cap) || t < 0 || !k || !v || misaligned16(k, v) || ((kst | vst | (B > 1 ? kb | vb : 0) | (H > 1 ? kh | vh : 0)) % 8)) return -2;
  if (t == 0) return 0;
  // t tokens touch this many blocks at most; none lies past the capacity
  const long long blocks = min(((long long)t + KB - 2) / KB + 1, (long long)cap / KB);
  const dim3 grid((unsigned)(2 * blocks), (unsigned)H, (unsigned)B);
  (D == 128 ? kv8_append_kernel<128> : kv8_append_kernel<64>)<<<grid, QT, 0, (cudaStream_t)stream>>>(
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

// qkv: bf16 rows of 3 * H * D, ldq apart; cosT, sinT: fp32 [rope_rows, D / 2]; y: bf16 [B, H * D]; window_tiles: of 128 tokens, 0 for all.
int bones_kv8_attention(const void* qkv, long long ldq, const float* cosT, const float* sinT, int rope_rows, void* k8, void* v8, float* ks, float* vs, void* kt,
                        void* vt, const int* pos, int pos_step, int pos0, const int* doc_start, void* y, int B, int H, int D, int cap, float scale,
                        int window_tiles, int pdl, void* stream) {
  const Kv8 c{(int8_t*)k8, (int8_t*)v8, ks, vs, (__nv_bfloat16*)kt, (__nv_bfloat16*)vt};
  if (kv8_refused(c, B, H, D, cap) || !qkv || !cosT || !sinT || !y || misaligned16(qkv, y) || (B > 1 && ldq % 8) || window_tiles < 0) return -2;
  (void)pdl;
  const dim3 grid((unsigned)H, (unsigned)B);
  (D == 128 ? kv8_attn_kernel<128> : kv8_attn_kernel<64>)<<<grid, 256, 0, (cudaStream_t)stream>>>(
      (const __nv_bfloat16*)qkv, ldq, cosT, sinT, rope_rows, c, PerSeq{pos, pos_step, pos0}, doc_start, (__nv_bfloat16*)y, H, cap, scale, window_tiles);
  return (int)cudaGetLastError();
}
}  // extern "C"
