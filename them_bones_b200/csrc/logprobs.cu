// What rows of logits say about tokens: log-probability of a given one, entropy, the most probable alternatives, and the gradient.
//
//   m = max z, w_v = z_v - m, S = sum e^w_v, T = sum e^w_v w_v
//   log p_v = w_v - log S,  entropy = log S - T / S
//   d z_v = -p_v (G + g_H (log p_v + entropy)) + [v = t] g + sum_j [v = id_j] g_j,   G = g + sum_j g_j
//
// Alternatives are ordered by their logits, equal ones by their index, a NaN before everything.
#include "common.cuh"

namespace bones {

constexpr int LP_T = 512;
constexpr int LP_TOP = 32;                      // alternatives at most

__device__ __forceinline__ float lp_load(const float* p) { return *p; }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void lp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void lp_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// Order-preserving code of a logit: larger logits have larger codes, -0 and +0 the same, NaN the largest.  0 is below every logit's.
__device__ __forceinline__ uint32_t lp_code(float v) {
  if (v != v) return 0xfffffffeu;              // no key is all ones
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// (logit, column) as one number: the larger comes first among alternatives
__device__ __forceinline__ unsigned long long lp_key(float v, int c) { return (unsigned long long)lp_code(v) << 32 | (uint32_t)~c; }

template <class F>
__device__ __forceinline__ F lp_block(F v, F* red, F (*op)(F, F)) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < LP_T / 32; ++w) v = op(v, red[w]);
  return v;
}
__device__ __forceinline__ float lp_add(float a, float b) { return a + b; }
__device__ __forceinline__ float lp_max(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ unsigned long long lp_first(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// One CTA a row.  stats [rows][4]: m, log S, entropy, 0.
template <class Z>
__global__ void __launch_bounds__(LP_T) logprobs_fwd_kernel(const Z* __restrict__ logits, long long ldl, int V, const long long* __restrict__ tokens, int k,
                                                            float* __restrict__ given, float* __restrict__ entropy, float* __restrict__ top,
                                                            long long* __restrict__ ids, float4* __restrict__ stats) {
  __shared__ float fred[LP_T / 32];
  __shared__ unsigned long long kred[LP_T / 32];
  const long long row = blockIdx.x;
  const Z* z = logits + row * ldl;
  float m = -INFINITY;
  for (int c = threadIdx.x; c < V; c += LP_T) m = fmaxf(m, lp_load(z + c));
  m = lp_block<float>(m, fred, lp_max);
  float s = 0.f, t = 0.f;
  for (int c = threadIdx.x; c < V; c += LP_T) {
    const float w = lp_load(z + c) - m, e = expf(w);
    s += e;
    t += e * fmaxf(w, -1000.f);                // e is 0 there; -inf has no part
  }
  s = lp_block<float>(s, fred, lp_add);
  t = lp_block<float>(t, fred, lp_add);
  const float ls = logf(s), h = ls - t / s;
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int c = threadIdx.x; c < V; c += LP_T) {
      const unsigned long long q = lp_key(lp_load(z + c), c);
      if (q < last && q > best) best = q;
    }
    best = lp_block<unsigned long long>(best, kred, lp_first);
    last = best;
    if (threadIdx.x == 0) {
      const int c = (int)~(uint32_t)best;
      ids[row * k + j] = c;
      top[row * k + j] = lp_load(z + c) - m - ls;
    }
  }
  if (threadIdx.x == 0) {
    const long long tk = tokens[row];
    given[row] = tk >= 0 && tk < V ? lp_load(z + tk) - m - ls : 0.f;
    entropy[row] = h;
    if (stats) stats[row] = make_float4(m, ls, h, 0.f);
  }
}

// One CTA a row; the given token's and the alternatives' columns are done once more, with what they get besides.
template <class Z>
__global__ void __launch_bounds__(LP_T) logprobs_bwd_kernel(const Z* __restrict__ logits, long long ldl, int V, int cols, const long long* __restrict__ tokens,
                                                            int k, const long long* __restrict__ ids, const float4* __restrict__ stats,
                                                            const float* __restrict__ g_given, const float* __restrict__ g_entropy,
                                                            const float* __restrict__ g_top, Z* __restrict__ dz, long long ldd) {
  const long long row = blockIdx.x;
  const Z* z = logits + row * ldl;
  Z* d = dz + row * ldd;
  const float4 st = stats[row];
  const long long tk = tokens[row];
  const bool some = tk >= 0 && tk < V;
  const float g = g_given && some ? g_given[row] : 0.f, gh = g_entropy ? g_entropy[row] : 0.f;
  float pull = g;
  if (g_top)
    for (int j = 0; j < k; ++j) pull += g_top[row * k + j];
  // nothing depends on this row: its gradient is 0 whatever the row holds
  bool idle = g == 0.f && gh == 0.f;
  if (g_top)
    for (int j = 0; j < k; ++j) idle &= g_top[row * k + j] == 0.f;
  if (idle) {
    for (int c = threadIdx.x; c < cols; c += LP_T) lp_store(d + c, 0.f);
    return;
  }
  auto grad = [&](int c) {
    const float lp = lp_load(z + c) - st.x - st.y;
    return -expf(lp) * (pull + gh * (fmaxf(lp, -1000.f) + st.z));
  };
  for (int c = threadIdx.x; c < cols; c += LP_T) lp_store(d + c, c < V ? grad(c) : 0.f);
  __syncthreads();
  if ((int)threadIdx.x <= k) {
    const bool own = (int)threadIdx.x == k;
    if (own ? some : g_top != nullptr) {
      const int c = (int)(own ? tk : ids[row * k + threadIdx.x]);
      float v = grad(c);
      if (some && c == tk) v += g;
      if (g_top)
        for (int j = 0; j < k; ++j)
          if (ids[row * k + j] == c) v += g_top[row * k + j];
      lp_store(d + c, v);
    }
  }
}

}  // namespace bones

extern "C" {
using namespace bones;

// logits: rows of bf16 (fp32: `wide`), ldl values apart; the first V columns are the vocabulary.  top, ids: [rows, k], k <= 32 and <= V.
int bones_logprobs_fwd(const void* logits, long long ldl, int wide, long long rows, int V, const long long* tokens, int k, float* given, float* entropy,
                       float* top, long long* ids, void* stats, void* stream) {
  if (rows == 0) return 0;                     // empty tensors have no address
  if (rows < 0 || rows > 0x7fffffffll || V < 1 || k < 0 || k > LP_TOP || k > V || (k && (!top || !ids)) || ((uintptr_t)stats & 15)) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (wide)
    logprobs_fwd_kernel<float><<<(unsigned)rows, LP_T, 0, s>>>((const float*)logits, ldl, V, tokens, k, given, entropy, top, ids, (float4*)stats);
  else
    logprobs_fwd_kernel<__nv_bfloat16><<<(unsigned)rows, LP_T, 0, s>>>((const __nv_bfloat16*)logits, ldl, V, tokens, k, given, entropy, top, ids,
                                                                        (float4*)stats);
  return (int)cudaGetLastError();
}

// g_given, g_entropy [rows] and g_top [rows, k]: null where there is no gradient; dz: `cols` columns, those behind the vocabulary become 0
int bones_logprobs_bwd(const void* logits, long long ldl, int wide, long long rows, int V, int cols, const long long* tokens, int k, const long long* ids,
                       const void* stats, const float* g_given, const float* g_entropy, const float* g_top, void* dz, long long ldd, void* stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > 0x7fffffffll || V < 1 || cols < V || k < 0 || k > LP_TOP || (k && g_top && !ids) || !stats || ((uintptr_t)stats & 15)) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (wide)
    logprobs_bwd_kernel<float><<<(unsigned)rows, LP_T, 0, s>>>((const float*)logits, ldl, V, cols, tokens, k, ids, (const float4*)stats, g_given, g_entropy,
                                                                g_top, (float*)dz, ldd);
  else
    logprobs_bwd_kernel<__nv_bfloat16><<<(unsigned)rows, LP_T, 0, s>>>((const __nv_bfloat16*)logits, ldl, V, cols, tokens, k, ids, (const float4*)stats,
                                                                        g_given, g_entropy, g_top, (__nv_bfloat16*)dz, ldd);
  return (int)cudaGetLastError();
}
}  // extern "C"
