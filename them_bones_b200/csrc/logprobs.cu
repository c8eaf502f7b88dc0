// What rows of logits say about tokens: log-probability of a given one, entropy, the most probable alternatives, and the gradient.
//
//   m = max z, w_v = z_v - m, S = sum e^w_v, T = sum e^w_v w_v
//   log p_v = w_v - log S,  entropy = log S - T / S
//   d z_v = -p_v (G + g_H (log p_v + entropy)) + [v = t] g + sum_j [v = id_j] g_j,   G = g + sum_j g_j
//
// Alternatives are ordered by their logits, equal ones by their index, a NaN before everything.
//
// Forward: one pass over the row.  A thread keeps a running maximum with its S and T.  The alternatives come out of that: among the maxima
// of groups of threads the k-th largest bounds the row's k-th largest logit from below, so only threads whose maximum reaches it hold an
// alternative, and only their columns (a few percent of the row, still in L2) are looked at again.
// Gradient: one element-wise pass; the few columns with a gradient of their own are written once more.
//
// Bound by bytes, and in bf16 nearly as much by the exponentials (65 % of the special-function units' rate): 4096 rows of 65536, forward 98 us
// in bf16 (0.83 of the copy rate) and 158 in fp32 (1.03), with five alternatives 106 and 167; gradient 183 (0.90) and 326 (1.0).  One row takes 3.4 us,
// with 20 alternatives 6.9: latencies of the choice, which has a barrier between any two of its steps.  Before, 4096 rows with five alternatives:
// a pass for the maximum, one for the sums and one for each alternative 1580 us in fp32; one pass, and every thread's best column looked for
// again 214 (146 in bf16); the columns of all rounds of the threads that hold one looked at again 193 (109).
#include "decode_common.cuh"

namespace bones {

constexpr int LP_T = 128;                       // threads of a CTA (256: as fast for long rows, 37 us for 27 where 4096 rows have 8192 columns)
constexpr int LP_U = 4;                         // 16-byte vectors of a thread in flight
constexpr int LP_TOP = 32;                      // alternatives at most
constexpr int LP_GROUPS = 64;                   // of threads, whose maxima give the bound: two for each alternative at most
constexpr int LP_BT = 256;                      // threads of the gradient's CTAs
constexpr int LP_CAND = 1024;                   // columns kept for the final choice; a row that needs more is gone over once for each alternative
constexpr int LP_SPLIT = 16;                    // CTAs of a cluster, one row
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float lp_load(const float* p) { return *p; }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void lp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void lp_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
// a 16-byte vector: four fp32 or eight bf16
__device__ __forceinline__ void lp_unpack(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& u, float (&f)[8]) { unpack8(u, f); }
__device__ __forceinline__ uint4 lp_pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 lp_pack(const float (&f)[8]) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lp_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Order-preserving code of a logit: larger logits have larger codes, -0 and +0 the same, NaN the largest.  0 is below every logit's.
__device__ __forceinline__ uint32_t lp_code(float v) {
  if (v != v) return 0xfffffffeu;              // no key is all ones
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t code) {
  return code == 0xfffffffeu ? __int_as_float(0x7fc00000) : __uint_as_float((code & 0x80000000u) ? code & 0x7fffffffu : ~code);
}
// (logit, column) as one number: the larger comes first among alternatives; no two are equal
typedef unsigned long long LpKey;
__device__ __forceinline__ LpKey lp_key(float v, int c) { return (LpKey)lp_code(v) << 32 | (uint32_t)~c; }
__device__ __forceinline__ LpKey lp_first(LpKey a, LpKey b) { return a > b ? a : b; }

// running maximum, sum and weighted sum
struct LpSum {
  float m, s, t;
  // a larger maximum `n`; 1000 is further than any probability reaches, and keeps infinities out of the products
  __device__ __forceinline__ void raise(float n) {
    const float d = fmaxf(m - n, -1000.f), f = lp_exp2(d * kLog2e);
    t = f * fmaf(d, s, t);
    s *= f;
    m = n;
  }
  __device__ __forceinline__ void add(float z) {
    const float w = z - m, e = lp_exp2(w * kLog2e);
    s += e;
    t = fmaf(e, fmaxf(w, -1000.f), t);         // -inf has probability 0 and no part
  }
  __device__ __forceinline__ void join(LpSum o) {
    const float n = fmaxf(m, o.m);
    raise(n);
    o.raise(n);
    s += o.s;
    t += o.t;
  }
};

// A thread's sums over its vectors, relative to 2^m2, m2 = m log2 e rounded: one operation between a logit and its exponent.  The rounding
// of m2 moves all of a thread's exponents alike, by up to |m| 2^-24 log2 e: less than 1.5 for maxima within 2^24, which is what it is for
// (from 2^30 on it would be more than an exponent holds).  The maximum begins at -2^24, so that a masked stretch never becomes one; a
// thread whose own lies outside goes over its vectors again.  T is in units of log2.
constexpr float kLpMost = 16777216.0f;
struct LpStream {
  float m, m2, s, t;
  __device__ __forceinline__ LpStream() : m(-kLpMost), m2(-kLpMost * kLog2e), s(0.f), t(0.f) {}
  __device__ __forceinline__ void raise(float n) {
    const float n2 = n * kLog2e, d = fmaxf(m2 - n2, -1000.f), f = lp_exp2(d);
    t = f * fmaf(d, s, t);
    s *= f;
    m = n;
    m2 = n2;
  }
  __device__ __forceinline__ void add(float w) {               // w = z log2 e - m2, finite
    const float e = lp_exp2(w);
    s += e;
    t = fmaf(e, w, t);
  }
  __device__ __forceinline__ LpSum sum() const {               // relative to e^m: what the rounding of m2 moved goes back
    const float r = fmaf(m, kLog2e, -m2), f = lp_exp2(-r);
    return LpSum{m, f * s, f * kLn2 * fmaf(-r, s, t)};
  }
};
__device__ __forceinline__ float lp_most(const uint4& u, float) {
  return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
__device__ __forceinline__ float lp_most(const uint4& u, __nv_bfloat16) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ void lp_consume(LpStream& a, const uint4& u, float) {
  float f[4];
  lp_unpack(u, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float w;                                    // -inf has probability 0 and no part; a NaN stays one
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(w) : "f"(fmaf(f[i], kLog2e, -a.m2)), "f"(-1000.f));
    a.add(w);
  }
}
__device__ __forceinline__ void lp_consume(LpStream& a, const uint4& u, __nv_bfloat16) {
  const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;                                 // the same by twos, before they are unpacked: -1e30
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(x[i]), "r"(0xf14af14au));
    a.add(fmaf(__uint_as_float(v << 16), kLog2e, -a.m2));
    a.add(fmaf(__uint_as_float(v & 0xffff0000u), kLog2e, -a.m2));
  }
}

struct LpShared {
  LpKey cand[LP_CAND], top[LP_TOP], all[LP_SPLIT][LP_TOP], red[LP_T / 32];
  float group[LP_GROUPS], bound;
  LpSum warp[LP_T / 32], part[LP_SPLIT];
  int n_cand, n_round, n_hold;
  int round[LP_T];                              // thread | round << 8: columns of one round of a thread's
  unsigned short hold[LP_T];                    // threads of which all columns are looked at
};

// Places among n keys: key i with fewer than k larger ones goes to out[that number].
__device__ __forceinline__ void lp_rank(const LpKey* keys, int n, int k, LpKey* out) {
  for (int i = threadIdx.x; i < n; i += LP_T) {
    const LpKey mine = keys[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += keys[j] > mine;
    if (r < k) out[r] = mine;
  }
}

// Row r of a cluster: the columns of this CTA are `vecs` 16-byte vectors from `body` on (column `col0`), and in the first CTA up to
// 2 * (VE - 1) single columns before and behind the row's vectors.
template <class Z>
__global__ void __launch_bounds__(LP_T, 10) logprobs_fwd_kernel(const Z* __restrict__ logits, long long ldl, int V, const long long* __restrict__ tokens, int k,
                                                               float* __restrict__ given, float* __restrict__ entropy, float* __restrict__ top,
                                                               long long* __restrict__ ids, float4* __restrict__ stats) {
  constexpr int VE = 16 / sizeof(Z);
  __shared__ LpShared sm;
  const int S = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // waited for before the first store to another CTA
  const long long row = blockIdx.x / S;
  const Z* z = logits + row * ldl;
  const long long tk = rank == 0 && tid == 0 ? tokens[row] : -1;
  const float zt = tk >= 0 && tk < V ? lp_load(z + tk) : 0.f;
  if (tid == 0) sm.n_cand = sm.n_round = sm.n_hold = 0;
  const int head = min(V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(Z)), nv = (V - head) / VE, rest = V - head - nv * VE;
  const int v0 = (int)((long long)nv * rank / S), vecs = (int)((long long)nv * (rank + 1) / S) - v0, col0 = head + v0 * VE;
  const uint4* body = reinterpret_cast<const uint4*>(z + col0);
  auto single = [&](int i) { return i < head ? i : V - rest + (i - head); };             // column of single i
  const int singles = rank == 0 ? head + rest : 0;

  LpSum a;
  float best = -INFINITY, second = -INFINITY;   // of the thread's rounds of vectors
  int at = 0;                                   // the best one
  {
    LpStream w;
    for (int i = tid, it = 0; i < vecs; i += LP_U * LP_T, ++it) {
      uint4 u[LP_U];
#pragma unroll
      for (int j = 0; j < LP_U; ++j)
        if (i + j * LP_T < vecs) u[j] = lp_stream(body + i + j * LP_T);
      float n = -INFINITY;
#pragma unroll
      for (int j = 0; j < LP_U; ++j)
        if (i + j * LP_T < vecs) n = fmaxf(n, lp_most(u[j], Z()));
      second = fmaxf(second, fminf(best, n));
      if (n > best) {
        best = n;
        at = it;
        if (n > w.m) w.raise(n);
      }
#pragma unroll
      for (int j = 0; j < LP_U; ++j)
        if (i + j * LP_T < vecs) lp_consume(w, u[j], Z());
    }
    a = w.sum();
    if (!(best > -kLpMost && best < kLpMost)) {
      a = LpSum{-3.402823466e38f, 0.f, 0.f};
      if (best > a.m) a.m = best;
      for (int i = tid; i < vecs; i += LP_T) {
        float f[VE];
        lp_unpack(lp_stream(body + i), f);
#pragma unroll
        for (int e = 0; e < VE; ++e) a.add(f[e]);
      }
    }
  }
  if (tid < singles) {
    const float v = lp_load(z + single(tid));
    if (v > a.m) a.raise(v);
    a.add(v);
  }
  // the CTA's sums, and the maxima of groups
  {
    LpSum w = a;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w.join(LpSum{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.s, o), __shfl_xor_sync(0xffffffffu, w.t, o)});
    if (lane == 0) sm.warp[warp] = w;
    if (k > 0) {
      constexpr int PER = LP_T / LP_GROUPS;
      float g = best;
#pragma unroll
      for (int o = 1; o < PER; o *= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
      if ((lane & (PER - 1)) == 0) sm.group[tid / PER] = g;
    }
  }
  __syncthreads();
  a = sm.warp[0];
#pragma unroll
  for (int w = 1; w < LP_T / 32; ++w) a.join(sm.warp[w]);
  if (k > 0) {
    bool one_by_one = a.s != a.s;               // a NaN comes first, and no maximum saw it
    if (tid < LP_GROUPS) {
      const float g = sm.group[tid];
      int r = 0;
#pragma unroll 16
      for (int j = 0; j < LP_GROUPS; ++j) r += sm.group[j] > g || (sm.group[j] == g && j < tid);
      if (r == k - 1) sm.bound = g;
    } else if (tid < LP_GROUPS + LP_TOP) {
      sm.top[tid - LP_GROUPS] = 0;
    }
    __syncthreads();
    const float bound = sm.bound;
    const int turns = (vecs + LP_T - 1) / LP_T;
    // columns from `bound` on (or above it), of the threads that have one
    auto collect = [&](bool above) {
      auto keep = [&](float v, int c) {
        if (above ? v > bound : v >= bound) {
          const int n = atomicAdd(&sm.n_cand, 1);
          if (n < LP_CAND) sm.cand[n] = lp_key(v, c);
        }
      };
      if (tid < singles) keep(lp_load(z + single(tid)), single(tid));
      auto vector = [&](int v) {
        if (v >= vecs) return;
        float f[VE];
        lp_unpack(lp_stream(body + v), f);
#pragma unroll
        for (int e = 0; e < VE; ++e) keep(f[e], col0 + v * VE + e);
      };
      const int rounds = sm.n_round * LP_U, all = sm.n_hold * turns;
      for (int i = tid; i < rounds; i += LP_T) {
        const int r = sm.round[i / LP_U];
        vector((r & 255) + ((r >> 8) * LP_U + i % LP_U) * LP_T);
      }
      for (int i = tid; i < all; i += LP_T) vector(sm.hold[i / turns] + i % turns * LP_T);
      __syncthreads();
    };
    if (!one_by_one) {
      if (tid < vecs && second >= bound) sm.hold[atomicAdd(&sm.n_hold, 1)] = (unsigned short)tid;
      else if (tid < vecs && best >= bound) sm.round[atomicAdd(&sm.n_round, 1)] = tid | at << 8;
      __syncthreads();
      collect(false);
      int n = sm.n_cand;
      if (n > LP_CAND) {                        // many equal ones: those above the bound, then the first ones that are equal to it
        __syncthreads();
        if (tid == 0) sm.n_cand = 0;
        __syncthreads();
        collect(true);
        n = sm.n_cand;
        int need = max(k - n, 0);
        one_by_one = n > LP_CAND - LP_TOP;
        if (!one_by_one) {
          auto first = [&](int c, float v, bool here) {        // one column a thread, columns ascending
            const unsigned who = __ballot_sync(0xffffffffu, here && v == bound);
            if (lane == 0) sm.red[warp] = __popc(who);
            __syncthreads();
            int before = __popc(who & ((1u << lane) - 1u)), total = 0;
            for (int w = 0; w < LP_T / 32; ++w) {
              before += w < warp ? (int)sm.red[w] : 0;
              total += (int)sm.red[w];
            }
            if (here && v == bound && before < need) sm.cand[n + before] = lp_key(v, c);
            n += min(total, need);
            need -= min(total, need);
            __syncthreads();
          };
          const int lowest = rank == 0 ? 0 : col0, highest = rank == 0 && S == 1 ? V : col0 + vecs * VE;
          for (int c = lowest; c < highest && need > 0; c += LP_T) first(c + tid, c + tid < highest ? lp_load(z + c + tid) : 0.f, c + tid < highest);
          if (rank == 0 && S > 1)
            for (int c = V - rest; c < V && need > 0; c += LP_T) first(c + tid, c + tid < V ? lp_load(z + c + tid) : 0.f, c + tid < V);
        }
      }
      if (!one_by_one) lp_rank(sm.cand, n, k, sm.top);
    }
    if (one_by_one) {
      LpKey last = ~0ull;
      for (int j = 0; j < k; ++j) {
        LpKey most = 0;
        auto look = [&](float v, int c) {
          const LpKey q = lp_key(v, c);
          if (q < last && q > most) most = q;
        };
        for (int i = tid; i < vecs; i += LP_T) {
          float f[VE];
          lp_unpack(lp_stream(body + i), f);
#pragma unroll
          for (int e = 0; e < VE; ++e) look(f[e], col0 + i * VE + e);
        }
        if (tid < singles) look(lp_load(z + single(tid)), single(tid));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = lp_first(most, __shfl_xor_sync(0xffffffffu, most, o));
        __syncthreads();
        if (lane == 0) sm.red[warp] = most;
        __syncthreads();
        most = sm.red[0];
        for (int w = 1; w < LP_T / 32; ++w) most = lp_first(most, sm.red[w]);
        last = most;
        if (tid == 0) sm.top[j] = most;
      }
    }
    __syncthreads();
  }
  if (S > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0) {
      const uint32_t to = map_to_rank(smem_u32(&sm.part[rank]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(a.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(a.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(a.t) : "memory");
    }
    if (tid < k) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_to_rank(smem_u32(&sm.all[rank][tid]), 0)), "l"(sm.top[tid]) : "memory");
    cluster_barrier();
    if (rank != 0) return;
    a = sm.part[0];
    for (int r = 1; r < S; ++r) a.join(sm.part[r]);
    // every CTA's descend: a lane each, the largest of their heads k times
    if (k > 0) {
      if (warp == 0) {
        LpKey cur = lane < S ? sm.all[lane][0] : 0, nxt = lane < S && k > 1 ? sm.all[lane][1] : 0;
        int i = 2;
        for (int j = 0; j < k; ++j) {
          const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(cur >> 32));
          const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(cur >> 32) == hi ? (uint32_t)cur : 0u);
          const LpKey most = (LpKey)hi << 32 | lo;
          if (cur == most) {
            sm.top[j] = most;
            cur = nxt;
            nxt = i < k ? sm.all[lane][i++] : 0;
          }
        }
      }
      __syncthreads();
    }
  }
  const float ls = logf(a.s);
  if (tid < k) {
    const LpKey q = sm.top[tid];
    ids[row * k + tid] = (long long)(uint32_t)~(uint32_t)q;
    top[row * k + tid] = lp_value((uint32_t)(q >> 32)) - a.m - ls;
  }
  if (tid == 0) {
    const float h = ls - a.t / a.s;
    given[row] = tk >= 0 && tk < V ? zt - a.m - ls : 0.f;
    entropy[row] = h;
    if (stats) stats[row] = make_float4(a.m, ls, h, 0.f);
  }
}

// One CTA for LP_U vectors a thread of a row.  `nic2`: -1 / cap^2 where the logits are z = cap tanh(x / cap) and the gradient is wanted of x
// (each is multiplied by 1 - (z / cap)^2), else 0.  dz may be the logits themselves.
template <class Z>
__global__ void __launch_bounds__(LP_BT) logprobs_bwd_kernel(const Z* logits, long long ldl, int V, int cols, const long long* __restrict__ tokens,
                                                            int k, const long long* __restrict__ ids, const float4* __restrict__ stats,
                                                            const float* __restrict__ g_given, const float* __restrict__ g_entropy,
                                                            const float* __restrict__ g_top, Z* dz, long long ldd, int chunks, float nic2) {
  constexpr int VE = 16 / sizeof(Z), CHUNK = LP_BT * LP_U * VE;
  const long long row = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - row * chunks), tid = threadIdx.x;
  const Z* z = logits + row * ldl;
  Z* d = dz + row * ldd;
  // vectors where rows of both begin alike, single columns where not, and before and behind the vectors
  const int mis = (int)((uintptr_t)d & 15), head = min(cols, (16 - mis & 15) / (int)sizeof(Z));
  const bool alike = (int)((uintptr_t)z & 15) == mis;
  // columns of this CTA
  const int c0 = chunk == 0 ? 0 : head + chunk * CHUNK, c1 = min(cols, head + (chunk + 1) * CHUNK);
  if (c0 >= cols) return;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  const int vb = head + chunk * CHUNK;
  uint4 u[LP_U];
  if (alike) {
#pragma unroll
    for (int j = 0; j < LP_U; ++j) {
      const int c = vb + (tid + j * LP_BT) * VE;
      u[j] = c + VE <= cols && c < V ? lp_stream(z + c) : none;
    }
  }
  const float4 st = stats[row];
  const long long tk = tokens[row];
  const bool some = tk >= 0 && tk < V;
  const float g = g_given && some ? g_given[row] : 0.f, gh = g_entropy ? g_entropy[row] : 0.f;
  float pull = g;
  bool idle = g == 0.f && gh == 0.f;            // nothing depends on this row: its gradient is 0 whatever the row holds
  if (g_top) {
    for (int j = 0; j < k; ++j) {
      const float x = g_top[row * k + j];
      pull += x;
      idle &= x == 0.f;
    }
  }
  // -p (pull + gh (log p + H)) with l = log2 p
  const float off = -st.y * kLog2e, ca = pull + gh * st.z, cb = gh * kLn2;
  auto grad = [&](float x) {
    const float l = fmaf(x - st.x, kLog2e, off);
    return -lp_exp2(l) * fmaf(cb, fmaxf(l, -1000.f), ca);
  };
  auto through = [&](float x) { return nic2 != 0.f ? fmaf(x * nic2, x, 1.0f) : 1.0f; };         // the soft-cap's own derivative
  // the columns with a gradient of their own, before anything is written
  const bool extra = !idle && tid <= k && (tid == k ? some : g_top != nullptr);
  const long long ec = !extra ? -1 : tid == k ? tk : ids[row * k + tid];
  const bool mine = ec >= c0 && ec < c1;
  const float ez = mine ? lp_load(z + ec) : 0.f;
  __syncthreads();
  auto one = [&](int c) {
    const float x = c < V && !idle ? lp_load(z + c) : 0.f;
    lp_store(d + c, c < V && !idle ? grad(x) * through(x) : 0.f);
  };
  if (alike) {
#pragma unroll
    for (int j = 0; j < LP_U; ++j) {
      const int c = vb + (tid + j * LP_BT) * VE;
      if (c + VE > cols) continue;
      float f[VE];
      lp_unpack(u[j], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = c + e < V && !idle ? grad(f[e]) * through(f[e]) : 0.f;
      *reinterpret_cast<uint4*>(d + c) = lp_pack(f);
    }
    const int full = head + (cols - head) / VE * VE;
    if (chunk == 0 && tid < head) one(tid);
    if (c1 == cols && tid < cols - full) one(full + tid);
  } else {
    for (int c = c0 + tid; c < c1; c += LP_BT) one(c);
  }
  if (idle) return;
  __syncthreads();
  if (mine) {
    float v = grad(ez);
    if (some && ec == tk) v += g;
    if (g_top)
      for (int j = 0; j < k; ++j)
        if (ids[row * k + j] == ec) v += g_top[row * k + j];
    lp_store(d + ec, v * through(ez));
  }
}

// CTAs of a cluster that share a row: doubled while there are few on an SM and every thread keeps two vectors; 16 only for a few rows.
// us, bf16 rows of 65536, 8 alternatives: 64 rows by 8 / 16 CTAs 9.5 / 10.5, 512 rows by 1 / 2 26 / 22.
inline int lp_splits(long long rows, int V, int per, int sms) {
  int s = 1;
  while (s < LP_SPLIT && rows * s < (s < 8 ? 4 : 1) * sms && V >= 2 * s * LP_T * per) s *= 2;
  return s;
}

template <class Z>
int launch_logprobs_fwd(const void* logits, long long ldl, long long rows, int V, const long long* tokens, int k, float* given, float* entropy, float* top,
                        long long* ids, void* stats, cudaStream_t s) {
  static OncePerDevice once;
  BONES_ONCE(once, {
    BONES_CHECK(cudaFuncSetAttribute(logprobs_fwd_kernel<Z>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  });
  int dev = 0, sms = 0;
  BONES_CHECK(cudaGetDevice(&dev));
  BONES_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int split = lp_splits(rows, V, 16 / (int)sizeof(Z), sms);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)(rows * split));
  cfg.blockDim = dim3(LP_T);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, split, 0);
  return (int)cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<Z>, (const Z*)logits, ldl, V, tokens, k, given, entropy, top, ids, (float4*)stats);
}
template <class Z>
int launch_logprobs_bwd(const void* logits, long long ldl, long long rows, int V, int cols, const long long* tokens, int k, const long long* ids,
                        const void* stats, const float* g_given, const float* g_entropy, const float* g_top, void* dz, long long ldd, float nic2, cudaStream_t s) {
  const int chunk = LP_BT * LP_U * (16 / (int)sizeof(Z)), chunks = (cols + chunk - 1) / chunk;
  if (rows * chunks > 0x7fffffffll) return -2;
  logprobs_bwd_kernel<Z><<<(unsigned)(rows * chunks), LP_BT, 0, s>>>((const Z*)logits, ldl, V, cols, tokens, k, ids, (const float4*)stats, g_given, g_entropy,
                                                                    g_top, (Z*)dz, ldd, chunks, nic2);
  return (int)cudaGetLastError();
}

}  // namespace bones

extern "C" {
using namespace bones;

// logits: rows of bf16 (fp32: `wide`), ldl values apart, at any multiple of their size; the first V columns are the vocabulary.
// top, ids: [rows, k], k <= 32 and <= V; stats: [rows] float4 or null where no gradient follows
int bones_logprobs_fwd(const void* logits, long long ldl, int wide, long long rows, int V, const long long* tokens, int k, float* given, float* entropy,
                       float* top, long long* ids, void* stats, void* stream) {
  if (rows == 0) return 0;                     // empty tensors have no address
  if (rows < 0 || rows > 0x7fffffffll || V < 1 || V > (1 << 30) || k < 0 || k > LP_TOP || k > V || (k && (!top || !ids)) || ((uintptr_t)stats & 15)) return -2;
  return wide ? launch_logprobs_fwd<float>(logits, ldl, rows, V, tokens, k, given, entropy, top, ids, stats, (cudaStream_t)stream)
              : launch_logprobs_fwd<__nv_bfloat16>(logits, ldl, rows, V, tokens, k, given, entropy, top, ids, stats, (cudaStream_t)stream);
}

// g_given, g_entropy [rows] and g_top [rows, k]: null where there is no gradient; dz: `cols` columns, those behind the vocabulary become 0;
// it may be the logits.  cap > 0: the logits are soft-capped, and the gradient is that of what they were before.
int bones_logprobs_bwd(const void* logits, long long ldl, int wide, long long rows, int V, int cols, const long long* tokens, int k, const long long* ids,
                       const void* stats, const float* g_given, const float* g_entropy, const float* g_top, void* dz, long long ldd, float cap,
                       void* stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > 0x7fffffffll || V < 1 || cols < V || cols > (1 << 30) || k < 0 || k > LP_TOP || (k && g_top && !ids) || !stats || ((uintptr_t)stats & 15)) return -2;
  const float nic2 = cap > 0.f ? -1.0f / (cap * cap) : 0.f;
  return wide ? launch_logprobs_bwd<float>(logits, ldl, rows, V, cols, tokens, k, ids, stats, g_given, g_entropy, g_top, dz, ldd, nic2, (cudaStream_t)stream)
              : launch_logprobs_bwd<__nv_bfloat16>(logits, ldl, rows, V, cols, tokens, k, ids, stats, g_given, g_entropy, g_top, dz, ldd, nic2, (cudaStream_t)stream);
}
}  // extern "C"
