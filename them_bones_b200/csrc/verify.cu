// Verification of drafted tokens.
//
// Row r says p = softmax(z_r / T) of the token behind it, and the draft x there was drawn from q (the draft rows' soft-max, or certainty).  It stands
// while u_r0 q(x) < p(x); at the first that does not, the token is drawn from max(p - q, 0), behind the last draft from p, by the inverse
// distribution function at u_r1.  T = 0: the arg-max throughout.
//
// Two kernels.  The first reads every row once and leaves its maximum and its sum of exponentials.  The second, a cluster a sequence, goes
// through the sequence's drafts and draws the token from the one row that decides.  Its sums are in 64 bits: a border of the distribution
// function in 32 would move by more than the gap of a rare token's interval, and the token with it (65536 columns: one draw in some hundred).
// A draft whose test is closer than the first kernel's 32-bit exponentials can tell is decided on sums in 64 bits too.
#include "decode_common.cuh"
#include "paged.cuh"

namespace bones {

struct RowStat {
  double sum;        // of exp((z - most) / T); 0: a row without a number
  float most;
  int best;          // the lowest index of the maximum
};

struct VerifyArgs {
  const void *z, *q;           // target's and draft's logits (or null)
  long long ldz, ldq;
  const long long* ids;
  const int* starts;
  const float* u;              // [N, 2]
  int B, N, V;
  double T;
  RowStat* stats;              // [N, 2]
  int* accepted;
  long long* token;
};

template <typename E>
__device__ __forceinline__ float logit(const E* p) {
  if constexpr (sizeof(E) == 2) return __bfloat162float(*p);
  else return *p;
}
// values a load of 16 bytes has
template <typename E>
constexpr int kVec = 16 / sizeof(E);
template <typename E>
__device__ __forceinline__ void load_vec(const E* p, float* f) {
  if constexpr (sizeof(E) == 2) unpack8(*reinterpret_cast<const uint4*>(p), f);
  else {
    const float4 a = *reinterpret_cast<const float4*>(p);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  }
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------------------------------------------------
// a row's maximum, sum and arg-max.  grid: (N, 1 or 2 models)
// ---------------------------------------------------------------------------------------------------------------
struct RowRun {
  float most, sum;
  int best;
  bool bad;          // GREEDY: a NaN or +inf came by (else the sum is NaN)
};

template <bool GREEDY, int W>
__device__ __forceinline__ void row_step(RowRun& r, const float* f, int at, float c) {
  if (GREEDY) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (!(f[i] < __int_as_float(0x7f800000))) r.bad = true;
      if (f[i] > r.most) {
        r.most = f[i];
        r.best = at + i;
      }
    }
  } else {
    float m = f[0];
#pragma unroll
    for (int i = 1; i < W; ++i) m = fmaxf(m, f[i]);
    if (m > r.most) {
      r.sum *= ex2((r.most - m) * c);
      r.most = m;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += ex2((f[i] - r.most) * c);
    r.sum += s;
  }
}

template <typename E, bool GREEDY>
__global__ void verify_stats_kernel(const VerifyArgs p) {
  const int row = blockIdx.x, model = blockIdx.y;
  pdl_launch();
  const int seq = paged_owner(p.starts, p.B, row);
  if (seq < 0 || seq >= p.B || (model && row + 1 >= p.starts[seq + 1])) return;      // no sequence's, or nothing was drawn from it
  const E* z = model ? (const E*)p.q + row * p.ldq : (const E*)p.z + row * p.ldz;
  const float c = GREEDY ? 0.f : (float)(1.4426950408889634 / p.T);
  RowRun r{-3.402823466e38f, 0.f, -1, false};
  constexpr int W = kVec<E>;
  // single values up to the first 16-byte boundary, vectors, single values
  const int head = min(p.V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(E)), vecs = (p.V - head) / W, tail = head + vecs * W;
  if (threadIdx.x < head) {
    const float f = logit(z + threadIdx.x);
    row_step<GREEDY, 1>(r, &f, threadIdx.x, c);
  }
  constexpr int U = 4;                               // loads of a thread in flight
  int i = threadIdx.x;
  for (; i + (U - 1) * (int)blockDim.x < vecs; i += U * blockDim.x) {
    float f[U][W];
#pragma unroll
    for (int j = 0; j < U; ++j) load_vec(z + head + (long long)(i + j * blockDim.x) * W, f[j]);
#pragma unroll
    for (int j = 0; j < U; ++j) row_step<GREEDY, W>(r, f[j], head + (i + j * blockDim.x) * W, c);
  }
  for (; i < vecs; i += blockDim.x) {
    float f[W];
    load_vec(z + head + (long long)i * W, f);
    row_step<GREEDY, W>(r, f, head + i * W, c);
  }
  if (tail + (int)threadIdx.x < p.V) {
    const float f = logit(z + tail + threadIdx.x);
    row_step<GREEDY, 1>(r, &f, tail + threadIdx.x, c);
  }
  // the threads' together; the lowest index of equals
  __shared__ float sm[32];
  __shared__ double ss[32];
  __shared__ int si[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float wm = warp_max(r.most);
  if (lane == 0) sm[warp] = wm;
  __syncthreads();
  float m = sm[0];
  for (int w = 1; w < warps; ++w) m = fmaxf(m, sm[w]);
  if (GREEDY) {
    const bool bad = __syncthreads_or(r.bad);
    const int b = __reduce_min_sync(0xffffffffu, r.most == m && r.best >= 0 ? r.best : 0x7fffffff);
    if (lane == 0) si[warp] = b;
    __syncthreads();
    if (threadIdx.x == 0) {
      int best = si[0];
      for (int w = 1; w < warps; ++w) best = min(best, si[w]);
      p.stats[row * 2ll + model] = RowStat{bad || best == 0x7fffffff ? 0.0 : 1.0, m, best};
    }
    return;
  }
  double s = r.sum == 0.f ? 0.0 : (double)(r.sum * ex2((r.most - m) * c));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) ss[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < warps; ++w) s += ss[w];
    p.stats[row * 2ll + model] = RowStat{s > 0.0 && s < 1e300 ? s : 0.0, m, -1};          // NaN or +inf: a sum that is NaN
  }
}

// ---------------------------------------------------------------------------------------------------------------
// a sequence: which drafts stand, and the token.  grid: (VC CTAs of a cluster, B)
// ---------------------------------------------------------------------------------------------------------------
constexpr int VC = 8, VT = 256, VW = VC * VT / 32;       // CTAs, threads of one, warps of a cluster
static_assert(VW == 64, "a lane has two warps' sums");

template <typename E>
struct Law {                  // exp((z - most) / T), 64 bits
  const E* z;
  double most, inv;
  __device__ __forceinline__ double operator()(double x) const { return exp((x - most) * inv); }
};

// eight columns from `at` on, -inf behind the last
template <typename E>
__device__ __forceinline__ void load8(const E* z, int at, int V, float* f) {
  if (at + 8 <= V && ((uintptr_t)(z + at) & 15) == 0) {
    load_vec(z + at, f);
    if constexpr (sizeof(E) == 4) load_vec(z + at + 4, f + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = at + i < V ? logit(z + at + i) : -__int_as_float(0x7f800000);
  }
}

// A double of each warp to all: lane l gets those of warps 2 l and 2 l + 1 of the cluster.
struct Both {
  double a, b;
};
__device__ __forceinline__ Both share(double mine, double* box) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) box[warp] = mine;
  __syncthreads();
  cluster_barrier();
  const uint32_t at = map_to_rank(smem_u32(box + (2 * lane) % (VT / 32)), (2 * lane) / (VT / 32));
  Both r;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(r.a) : "r"(at));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(r.b) : "r"(at + 8));
  __syncwarp();
  cluster_barrier();
  return r;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename E>
__global__ void __cluster_dims__(VC, 1, 1) __launch_bounds__(VT) verify_draw_kernel(const VerifyArgs p) {
  __shared__ double box[VT / 32];
  pdl_wait();
  const int seq = blockIdx.y, lane = threadIdx.x & 31, gw = (int)cluster_rank() * (VT / 32) + (threadIdx.x >> 5);
  const int a = min(max(p.starts[seq], 0), p.N), e = min(max(p.starts[seq + 1], a), p.N);
  const bool writer = cluster_rank() == 0 && threadIdx.x == 0;
  if (a == e) {
    if (writer) {
      p.accepted[seq] = 0;
      p.token[seq] = -1;
    }
    return;
  }
  const double inv = 1.0 / p.T;
  // this warp's columns: whole tiles of 256, consecutive warps consecutive columns
  const int tiles = (p.V + 255) / 256, mine = (tiles + VW - 1) / VW, t0 = min(gw * mine, tiles), t1 = min(t0 + mine, tiles);
  auto total = [&](const E* z, double most) {
    const Law<E> law{z, most, inv};
    double s = 0.0;
    for (int t = t0; t < t1; ++t) {
      float f[8];
      load8(z, t * 256 + lane * 8, p.V, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += law(f[i]);
    }
    const Both r = share(warp_sum64(s), box);
    return warp_sum64(r.a + r.b);
  };
  auto target = [&](int r) { return (const E*)p.z + r * p.ldz; };
  auto draft = [&](int r) { return (const E*)p.q + r * p.ldq; };

  // 32 rows at a time, a lane a row.  All warps come to the same.
  enum { STANDS, FALLS, CLOSE, GONE };
  int row = e - 1, why = FALLS;
  for (int r0 = a; r0 < e; r0 += 32) {
    const int r = r0 + lane;
    int is = FALLS;
    if (r < e) {
      const RowStat st = p.stats[r * 2ll];
      if (!(st.sum > 0.0)) is = GONE;
      else if (r + 1 < e) {
        const long long x = p.ids[r + 1];
        const RowStat sq = p.q ? p.stats[r * 2ll + 1] : RowStat{1.0, 0.f, 0};
        if (x >= 0 && x < p.V && sq.sum > 0.0) {
          const double px = exp(((double)logit(target(r) + x) - st.most) * inv) / st.sum;
          const double qx = p.q ? exp(((double)logit(draft(r) + x) - sq.most) * inv) / sq.sum : 1.0, need = p.u[2ll * r] * qx;
          is = fabs(need - px) <= 1e-4 * (need + px) ? CLOSE : need < px ? STANDS : FALLS;
        }
      }
    }
    uint32_t open = __ballot_sync(0xffffffffu, is != STANDS);
    while (open) {
      const int l = __ffs(open) - 1;
      const int it = __shfl_sync(0xffffffffu, is, l);
      if (it == CLOSE) {
        const int rr = r0 + l;
        const float mp = p.stats[rr * 2ll].most, mq = p.q ? p.stats[rr * 2ll + 1].most : 0.f;
        const long long x = p.ids[rr + 1];
        const double sp = total(target(rr), mp), sq = p.q ? total(draft(rr), mq) : 1.0;
        const double px = exp(((double)logit(target(rr) + x) - mp) * inv) / sp;
        const double qx = p.q ? exp(((double)logit(draft(rr) + x) - mq) * inv) / sq : 1.0;
        if (p.u[2ll * rr] * qx < px) {
          open &= open - 1;
          continue;
        }
      }
      row = r0 + l;
      why = it == GONE ? GONE : FALLS;
      break;
    }
    if (open) break;
  }
  row = min(row, e - 1);
  if (writer) p.accepted[seq] = row - a;
  if (why == GONE) {
    if (writer) p.token[seq] = -1;
    return;
  }
  // the row that decides: w = p, max(p - q, 0) or p without the draft
  const bool refused = row + 1 < e;
  const RowStat st = p.stats[row * 2ll], sq = refused && p.q ? p.stats[row * 2ll + 1] : RowStat{0.0, 0.f, 0};
  const E *z = target(row), *zq = sq.sum > 0.0 ? draft(row) : nullptr;
  const long long without = refused && !p.q ? p.ids[row + 1] : -1;
  const Law<E> lp{z, st.most, inv}, lq{zq, sq.most, inv};
  double sp = 1.0, sd = 1.0;
  if (zq) {                                    // p's and q's scales matter only beside one another
    sp = 1.0 / total(z, st.most);
    sd = 1.0 / total(zq, sq.most);
  }
  bool plain = false;                          // of p alone
  auto weights = [&](int t, double* w) {
    const int at = t * 256 + lane * 8;
    float f[8], g[8];
    load8(z, at, p.V, f);
    if (zq && !plain) load8(zq, at, p.V, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double x = lp(f[i]) * sp;
      if (zq && !plain) x = fmax(x - lq(g[i]) * sd, 0.0);
      if (at + i == without && !plain) x = 0.0;
      w[i] = x;
    }
  };
  for (int round = 0; round < 2; ++round) {
    double s = 0.0;
    for (int t = t0; t < t1; ++t) {
      double w[8];
      weights(t, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += w[i];
    }
    const Both r = share(warp_sum64(s), box);
    // sums up to and with each warp's
    double up = r.a + r.b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    const double all = __shfl_sync(0xffffffffu, up, 31);
    double prev = __shfl_up_sync(0xffffffffu, up, 1);
    if (lane == 0) prev = 0.0;
    if (!(all > 0.0) && !plain) {              // p and q the same but for rounding: of p
      plain = true;
      continue;
    }
    const double need = (double)p.u[2ll * row + 1] * all;
    // the first warp with weight whose sum reaches above; by rounding there may be none: the last with weight
    const double first = prev + r.a;
    int w = r.a > 0.0 && first > need ? 2 * lane : r.b > 0.0 && up > need ? 2 * lane + 1 : VW;
    w = __reduce_min_sync(0xffffffffu, w);
    if (w == VW) w = __reduce_max_sync(0xffffffffu, r.b > 0.0 ? 2 * lane + 1 : r.a > 0.0 ? 2 * lane : 0);
    if (w == gw) {
      double before = __shfl_sync(0xffffffffu, (w & 1) ? first : prev, w >> 1);
      int found = -1, last = -1;
      for (int t = t0; t < t1 && found < 0; ++t) {
        double x[8], sum = 0.0;
        weights(t, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[i];
        double to = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, to, o);
          if (lane >= o) to += y;
        }
        double at = before + to - sum;
        int hit = 0x7fffffff, tail = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          at += x[i];
          if (x[i] > 0.0) {
            tail = t * 256 + lane * 8 + i;
            if (at > need && hit == 0x7fffffff) hit = tail;
          }
        }
        hit = __reduce_min_sync(0xffffffffu, hit);
        last = max(last, __reduce_max_sync(0xffffffffu, tail));
        if (hit != 0x7fffffff) found = hit;
        before += __shfl_sync(0xffffffffu, to, 31);
      }
      if (lane == 0) p.token[seq] = found >= 0 ? found : last;
    }
    break;
  }
}

// T = 0.  A warp a sequence.
__global__ void __launch_bounds__(128) verify_greedy_kernel(const VerifyArgs p) {
  pdl_wait();
  const int seq = (int)((blockIdx.x * 128 + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  if (seq >= p.B) return;
  const int a = min(max(p.starts[seq], 0), p.N), e = min(max(p.starts[seq + 1], a), p.N);
  int row = a;
  long long token = -1;
  for (int r0 = a; r0 < e; r0 += 32) {
    const int r = r0 + lane;
    bool stop = true;
    int best = -1;
    if (r < e) {
      const RowStat st = p.stats[r * 2ll];
      best = st.sum > 0.0 ? st.best : -1;
      stop = r + 1 == e || best < 0 || p.ids[r + 1] != best;
    }
    const uint32_t open = __ballot_sync(0xffffffffu, stop);
    if (open) {
      const int l = __ffs(open) - 1;
      row = r0 + l;
      token = __shfl_sync(0xffffffffu, best, l);
      break;
    }
  }
  if (lane == 0) {
    p.accepted[seq] = row - a;
    p.token[seq] = token;
  }
}

template <typename E>
static int launch_verify(const VerifyArgs& p, cudaStream_t s) {
  const dim3 grid((unsigned)p.N, p.q ? 2 : 1);
  // few rows: many threads for each, so that all of a row is on its way at once
  const unsigned threads = (long long)p.N * grid.y <= 296 ? 1024 : 256;
  if (p.N) {
    if (p.T == 0.0) verify_stats_kernel<E, true><<<grid, threads, 0, s>>>(p);
    else verify_stats_kernel<E, false><<<grid, threads, 0, s>>>(p);
    BONES_CHECK(cudaGetLastError());
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  if (p.T == 0.0) {
    cfg.gridDim = dim3((unsigned)((p.B + 3) / 4));
    cfg.blockDim = dim3(128);
    return (int)cudaLaunchKernelEx(&cfg, verify_greedy_kernel, p);
  }
  cfg.gridDim = dim3(VC, (unsigned)p.B);
  cfg.blockDim = dim3(VT);
  return (int)cudaLaunchKernelEx(&cfg, verify_draw_kernel<E>, p);
}

}  // namespace bones

extern "C" {
using namespace bones;

// z, q (or null): rows of bf16 or (f32) fp32, ldz and ldq values apart; ids: int64 [N]; starts: int32 [B + 1]; u: fp32 [N, 2] (not read at T = 0);
// stats: room for 4 N doubles, of this call alone until it ends; accepted: int32 [B]; token: int64 [B].
int bones_verify(const void* z, long long ldz, const void* q, long long ldq, int f32, const long long* ids, const int* starts, const float* u, int B, int N, int V,
                 double T, double* stats, int* accepted, long long* token, void* stream) {
  if (!z || !ids || !starts || (!u && T != 0.0) || B < 1 || B > 65535 || N < 0 || V < 1 || !(T >= 0.0) || !stats || !accepted || !token || misaligned16(stats)) return -2;
  if (N && ((N > 1 && (ldz < V || (q && ldq < V))))) return -2;
  const VerifyArgs p{z, T == 0.0 ? nullptr : q, ldz, ldq, ids, starts, u, B, N, V, T, (RowStat*)stats, accepted, token};
  return f32 ? launch_verify<float>(p, (cudaStream_t)stream) : launch_verify<__nv_bfloat16>(p, (cudaStream_t)stream);
}
}  // extern "C"
