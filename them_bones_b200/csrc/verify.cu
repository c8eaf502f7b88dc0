// Verification of drafted tokens.
//
// Row r says p = softmax(z_r / T) of the token behind it, and the draft x there was drawn from q (the draft rows' soft-max, or certainty).  It stands
// while u_r0 q(x) < p(x); at the first that does not, the token is drawn from max(p - q, 0), behind the last draft from p, by the inverse
// distribution function at u_r1.  T = 0: the arg-max throughout.
//
// Two kernels.  The first reads every row once and leaves its maximum and its sum of exponentials.  The second, a cluster a sequence, goes
// through the sequence's drafts and draws the token from the one row that decides.  Its sums are in 64 bits: a border of the distribution
// function in 32 would move by more than the gap of a rare token's interval, and the token with it (65536 columns: one draw in some hundred).
// A draft whose test is closer than the first kernel's 32-bit exponentials and sums can tell is decided on sums in 64 bits too.
//
// Measured, us of a whole call: 64 sequences of a token and three drafts each, 65536 bf16 columns, drafts from a model, 39.6; one sequence of seven looked-up drafts, 8191 fp32
// columns, 8.9; with arg-max throughout 11.2 and 4.2.  By itself the first kernel takes 17.5 in the first case (59 MB at the copy rate: 9.0), the second 30, part of it beside the
// first's end.  The first is held up by neither memory (0.5 of that rate) nor its 29.4 million exponentials alone (12400 of 23500 clocks at 16 a clock and SM): 448
// rows are three an SM and four on some, the exponentials' pipe is active 0.62 of the time on the mean and 0.81 on the fullest SM, and a thread asks for its next four loads when
// it is done with the last.  The second: 8.4 million exponentials in 64 bits, at most seven operations each with the table's reads between them, by warps
// that wait for one another's results (the pipe of 64 bits 0.17, the schedulers 0.37 of the time).  Twice the warps with half the columns each: 55 us, and with four values
// side by side instead of eight 58 to 61 (of 38.2 then; the nearest column, tracked beside the sums, is 1.3 of the 39.6).
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
  float close;                   // how near to its border, of both sides' sum, a draft is not decided on the first kernel's sums
  double T, inv, steps, reach;   // 1 / T, K / T, 2^30 T / K
  RowStat* stats;              // [N, 2]
  int* accepted;
  long long* token;
};
static_assert(sizeof(VerifyArgs) == 128, "eight bytes more cost 1.5 us in the first case and 0.4 in the second");

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
// 16 bytes past the first-level cache, in the order of the program: left to itself the compiler waits for each load to save registers
__device__ __forceinline__ uint4 load_ahead(const void* p) {
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
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

// A CTA a row.  us of the whole call for 64 sequences, 448 rows of 65536 columns, with 256 / 512 / 1024 threads: 49.7 / 38.5 / 48.8; rows cut into four parts of 256 threads
// each 41.9; two values an instruction the same.
constexpr int VST = 512;
template <typename E, bool GREEDY>
__global__ void __launch_bounds__(VST, 4) verify_stats_kernel(const VerifyArgs p) {
  const int row = blockIdx.x, model = blockIdx.y;
  pdl_wait();
  pdl_launch();
  const int seq = paged_owner(p.starts, p.B, row);
  if (seq < 0 || seq >= p.B || (model && row + 1 >= p.starts[seq + 1])) return;      // no sequence's, or nothing was drawn from it
  const E* z = model ? (const E*)p.q + row * p.ldq : (const E*)p.z + row * p.ldz;
  const float c = GREEDY ? 0.f : (float)(1.4426950408889634 * p.inv);
  RowRun r{GREEDY ? -__int_as_float(0x7f800000) : -3.402823466e38f, 0.f, -1, false};
  constexpr int W = kVec<E>;
  // single values up to the first 16-byte boundary, vectors, single values
  const int head = min(p.V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(E)), vecs = (p.V - head) / W, tail = head + vecs * W;
  if (threadIdx.x < head) {
    const float f = logit(z + threadIdx.x);
    row_step<GREEDY, 1>(r, &f, threadIdx.x, c);
  }
  constexpr int U = 4;                               // loads of a thread in flight
  int i = threadIdx.x;
  for (; i + (U - 1) * VST < vecs; i += U * VST) {
    uint4 raw[U];
#pragma unroll
    for (int j = 0; j < U; ++j) raw[j] = load_ahead(z + head + (long long)(i + j * VST) * W);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[W];
      load_vec(reinterpret_cast<const E*>(&raw[j]), f);
      row_step<GREEDY, W>(r, f, head + (i + j * VST) * W, c);
    }
  }
  for (; i < vecs; i += VST) {
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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = VST / 32;
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
constexpr int VC = 8, VT = 128, VW = VC * VT / 32;       // CTAs, threads of one, warps of a cluster
constexpr int VS = 8;                                    // steps of a warp at most
constexpr int PARTS = VS * 32 + 1;                       // a warp's parts: a lane's of a step, and its nearest column
static_assert(VW == 32, "a lane has a warp's sums");

// A row's law, exp((z - most) / T), in 64 bits, by a table of powers of two (the method of Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic", 1989): with K = 256 / ln 2, z K / T - S = 256 m + j + f, |f| <= 1/2, the law is 2^m 2^(j/256)
// (1 + a f + a^2 f^2 / 2 + a^3 f^3 / 6), a = ln 2 / 256, whose remainder is 1.4e-13 at most.  Seven operations in 64 bits, which run at half the rate of those in 32
// and take 25 clocks each:
//  - what is a multiple of all values does not matter (the row's largest comes out as 1 to 0.2 %), so S is most K / T to a whole number, and z K / T - S
//    needs no more than the two sums with it;
//  - a conversion to 64 bits runs at 16 a clock and SM, so it is made of the value's bits: the exponent's other bias, the fraction moved;
//  - the table has a column for each lane of a half-warp (with a common one their reads met in the same banks, 6 clocks a warp), and its high words are
//    short of j 2^12, so that adding n 2^12 for n = 256 m + j makes 2^m of them;
//  - a value far below the largest (-inf, masks) is first raised to where the whole number has 31 bits, and that to -256000: it counts as 2^-1000, below
//    kNothing, instead of 0.
constexpr int EXP_ROWS = 256, EXP_COLS = 16;
constexpr double kNothing = 1e-280;
constexpr double kMagic = 6755399441055744.0;                // 1.5 * 2^52: a sum's low word is the whole number
struct Law {
  double scale, offset;                                      // K / T, kMagic - S
  float least;
  const double* powers;                                      // at this lane's column
  // steps: K / T; reach: 2^30 steps
  __device__ __forceinline__ Law(float most, double steps, double reach, const double* powers_) : scale(steps), powers(powers_) {
    if (fabs((double)most) * steps > 0x1p49) {               // S stays below: there the next value of fp32 is 90000 T away from the largest, and any scale does
      scale = 0x1p49 / fabs((double)most);
      reach = 0x1p30 / scale;
    }
    offset = kMagic - rint((double)most * scale);
    least = (float)((double)most - reach);                   // -inf where that leaves fp32: from there -inf itself, as 2^128, is as near
  }
  // W values side by side: one value's chain would leave the pipe idle
  template <int W>
  __device__ __forceinline__ void of(const float* z, double* e) const {
    double f[W], q[W];
    int n[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t u = __float_as_uint(fmaxf(z[i], least));
      const double v = __hiloint2double((int)(((uint32_t)((int)u >> 3) & 0x8fffffffu) + (896u << 20)), (int)(u << 29));
      const double t = fma(v, scale, offset);
      n[i] = max(__double2loint(t), -1000 * EXP_ROWS);
      f[i] = fma(v, scale, offset - t);                      // offset - t = -(S + 256 m + j)
    }
#pragma unroll
    for (int i = 0; i < W; ++i) q[i] = fma(f[i], 0x1.c6b08d704a0bfp-29, 0x1.ebfbdff82c58ep-19);
#pragma unroll
    for (int i = 0; i < W; ++i) q[i] = fma(f[i], q[i], 0x1.62e42fefa39efp-9);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const double j = powers[(n[i] & (EXP_ROWS - 1)) * EXP_COLS], w = __hiloint2double(__double2hiint(j) + n[i] * 4096, __double2loint(j));
      e[i] = fma(w, f[i] * q[i], w);
    }
  }
  __device__ __forceinline__ double operator()(float z) const {
    double e;
    of<1>(&z, &e);
    return e;
  }
};
__device__ __forceinline__ void fill_powers(double* table) {
  for (int j = threadIdx.x; j < EXP_ROWS; j += blockDim.x) {
    const double x = exp2(j * (1.0 / EXP_ROWS)), y = __hiloint2double(__double2hiint(x) - j * 4096, __double2loint(x));
    for (int i = 0; i < EXP_COLS; ++i) table[j * EXP_COLS + (i + j) % EXP_COLS] = y;          // (all columns; threads in different banks)
  }
}

// Eight consecutive columns as they lie in memory
template <typename E>
struct Eight {
  uint4 v[sizeof(E) / 2];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(E) == 2) {
      const uint32_t pair = (&v[0].x)[i >> 1];
      return __uint_as_float(i & 1 ? pair & 0xffff0000u : pair << 16);
    } else {
      return __uint_as_float((&v[i >> 2].x)[i & 3]);
    }
  }
};
// Columns at .. at + 7; -inf behind the last
template <typename E>
__device__ __forceinline__ Eight<E> load8(const E* z, int at, int V) {
  Eight<E> f;
  if (((uintptr_t)(z + at) & 15) == 0 && at + 8 <= V) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) f.v[i] = reinterpret_cast<const uint4*>(z + at)[i];
  } else {
    uint32_t w[2 * sizeof(E)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = at + i < V;
      if constexpr (sizeof(E) == 2) {
        const uint32_t x = in ? reinterpret_cast<const unsigned short*>(z)[at + i] : 0xff80u;
        if (i & 1) w[i >> 1] |= x << 16;
        else w[i >> 1] = x;
      } else {
        w[i] = in ? reinterpret_cast<const uint32_t*>(z)[at + i] : 0xff800000u;
      }
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) f.v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  return f;
}

// A warp's columns: consecutive steps, of which each lane has 8 * wide consecutive columns
struct Cut {
  int from, to, wide;
  __device__ __forceinline__ int column(int step, int lane) const { return (step * 32 + lane) * wide * 8; }
};

// The sums of each warp to all: lane l gets those of warp l of the cluster.
struct Sums {
  double p, q;         // of the law's own terms
  double p_up, q_up;   // of those columns' where p is above q
};
struct Shared : Sums {
  int gap;             // the least of |p - ratio q| / p in the warp's columns, as what the high words differ by (with q)
};
__device__ __forceinline__ Shared share(const Sums& s, Sums* box, const double2* parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) box[warp] = s;
  __syncthreads();
  cluster_barrier();
  const uint32_t at = map_to_rank(smem_u32(box + lane % (VT / 32)), lane / (VT / 32));
  Shared r;
  double* v = &r.p;
#pragma unroll
  for (int i = 0; i < 4; ++i) asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v[i]) : "r"(at + 8 * i));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(r.gap) : "r"(map_to_rank(smem_u32(parts + (lane % (VT / 32) - warp) * PARTS + VS * 32), lane / (VT / 32))));
  __syncwarp();
  cluster_barrier();
  return r;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A warp's sums over its columns; p_up and q_up those of the columns where p's law is above `ratio` times q's (without q: p's but for column `without`), in
// `parts` also lane by lane for each step.  Not unrolled over columns: with four tiles' exponentials written out the kernel waited for its
// instructions more than for anything else.
template <typename E, bool BOTH>
__device__ __noinline__ Sums row_sums(const E* z, const E* q, const Law lp, const Law lq, double ratio, int without, const Cut cut, int V, double2* parts) {
  const int lane = threadIdx.x & 31, n = (cut.to - cut.from) * cut.wide;
  Sums s = {};
  int gap = 0x7fffffff;
  if (n > 0) {
    int at = cut.column(cut.from, lane), k = 0;
    double up = 0.0, q_up = 0.0;
    Eight<E> f = load8(z, at, V), g;
    if (BOTH) g = load8(q, at, V);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      float u[8];
      double x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = f[j];
      const int here = at, next = k + 1 == cut.wide ? at + 8 + 31 * 8 * cut.wide : at + 8;
      if (i + 1 < n) f = load8(z, next, V);
      lp.of<8>(u, x);
      s.p += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      if (BOTH) {
        double y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = g[j];
        if (i + 1 < n) g = load8(q, next, V);
        lq.of<8>(u, y);
        s.q += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = __double2hiint(fma(-ratio, y[j], x[j]));
          const bool above = d > 0;                                                     // by the difference's sign
          gap = min(gap, (d & 0x7fffffff) - __double2hiint(x[j]));
          x[j] = __hiloint2double(above ? __double2hiint(x[j]) : 0, __double2loint(x[j]));        // (what is left without the high word is below 1e-310)
          y[j] = __hiloint2double(above ? __double2hiint(y[j]) : 0, __double2loint(y[j]));
        }
        q_up += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (here + j == without) x[j] = 0.0;
      }
      up += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      at = next;
      if (++k == cut.wide) {
        k = 0;
        parts[i / cut.wide * 32 + lane] = make_double2(up, q_up);
        s.p_up += up;
        s.q_up += q_up;
        up = q_up = 0.0;
      }
    }
  }
  s.p = warp_sum64(s.p);
  s.q = warp_sum64(s.q);
  s.p_up = warp_sum64(s.p_up);
  s.q_up = warp_sum64(s.q_up);
  if (BOTH) {
    gap = __reduce_min_sync(0xffffffffu, gap);
    if (lane == 0) *reinterpret_cast<int*>(parts + VS * 32) = gap;
  }
  return s;
}

// Whether p_up - ratio q_up is weight, and not what rounding leaves of columns where p and q are the same
__device__ __forceinline__ bool weighs(double w, double p_up) { return w > fmax(kNothing, 1e-12 * p_up); }

template <typename E>
__global__ void __cluster_dims__(VC, 1, 1) __launch_bounds__(VT, 4) verify_draw_kernel(const VerifyArgs p) {
  __shared__ Sums box[VT / 32];
  extern __shared__ __align__(16) double table[];                // the powers, and behind them the warps' parts
  double2* parts = reinterpret_cast<double2*>(table + EXP_ROWS * EXP_COLS) + (threadIdx.x >> 5) * PARTS;
  const double* powers = table + threadIdx.x % EXP_COLS;
  fill_powers(table);
  // What does not come from the first kernel is read before its end (it began behind all that came before): of the first 32 rows the draft behind each,
  // its logits and its number.
  const int seq = blockIdx.y, lane = threadIdx.x & 31, gw = (int)cluster_rank() * (VT / 32) + (threadIdx.x >> 5);
  const int a = min(max(p.starts[seq], 0), p.N), e = min(max(p.starts[seq + 1], a), p.N);
  const bool writer = cluster_rank() == 0 && threadIdx.x == 0;
  struct Draft {
    bool is;
    float p, q, u;
  };
  auto draft_behind = [&](int r) {
    Draft d{false, 0.f, 0.f, 0.f};
    if (r + 1 < e) {
      const long long x = p.ids[r + 1];
      d.is = x >= 0 && x < p.V;
      if (d.is) {
        d.p = logit((const E*)p.z + r * p.ldz + x);
        if (p.q) d.q = logit((const E*)p.q + r * p.ldq + x);
        d.u = p.u[2ll * r];
      }
    }
    return d;
  };
  Draft next = draft_behind(a + lane);
  pdl_wait();
  pdl_launch();
  __syncthreads();
  if (a == e) {
    if (writer) {
      p.accepted[seq] = 0;
      p.token[seq] = -1;
    }
    return;
  }
  // consecutive warps have consecutive columns; VS steps at most (one of 256 columns or more each)
  const int wide = (p.V + VW * VS * 256 - 1) / (VW * VS * 256), steps = (p.V + 256 * wide - 1) / (256 * wide), mine = (steps + VW - 1) / VW;
  const Cut cut{min(gw * mine, steps), min(gw * mine + mine, steps), wide};
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
      else if (next.is) {
        const RowStat sq = p.q ? p.stats[r * 2ll + 1] : RowStat{1.0, 0.f, 0};
        if (sq.sum > 0.0) {
          const double px = exp(((double)next.p - st.most) * p.inv) / st.sum, qx = p.q ? exp(((double)next.q - sq.most) * p.inv) / sq.sum : 1.0, need = next.u * qx;
          is = fabs(need - px) <= p.close * (need + px) ? CLOSE : need < px ? STANDS : FALLS;
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
        const Law lp(mp, p.steps, p.reach, powers), lq(mq, p.steps, p.reach, powers);
        const Shared both = share(p.q ? row_sums<E, true>(target(rr), draft(rr), lp, lq, 0.0, -1, cut, p.V, parts)
                                    : row_sums<E, false>(target(rr), nullptr, lp, lq, 0.0, -1, cut, p.V, parts), box, parts);
        const double sum_p = warp_sum64(both.p), sum_q = warp_sum64(both.q);
        const double px = exp(((double)logit(target(rr) + x) - mp) * p.inv) * lp(mp) / sum_p;
        const double qx = p.q ? exp(((double)logit(draft(rr) + x) - mq) * p.inv) * lq(mq) / sum_q : 1.0;
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
    next = draft_behind(r0 + 32 + lane);
  }
  row = min(row, e - 1);
  if (writer) p.accepted[seq] = row - a;
  if (why == GONE) {
    if (writer) p.token[seq] = -1;
    return;
  }
  // the row that decides: w = p, max(p - q, 0) or p without the draft
  const long long drafted = row + 1 < e ? p.ids[row + 1] : -1;
  const bool refused = drafted >= 0 && drafted < p.V;         // a draft outside the vocabulary was not drawn from q: what falls with it leaves all of p
  const RowStat st = p.stats[row * 2ll], sq = refused && p.q ? p.stats[row * 2ll + 1] : RowStat{0.0, 0.f, 0};
  const E *z = target(row), *zq = sq.sum > 0.0 ? draft(row) : nullptr;
  const Law lp(st.most, p.steps, p.reach, powers), lq(sq.most, p.steps, p.reach, powers);
  // One pass for both laws' sums and those of the columns where p is above q, with the first kernel's 32-bit sums for the ratio of the scales.  The ratio in
  // 64 bits follows, some 1e-7 of itself away.  Where p and q of some column are as near to each other as that, the first may have put it on the wrong side, and
  // the pass is made again; the weights' sums are with the ratio in 64 bits either way.
  const E* other = zq;
  double ratio = zq ? st.sum * lp(st.most) / (sq.sum * lq(sq.most)) : 0.0;
  int skip = refused && !p.q ? (int)drafted : -1;
  bool alone = !other && skip < 0;
  for (int round = 0; round < 3; ++round) {
    const Shared r = share(other ? row_sums<E, true>(z, other, lp, lq, ratio, -1, cut, p.V, parts)
                               : row_sums<E, false>(z, nullptr, lp, lq, 0.0, skip, cut, p.V, parts), box, parts);
    const double all_p = warp_sum64(r.p);
    if (other) {
      const double first = ratio;
      ratio = all_p / warp_sum64(r.q);
      // A column changes sides only where |p - first q| <= off q, so where |p - first q| / p is below twice off / first (off is 1e-8 of it, and with
      // 2^30 columns not half of it); another factor of two covers that high words tell either quotient to 6.2 %.  In 425 rows drawn as in the first case
      // above off was 4e-8 at most and no row went through twice.
      const double off = fabs(ratio - first);
      if (round == 0 && off > 0.0 && __reduce_min_sync(0xffffffffu, r.gap) <= __double2hiint(4.0 * off) - __double2hiint(first)) continue;
    }
    const double w = r.p_up - ratio * r.q_up;                 // of warp `lane`
    const bool some = __any_sync(0xffffffffu, weighs(w, r.p_up)), much = !other || warp_sum64(fmax(w, 0.0)) > 1e-12 * all_p;
    if (!(some && much) && !alone) {                          // p and q the same: of p alone.  (What is left of 1e-12 of p hangs on the last bits of its sums.)
      alone = true;
      other = nullptr;
      ratio = 0.0;
      skip = -1;
      continue;
    }
    auto up_to = [&](double x) {                              // sums up to and with each lane's
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      return x;
    };
    // the first with weight whose sum reaches above; by rounding there may be none: the last with weight
    auto pick = [&](bool heavy, double upto, double need) {
      const uint32_t has = __ballot_sync(0xffffffffu, heavy), above = __ballot_sync(0xffffffffu, heavy && upto > need);
      return above ? __ffs(above) - 1 : has ? 31 - __clz(has) : -1;
    };
    const double up = up_to(w), need = (double)p.u[2ll * row + 1] * __shfl_sync(0xffffffffu, up, 31);
    const int owner = pick(weighs(w, r.p_up), up, need);
    double before = __shfl_sync(0xffffffffu, up - w, max(owner, 0));
    if (owner == gw) {
      // its step (a lane a step), the lane in it, the column
      double mine_w = 0.0, mine_p = 0.0, lane_w = 0.0, lane_p = 0.0;
#pragma unroll
      for (int j = 0; j < VS; ++j) {
        if (cut.from + j >= cut.to) break;
        const double2 part = parts[j * 32 + lane];
        const double a_w = warp_sum64(part.x - ratio * part.y), a_p = warp_sum64(part.x);
        if (lane == j) {
          mine_w = a_w;
          mine_p = a_p;
        }
      }
      const double step_up = before + up_to(mine_w);
      const int step = max(pick(weighs(mine_w, mine_p), step_up, need), 0);
      before = __shfl_sync(0xffffffffu, step_up - mine_w, step);
      lane_p = parts[step * 32 + lane].x;
      lane_w = lane_p - ratio * parts[step * 32 + lane].y;
      const double lane_up = before + up_to(lane_w);
      const int from = max(pick(weighs(lane_w, lane_p), lane_up, need), 0);
      before = __shfl_sync(0xffffffffu, lane_up - lane_w, from);
      const int at = cut.column(cut.from + step, from);
      int found = -1, last = at;
      for (int k = 0; k < wide && found < 0; ++k) {
        const int col = at + k * 8 + lane;
        double x = 0.0, y = 0.0;
        if (lane < 8 && col < p.V) {
          x = lp(logit(z + col));
          if (other) y = lq(logit(other + col));
        }
        const double weight = col == skip ? 0.0 : fmax(x - ratio * y, 0.0), upto = before + up_to(weight);
        const bool heavy = weighs(weight, x);
        const uint32_t has = __ballot_sync(0xffffffffu, heavy), above = __ballot_sync(0xffffffffu, heavy && upto > need);
        if (has) last = at + k * 8 + 31 - __clz(has);
        if (above) found = at + k * 8 + __ffs(above) - 1;
        before = __shfl_sync(0xffffffffu, upto, 31);
      }
      if (lane == 0) p.token[seq] = min(found >= 0 ? found : last, p.V - 1);
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

// What the first kernel's sums may be off by.  A thread adds V / (512 W) times; each time the sum is rounded, and where a larger value came by scaled by an exponential
// (2^-22 of itself) and rounded: 6 * 2^-24 in all, of the target's and of the draft's sum, each over twice what it is compared with.  What does not grow with
// the columns (the exponentials of the values themselves, the threads' together) is some 1e-5, and 1e-4 covers it.  65536 bf16 columns: 1.07e-4; 2^27 of fp32: 0.026.
template <typename E>
static float too_close(int V) {
  return 1e-4f + (V / (VST * kVec<E>) + 2) * (6.0f * 0x1p-24f);
}

template <typename E>
static int launch_verify(VerifyArgs p, cudaStream_t s) {
  p.close = too_close<E>(p.V);
  const dim3 grid((unsigned)p.N, p.q ? 2 : 1);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)dec_launch_attrs(at, 1, 1);
  if (p.N) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(VST);
    BONES_CHECK(p.T == 0.0 ? cudaLaunchKernelEx(&cfg, verify_stats_kernel<E, true>, p) : cudaLaunchKernelEx(&cfg, verify_stats_kernel<E, false>, p));
  } else {
    cfg.numAttrs = 0;                            // without a first kernel, what comes before is not what the second may begin beside
  }
  if (p.T == 0.0) {
    cfg.gridDim = dim3((unsigned)((p.B + 3) / 4));
    cfg.blockDim = dim3(128);
    return (int)cudaLaunchKernelEx(&cfg, verify_greedy_kernel, p);
  }
  constexpr size_t smem = (EXP_ROWS * EXP_COLS + VT / 32 * PARTS * 2) * sizeof(double);
  static OncePerDevice limit;
  BONES_ONCE(limit, {
    BONES_CHECK(cudaFuncSetAttribute(verify_draw_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  });
  cfg.gridDim = dim3(VC, (unsigned)p.B);
  cfg.blockDim = dim3(VT);
  cfg.dynamicSmemBytes = smem;
  return (int)cudaLaunchKernelEx(&cfg, verify_draw_kernel<E>, p);
}

}  // namespace bones

extern "C" {
using namespace bones;

// z, q (or null): rows of bf16 or (f32) fp32, ldz and ldq values apart; ids: int64 [N]; starts: int32 [B + 1]; u: fp32 [N, 2] (not read at T = 0);
// stats: room for 4 N doubles, of this call alone until it ends; accepted: int32 [B]; token: int64 [B].
int bones_verify(const void* z, long long ldz, const void* q, long long ldq, int f32, const long long* ids, const int* starts, const float* u, int B, int N, int V,
                 double T, double* stats, int* accepted, long long* token, void* stream) {
  if ((N && (!z || !ids || (!u && T != 0.0))) || !starts || B < 1 || B > 65535 || N < 0 || V < 1 || !(T >= 0.0) || !stats || !accepted || !token || misaligned16(stats)) return -2;
  if (N && ((N > 1 && (ldz < V || (q && ldq < V))))) return -2;
  const double inv = T == 0.0 ? 0.0 : 1.0 / T, steps = 0x1.71547652b82fep+8 * inv;
  const VerifyArgs p{z, T == 0.0 ? nullptr : q, ldz, ldq, ids, starts, u, B, N, V, 0.f, T, inv, steps, 0x1p30 / steps, (RowStat*)stats, accepted, token};
  return f32 ? launch_verify<float>(p, (cudaStream_t)stream) : launch_verify<__nv_bfloat16>(p, (cudaStream_t)stream);
}
}  // extern "C"
