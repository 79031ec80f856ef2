// Learning from feedback on label paths: log-probabilities of paths, the preference loss and the clipped policy loss, forward and backward.
//
// A classifier's logits row z [C] is cut into L levels (network/loss.py:29-38 slices it the same way); each level has a softmax of its own.  A PATH is one class
// per level, -1 where it is not known; G paths may share a row (two answers of an annotator, the samples of a policy).
//   lse_l       = m_l + log sum_i exp(z_i - m_l)                       i over level l
//   logp[r,g,l] = z[r, start_l + y] - lse_l                             (0 where y < 0; NaN where y is no class of the level: nothing is read there)
//   dz[r,i]     = sum_g c[r,g,l] [y_g = i]  -  (sum_g c[r,g,l]) softmax_l(z)_i       c = d loss / d logp
// Both losses are functions of logp, so one pair of passes over the logits serves all three: `path_stats` (read z once) and `path_grad` (read z, write dz); between
// them a small kernel per loss works on [R, G, L] numbers in 64 bits and leaves c.
//
// What bounds it: HBM, and at the small sizes the launches (2 forward -- 1 for the log-probabilities of a hierarchy whose levels are all one run --, 1 backward).  A WAVE owns
// a run of at most 64 * NL 16-byte vectors of one level of one row, all loaded before the first use, so a level of 39 078 classes spreads over 16 waves and a row of 723 over 4,
// with no barrier and no LDS; (max, sum) of each run goes to `partials`, and whoever needs a level's lse merges its few runs again in the same order (the saved state of the
// backward pass IS `partials`).  Vectors start at the level's first class, which no alignment is promised for: the loads are 16 bytes wide at element alignment.
// Measured (a copy of 1 GiB on the same card moves 5.1 TB/s):
//   4 096 rows x 50 000 classes, bf16:   path_stats 85 us = 4.8 TB/s;  path_grad 160 us = 5.1 TB/s;  policy, 16 paths a row: 25 us (40 where an entry of the
//     largest level has to be summed again)
//   2 048 x 50 000, fp32, two paths a row: path_stats 83 us (114 behind a pass that left 410 MB of gradient to be written back);  preference 9 us;  path_grad 71 us = 5.8 TB/s
//     (written only: see there).  A row a path, and policy with 8 paths a row: path_grad reads too, 123 us = 6.6 TB/s (the end of the statistics pass's reading is still in
//     the caches); policy 12 us
//   256 x 723, fp32:                     4.6 | 6 | 6 us
// Bypassing the caches with the gradient's stores moved its write-back from the next pass into this one and gained nothing; so did walking the rows backwards in one of the
// two passes.
#include "lec_common.h"
#include "conv_geo.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <algorithm>
#include <cmath>

namespace lec {

constexpr int kMaxLevels = 16;
constexpr int kMaxClasses = 1 << 30;                             // an element's index within its level, padded to whole waves of vectors, stays within 31 bits
constexpr float kLog2e = 1.44269504088896340736f;

struct PathTable {
  int L, S, G;
  int start[kMaxLevels + 1];     // first class of a level
  int first[kMaxLevels + 1];     // first run of a level
  int vpr[kMaxLevels];           // 16-byte vectors of a run
  FastDiv byS, byG;              // task / S, path / G where the tasks, the paths fit 31 bits
};
__device__ __forceinline__ int64_t row_of(const PathTable& t, int64_t task, int64_t ntask) { return ntask <= INT32_MAX ? (int64_t)fdiv((int)task, t.byS) : task / t.S; }

template <typename T> struct Elt;
template <> struct Elt<float> {
  static constexpr int V = 4, NL = 9;
  static __device__ __forceinline__ float get(const uint4& w, int e) { return __uint_as_float(e == 0 ? w.x : e == 1 ? w.y : e == 2 ? w.z : w.w); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ void put(uint4& w, int e, const float* p) { (e == 0 ? w.x : e == 1 ? w.y : e == 2 ? w.z : w.w) = __float_as_uint(*p); }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) { return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])); }
  static __device__ __forceinline__ float cvt(float f) { return f; }
};
__device__ __forceinline__ void put_half(uint4& w, int e, unsigned short h) {
  unsigned int& u = (e >> 1) == 0 ? w.x : (e >> 1) == 1 ? w.y : (e >> 1) == 2 ? w.z : w.w;
  u = (e & 1) ? (u & 0xffffu) | ((unsigned int)h << 16) : (u & 0xffff0000u) | h;
}
__device__ __forceinline__ unsigned int word_of(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
template <> struct Elt<__hip_bfloat16> {
  static constexpr int V = 8, NL = 5;
  static __device__ __forceinline__ float get(const uint4& w, int e) { const unsigned int u = word_of(w, e >> 1); return __uint_as_float((e & 1) ? (u & 0xffff0000u) : (u << 16)); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ void put(uint4& w, int e, const __hip_bfloat16* p) { put_half(w, e, *(const unsigned short*)p); }
  static __device__ __forceinline__ float load(const __hip_bfloat16* p) { return __uint_as_float((unsigned int)*(const unsigned short*)p << 16); }
  static __device__ __forceinline__ __hip_bfloat16 cvt(float f) { return __float2bfloat16(f); }        // nearest, ties to even; NaN stays NaN
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    unsigned int u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __hip_bfloat16 a = cvt(f[2 * i]), b = cvt(f[2 * i + 1]);
      u[i] = (unsigned int)*(const unsigned short*)&a | ((unsigned int)*(const unsigned short*)&b << 16);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <> struct Elt<_Float16> {
  static constexpr int V = 8, NL = 5;
  static __device__ __forceinline__ float get(const uint4& w, int e) {
    const unsigned int u = word_of(w, e >> 1);
    const unsigned short h = (unsigned short)((e & 1) ? (u >> 16) : (u & 0xffffu));
    return (float)__builtin_bit_cast(_Float16, h);
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ void put(uint4& w, int e, const _Float16* p) { put_half(w, e, __builtin_bit_cast(unsigned short, *p)); }
  static __device__ __forceinline__ float load(const _Float16* p) { return (float)*p; }
  static __device__ __forceinline__ _Float16 cvt(float f) { return (_Float16)f; }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    unsigned int u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = (unsigned int)__builtin_bit_cast(unsigned short, cvt(f[2 * i])) | ((unsigned int)__builtin_bit_cast(unsigned short, cvt(f[2 * i + 1])) << 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// 16 bytes at element alignment (the compiler emits one dwordx4 access: the target's unaligned access mode)
template <typename T> __device__ __forceinline__ uint4 load16(const T* p) { uint4 w; __builtin_memcpy(&w, (const void*)p, 16); return w; }
template <typename T> __device__ __forceinline__ void store16(T* p, const uint4& w) { __builtin_memcpy((void*)p, &w, 16); }

// exp(t) for t <= 0 by the base-2 instruction: relative error below (3 |t| + 2) 2^-24
__device__ __forceinline__ float fast_exp(float t) { return __builtin_amdgcn_exp2f(t * kLog2e); }

// exp(x - m) for many x and one m, times a constant: one fma and one exponential an element.  x log2e - M, M = fl(m log2e), is exact but for its own rounding; what M lacks,
// r = m log2e - M (exact in one fma), is the same for all and goes into the constant: exp(x - m) = 2^(x log2e - M) 2^-r.  r is half a unit in the last place of M at most:
// below 2^-4 for |m| < 2^20; beyond that the difference is taken first.  m = -inf (nothing finite): every term is exp(-inf) = 0.
struct ExpAt {
  float m, M, unit;                                              // unit = 2^-r
  bool plain;
  __device__ __forceinline__ explicit ExpAt(float top) {
    m = top == -INFINITY ? 0.0f : top;
    plain = fabsf(m) < 1048576.0f;                               // (the same in all lanes: the branch below is scalar)
    M = m * kLog2e;
    unit = plain ? __builtin_amdgcn_exp2f(-__builtin_fmaf(m, kLog2e, -M)) : 1.0f;
  }
  template <bool PLAIN> __device__ __forceinline__ float at(float x) const {      // times unit
    return PLAIN ? __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, -M)) : fast_exp(x - m);
  }
};

// One run of a level of n elements at z: vectors v0 .. v0 + nv, one in 64 a lane, raw; -inf where there is none.
template <typename T, int NL = Elt<T>::NL>
struct Run {
  static constexpr int V = Elt<T>::V;
  uint4 w[NL];
  __device__ __forceinline__ void load(const T* z, int v0, int nv, int n, int lane) {
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int k = j * 64 + lane, e0 = (v0 + k) * V;
      w[j] = Elt<T>::none();
      if (k < nv && e0 + V <= n) w[j] = load16(z + e0);
    }
    const int last = n / V - v0;                                 // the level's last, incomplete vector, if it has one and it is this run's
    if (n % V && last < nv && (last & 63) == lane) {
#pragma unroll
      for (int j = 0; j < NL; ++j)
        if (j == last >> 6) {
#pragma unroll
          for (int e = 0; e < V - 1; ++e) if (e < n % V) Elt<T>::put(w[j], e, z + (v0 + last) * V + e);
        }
    }
  }
  __device__ __forceinline__ float get(int j, int e) const { return Elt<T>::get(w[j], e); }
};

__device__ __forceinline__ int level_of(const PathTable& t, int slot) {
  int l = 0;
  while (l + 1 < t.L && slot >= t.first[l + 1]) ++l;
  return l;
}

// LOGP: every level is one run, and the wave writes its entries' log-probabilities too.
template <typename T, bool LOGP>
__global__ __launch_bounds__(256) void path_stats_kernel(const T* __restrict__ z, int64_t ld, int64_t R, PathTable t, float2* __restrict__ partials, unsigned int* counters,
                                                         const int64_t* __restrict__ paths, float* __restrict__ logp) {
  const int lane = threadIdx.x & 63;
  if (counters && blockIdx.x == 0 && threadIdx.x <= 32) counters[threadIdx.x * 32] = 0;      // armed for the loss kernel behind this launch (grid_sum)
  const int64_t ntask = R * t.S, nwave = (int64_t)gridDim.x * 4;
  for (int64_t task = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); task < ntask; task += nwave) {
    const int64_t r = row_of(t, task, ntask);
    const int slot = (int)(task - r * t.S), l = level_of(t, slot), n = t.start[l + 1] - t.start[l];
    constexpr int V = Elt<T>::V, NL = Elt<T>::NL;
    const int v0 = (slot - t.first[l]) * t.vpr[l], nv = min(t.vpr[l], (n + V - 1) / V - v0);
    const T* zl = z + r * ld + t.start[l];
    const int64_t entry = (r * t.G + lane) * t.L + l;
    int64_t y = -1;
    if (LOGP && lane < t.G) y = paths[entry];
    Run<T> run;
    run.load(zl, v0, nv, n, lane);
    const float zy = LOGP && y >= 0 && y < n ? Elt<T>::load(zl + y) : __builtin_nanf("");
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NL; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) m = fmaxf(m, run.get(j, e));
    m = group_max<64>(m);
    const ExpAt ex(m);
    float s = 0.0f;
    auto sum = [&](auto plain) {
#pragma unroll
      for (int j = 0; j < NL; ++j)
        if (j * 64 < nv) {
#pragma unroll
          for (int e = 0; e < V; ++e) s += ex.template at<decltype(plain)::value>(run.get(j, e));
        }
    };
    if (ex.plain) sum(std::true_type{}); else sum(std::false_type{});
    s = group_sum<64>(s) * ex.unit;
    if (lane == 0) partials[task] = make_float2(m, s);
    if (LOGP && lane < t.G) logp[entry] = y < 0 ? 0.0f : (float)(((double)zy - (double)m) - log((double)s));
  }
}

// (max, sum) of a whole level from its n runs, eight at a time (their loads in flight together), in the order of the runs
__device__ __forceinline__ float2 merge_runs(const float2* __restrict__ p, int n) {
  float m = -INFINITY, s = 0.0f;
  for (int i = 0; i < n; i += 8) {
    float2 q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = p[min(i + j, n - 1)];
    float mq = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) mq = fmaxf(mq, q[j].x);
    s = m == mq ? s : s * fast_exp(m - mq);                                      // (m = -inf beside a finite mq: 0)
    m = mq;
#pragma unroll
    for (int j = 0; j < 8; ++j) if (i + j < n) s += q[j].x == m ? q[j].y : q[j].y * fast_exp(q[j].x - m);
  }
  return make_float2(m, s);
}
// The same by a wave: lane i takes run i (a level of more than 64 runs: the lane merges every 64th first)
__device__ __forceinline__ float2 merge_runs_wave(const float2* __restrict__ p, int n, int lane) {
  float m = -INFINITY, s = 0.0f;
  for (int i = lane; i < n; i += 64) {
    const float2 q = p[i];
    const float mq = fmaxf(m, q.x);
    s = (m == mq ? s : s * fast_exp(m - mq)) + (q.x == mq ? q.y : q.y * fast_exp(q.x - mq));
    m = mq;
  }
  const float mw = group_max<64>(m);
  return make_float2(mw, group_sum<64>(m == mw ? s : s * fast_exp(m - mw)));
}

// log-probability of class y of level l of row r in 64 bits: (z - m) - log s; NaN where the level has no such class
template <typename T>
__device__ __forceinline__ float named_logit(const T* __restrict__ z, int64_t ld, int64_t r, const PathTable& t, int l, int64_t y) {
  return y < t.start[l + 1] - t.start[l] ? Elt<T>::load(z + r * ld + t.start[l] + y) : __builtin_nanf("");
}
template <typename T>
__device__ __forceinline__ double entry_logp(const T* __restrict__ z, int64_t ld, int64_t r, const PathTable& t, int l, int64_t y, const float2* __restrict__ partials) {
  const float zy = named_logit(z, ld, r, t, l, y);
  const float2 ms = merge_runs(partials + r * t.S + t.first[l], t.first[l + 1] - t.first[l]);
  return ((double)zy - (double)ms.x) - log((double)ms.y);
}

template <typename T>
__global__ __launch_bounds__(256) void path_logp_kernel(const T* __restrict__ z, int64_t ld, int64_t n_entries, PathTable t, const int64_t* __restrict__ paths,
                                                        const float2* __restrict__ partials, float* __restrict__ logp) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_entries; i += (int64_t)gridDim.x * 256) {
    const int l = (int)(i % t.L);
    const int64_t r = i / ((int64_t)t.L * t.G), y = paths[i];
    logp[i] = y < 0 ? 0.0f : (float)entry_logp(z, ld, r, t, l, y, partials);
  }
}

// Sum of N doubles over the grid in a fixed order; true in one thread of the last block to arrive, `total` valid there.  `counters` were zeroed by the launch before.  All
// threads of the block call it (256 threads).  A block draws a ticket from one of 32 counters, a cache line each, and the last of each counter one from a 33rd: tickets of one
// word are drawn one after the other (up to 64 blocks share one).  The blocks' sums are handed over by agent-scope accesses alone, which act at the coherence point past the XCDs' L2s: a sum is
// there (vmcnt 0) before its block's ticket is drawn, and the last block asks for the sums after its own ticket has come back.  A release fence in every block would say the
// same and write the L2 back each time.  65 536 paths in 2 048 blocks: 57 us with the fence and one counter, 46 without the fence, 26 with 33 counters and all of the last
// block's threads at the sums.
constexpr unsigned int kTickets = 32;
template <int N>
__device__ __forceinline__ bool grid_sum(double (&v)[N] /* one value a thread */, double* __restrict__ block_sums, unsigned int* counters, double (&total)[N]) {
  __shared__ double s_w[4][N];
  __shared__ int s_last;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    for (int m = 32; m >= 1; m >>= 1) v[k] += __shfl_xor(v[k], m, 64);
    if (lane == 0) s_w[w][k] = v[k];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      __hip_atomic_store(&block_sums[(int64_t)blockIdx.x * N + k], s_w[0][k] + s_w[1][k] + s_w[2][k] + s_w[3][k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned int groups = gridDim.x <= 64 ? 1 : kTickets, g = blockIdx.x % groups, of_g = (gridDim.x - g + groups - 1) / groups;
    int last = __hip_atomic_fetch_add(counters + g * 32, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of_g - 1;
    if (last && groups > 1) last = __hip_atomic_fetch_add(counters + kTickets * 32, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
    s_last = last;
  }
  __syncthreads();
  if (!s_last) return false;
  double part[N];
#pragma unroll
  for (int k = 0; k < N; ++k) part[k] = 0.0;
  for (unsigned int i0 = 0; i0 < gridDim.x; i0 += 1024) {                        // four blocks' sums a thread, in flight together
    double q[4][N];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned int i = i0 + 256 * j + threadIdx.x;
#pragma unroll
      for (int k = 0; k < N; ++k) q[j][k] = i < gridDim.x ? __hip_atomic_load(&block_sums[(int64_t)i * N + k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < N; ++k) part[k] += q[j][k];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    for (int m = 32; m >= 1; m >>= 1) part[k] += __shfl_xor(part[k], m, 64);
    if (lane == 0) s_w[w][k] = part[k];                          // (s_w was read before the barrier above)
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) total[k] = s_w[0][k] + s_w[1][k] + s_w[2][k] + s_w[3][k];
  return threadIdx.x == 0;
}

// Preference loss.  Pair p: reward of a side = beta * sum_l (logp - ref), d = chosen - rejected,
//   loss = mean_p (1 - eps) softplus(-d) + eps softplus(d) ;  d loss / d d = (eps sigma(d) - (1 - eps) sigma(-d)) / P .
// A side is LW = the power of two >= L lanes (one a level), a pair 2 LW.  shared: both paths score row p; otherwise rows p and P + p.
template <typename T>
__global__ __launch_bounds__(256) void preference_kernel(const T* __restrict__ z, int64_t ld, int64_t P, int shared, int LW, PathTable t, const int64_t* __restrict__ paths,
                                                         const float* __restrict__ ref, float beta, float eps, const float2* __restrict__ partials, float* __restrict__ coef,
                                                         float* __restrict__ rewards, float* __restrict__ loss, double* __restrict__ block_sums, unsigned int* counters) {
  const int sh = 31 - __builtin_clz(LW), l = threadIdx.x & (LW - 1), side = (threadIdx.x >> sh) & 1, per_block = 128 >> sh;
  double acc[1] = {0.0};
  // every lane of a wave takes part in the shuffles: the loop bound is the block's, a lane past the last pair works on nothing
  for (int64_t p0 = (int64_t)blockIdx.x * per_block; p0 < P; p0 += (int64_t)gridDim.x * per_block) {
    const int64_t p = p0 + (threadIdx.x >> (sh + 1));
    const bool in = p < P && l < t.L;
    const int64_t row = shared ? p : side * P + p, entry = ((shared ? p * 2 + side : row)) * t.L + l;
    const int64_t y = in ? paths[entry] : -1;
    const double rf = in ? (double)ref[entry] : 0.0;
    double r = 0.0;
    if (y >= 0) r = entry_logp(z, ld, row, t, l, y, partials) - rf;
    for (int m = LW >> 1; m >= 1; m >>= 1) r += __shfl_xor(r, m, LW);
    r *= (double)beta;
    const double other = __shfl_xor(r, LW, 2 * LW), d = side ? other - r : r - other;
    const double e = exp(-fabs(d)), lp = log1p(e);                               // softplus(-d) = max(-d, 0) + log1p(exp(-|d|))
    const double sp = 1.0 / (1.0 + e), sm = e / (1.0 + e);                       // sigma(|d|), sigma(-|d|)
    const double sig = d >= 0.0 ? sp : (d < 0.0 ? sm : d), sigm = d >= 0.0 ? sm : (d < 0.0 ? sp : d);      // (NaN stays NaN)
    if (p < P && l == 0) rewards[p * 2 + side] = (float)r;
    if (p < P && l == 0 && side == 0)
      acc[0] += (1.0 - (double)eps) * ((d < 0.0 ? -d : d > 0.0 ? 0.0 : d * 0.0) + lp) + (eps != 0.0f ? (double)eps * ((d > 0.0 ? d : d < 0.0 ? 0.0 : d * 0.0) + lp) : 0.0);
    if (in) {
      const double g = ((double)eps * sig - (1.0 - (double)eps) * sigm) * (double)beta / (double)P;
      coef[entry] = y >= 0 ? (float)(side ? -g : g) : 0.0f;
    }
  }
  double total[1];
  if (grid_sum<1>(acc, block_sums, counters, total)) loss[0] = (float)(total[0] / (double)P);
}

// How far, relatively, a level's 32-bit sum may be off, in units of u = 2^-24.  n classes; a lane adds up to V ceil(vectors of a run / 64) of them, the wave its lanes, `lanes`
// lanes the runs.  A term exp(z - m): the difference, its product with log2 e and the constant, together 2.3 |z - m| over every frame it passes through, and the mean of m - z
// under the softmax is at most log n; 2 of the exponential, 3 of ExpAt's constant.  An addition: 1 (nothing where one side is 0).  A merge of two runs: 4 (the smaller side's
// exponential 2, its product, the addition).  4 for the products of these errors.  39 078 classes in 16 bits: 94 u.  Measured: 44 u where one class holds 92 % and 39 077 share
// the rest, each of them losing in the same direction.
static double sum_error(int n, int V, int vpr, int runs, int lanes) {
  const auto halvings = [](int k) { int h = 0; while ((1 << h) < k) ++h; return h; };
  const int adds = std::min(n, V * ((vpr + 63) / 64)) - 1 + halvings(std::min(vpr, 64)), merges = (runs + lanes - 1) / lanes - 1 + halvings(std::min(runs, lanes));
  return (2.3 * log((double)n) + 9.0 + adds + 4.0 * merges) * 0x1p-24;
}
struct SumErrors { double most; float of[kMaxLevels]; };         // of a row's levels

// Clipped policy loss.  Entry (r, g, l) counted: rho = exp(logp - old), A = advantage[r, g],
//   t = -min(rho A, clip(rho, 1 - lo, 1 + hi) A) + kl (exp(q) - q - 1),  q = ref - logp ;  dt/dlogp = -rho A [inside or on the bound] - kl expm1(q)
// loss = sum w t.  mean over counted entries: w = 1 / N, N known only at the end of this launch -- c is left without it and `norm` = 1 / max(N, 1) multiplies it in
// the backward pass; mean over paths: w = 1 / (entries of the path) / (R G), norm = 1.  stats = {sum w k3, sum w [clipped]}.
// The gradient jumps where rho passes the bound, and s is a sum of 32-bit exponentials: an entry whose rho lies within what that sum may be off by (sum_error) of the bound it
// may cross has its level summed again by the whole block in 64 bits before it is decided.  One sum serves all entries of that level of that row -- paths that name the same
// class with the same old log-probability are next to the bound together --, and every one of them is decided by it.  One entry in 165 000 of a level of 39 078 classes where
// log rho is spread over 0.1, and fewer of smaller levels: 14 us more for a launch that has one (4 096 rows x 16 paths x 50 000 classes, bf16).  Every entry at its bound, the
// most there can be: 390 us instead of 110 for statistics and loss at that size, 87 instead of 12 at 512 x 8 of 723 classes.  (Told that the loop's body is rare, the compiler
// keeps it out of the way: 0.3 us of a small launch.)
// A path is LW = the power of two >= L lanes of a wave.  The block's paths belong to a few consecutive rows: it first merges the runs of those rows' levels into LDS, as many
// lanes to a level as there are for it (a lane that merged its own level would wait for the level of the most runs, sixteen times over for sixteen paths of a row).
template <typename T>
__global__ __launch_bounds__(256, 4) void policy_kernel(const T* __restrict__ z, int64_t ld, int64_t n_paths, int LW, PathTable t, const int64_t* __restrict__ paths,
                                                     const float* __restrict__ adv, const float* __restrict__ old, const float* __restrict__ ref, SumErrors off, double lo, double hi,
                                                     float kl, int per_path, const float2* __restrict__ partials, float* __restrict__ coef, float* __restrict__ loss, float* __restrict__ stats,
                                                     float* __restrict__ norm, double* __restrict__ block_sums, unsigned int* counters) {
  constexpr int V = Elt<T>::V, kAgain = 4;                       // vectors a lane asks for together when a level is summed again
  __shared__ uint4 s_raw[256 * kAgain];                          // ... a thread's own place: the sum's loop over them is short, its 64-bit exponentials are not
  __shared__ int s_near[4];
  __shared__ double s_again[4];
  __shared__ double s_lse[256][2];                               // (m, log s) of the block's rows' levels: at most 256 (G = 1: one a lane; G > 1: half of that and two rows)
  const int sh = 31 - __builtin_clz(LW), l = threadIdx.x & (LW - 1), per_block = 256 >> sh;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t q0 = (int64_t)blockIdx.x * per_block; q0 < n_paths; q0 += (int64_t)gridDim.x * per_block) {
    const int64_t q = q0 + (threadIdx.x >> sh);
    const bool in = q < n_paths && l < t.L;
    const int64_t entry = q * t.L + l, y = in ? paths[entry] : -1;
    const auto row_at = [&](int64_t path) { return n_paths <= INT32_MAX ? (int64_t)fdiv((int)path, t.byG) : path / t.G; };
    const int64_t row = row_at(in ? q : q0), row0 = row_at(q0), row1 = row_at(min(q0 + per_block, n_paths) - 1);
    const bool on = y >= 0;
    double A = 0.0, lo_ = 0.0, lr_ = 0.0;
    float zy = 0.0f;
    if (on) {                                                    // asked for before the merge below
      A = (double)adv[q];
      if (old) lo_ = (double)old[entry];
      if (ref) lr_ = (double)ref[entry];
      zy = named_logit(z, ld, row, t, l, y);
    }
    const int units = (int)(row1 - row0 + 1) * t.L;
    int LP = 256;                                                // lanes to a unit
    while (LP > 64 || LP * units > 256) LP >>= 1;
    const int u = threadIdx.x / LP, ul = u % t.L, i0 = threadIdx.x & (LP - 1);
    float m = -INFINITY, s = 0.0f;
    if (u < units) {
      const float2* pr = partials + (row0 + u / t.L) * t.S + t.first[ul];
      const int n = t.first[ul + 1] - t.first[ul];
      for (int i = i0; i < n; i += LP) {
        const float2 v = pr[i];
        const float mv = fmaxf(m, v.x);
        s = (m == mv ? s : s * fast_exp(m - mv)) + (v.x == mv ? v.y : v.y * fast_exp(v.x - mv));
        m = mv;
      }
    }
    for (int w = LP >> 1; w >= 1; w >>= 1) {
      const float mo = __shfl_xor(m, w, 64), so = __shfl_xor(s, w, 64), mv = fmaxf(m, mo);
      const float own = m == mv ? s : s * fast_exp(m - mv), oth = mo == mv ? so : so * fast_exp(mo - mv);
      s = own + oth; m = mv;                                     // (a sum of two: the same in both lanes)
    }
    if (u < units && i0 == 0) { s_lse[u][0] = (double)m; s_lse[u][1] = log((double)s); }
    __syncthreads();
    const unsigned long long mask = __ballot(on) >> ((threadIdx.x & 63) & ~(LW - 1));
    const int cnt = __popcll(mask & ((1ull << LW) - 1ull));
    double lp = 0.0, rho = 1.0;                         // (no old log-probabilities: on-policy, the ratio is 1)
    bool near = false;
    const double bound = A > 0.0 ? 1.0 + hi : 1.0 - lo;
    const int k = (int)(row - row0) * t.L + l;
    if (on) {
      lp = ((double)zy - s_lse[k][0]) - s_lse[k][1];
      rho = exp(lp - (old ? lo_ : lp));
      near = old && A != 0.0 && fabs(rho - bound) < bound * off.most;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (;;) {                                                   // the undecided entries' levels, one after the other in their order in s_lse
      int next = 256;
      if (__builtin_expect(__ballot(near) != 0, 0)) {
        near = near && fabs(rho - bound) < bound * (double)off.of[l];
        next = near ? k : 256;
        for (int w = 32; w >= 1; w >>= 1) next = min(next, __shfl_xor(next, w, 64));
      }
      if (lane == 0) s_near[wave] = next;
      __syncthreads();                                           // (the last one: everybody has read s_lse, which the next round writes)
      next = min(min(s_near[0], s_near[1]), min(s_near[2], s_near[3]));
      if (__builtin_expect(next == 256, 1)) break;
      const int nl = next % t.L, n = t.start[nl + 1] - t.start[nl];
      const T* zl = z + (row0 + next / t.L) * ld + t.start[nl];
      const double top = s_lse[next][0];
      double sum = 0.0;
      const int nvec = (n + V - 1) / V;
      for (int v0 = wave * 64 * kAgain; v0 < nvec; v0 += 256 * kAgain) {
        const int nv = min(64 * kAgain, nvec - v0);
        Run<T, kAgain> run;
        run.load(zl, v0, nv, n, lane);
#pragma unroll
        for (int j = 0; j < kAgain; ++j) s_raw[j * 256 + threadIdx.x] = run.w[j];
#pragma unroll 1
        for (int j = 0; j * 64 < nv; ++j) {
          const uint4 w = s_raw[j * 256 + threadIdx.x];
#pragma unroll
          for (int e = 0; e < V; ++e) sum += exp((double)Elt<T>::get(w, e) - top);
        }
      }
      for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
      if (lane == 0) s_again[wave] = sum;
      __syncthreads();
      if (near && k == next) {
        lp = ((double)zy - top) - log(s_again[0] + s_again[1] + s_again[2] + s_again[3]);
        rho = exp(lp - lo_);
        near = false;
      }
    }
    float c = 0.0f;
    if (on) {
      const bool clipped = (A > 0.0 && rho > bound) || (A < 0.0 && rho < bound);
      const double gain = clipped ? bound * A : rho * A;
      double k3 = 0.0, dk = 0.0;
      if (ref) { const double d = lr_ - lp, em = expm1(d); k3 = em - d; dk = em; }
      const double w = per_path ? 1.0 / ((double)cnt * (double)n_paths) : 1.0;
      acc[0] += w * ((kl != 0.0f ? (double)kl * k3 : 0.0) - gain);
      acc[1] += w * k3;
      acc[2] += clipped ? w : 0.0;
      acc[3] += 1.0;
      c = (float)(w * ((clipped ? 0.0 : -rho * A) - (kl != 0.0f ? (double)kl * dk : 0.0)));
    }
    if (in) coef[entry] = c;
  }
  double total[4];
  if (grid_sum<4>(acc, block_sums, counters, total)) {
    const double inv = per_path ? 1.0 : 1.0 / (total[3] > 1.0 ? total[3] : 1.0);
    loss[0] = (float)(total[0] * inv); stats[0] = (float)(total[1] * inv); stats[1] = (float)(total[2] * inv); norm[0] = (float)inv;
  }
}

// dz of one run.  Lane g holds path g of the row (G <= 64): its class y, its coefficient c.  A = sum of the counted c; the softmax part is -A exp(z - m) / s.
// A == 0 (nothing counted, everything clipped, or the two sides of a preference on one row, whose coefficients are opposite): the part is zero and z is not read.
// The classes the paths name are written again, by the first lane that names them, with every path's coefficient added in lane order -- after the wave's own
// vector stores have been acknowledged (one wave writes the whole run, so no other wave is involved).
template <typename T>
__global__ __launch_bounds__(256) void path_grad_kernel(const T* __restrict__ z, int64_t ld, int64_t R, PathTable t, const int64_t* __restrict__ paths,
                                                        const float2* __restrict__ partials, const float* __restrict__ coef, const float* __restrict__ up,
                                                        const float* __restrict__ norm, T* __restrict__ dz, int64_t ldg) {
  const int lane = threadIdx.x & 63;
  const int64_t ntask = R * t.S, nwave = (int64_t)gridDim.x * 4;
  const float scale = (up ? *up : 1.0f) * (norm ? *norm : 1.0f);
  for (int64_t task = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); task < ntask; task += nwave) {
    constexpr int V = Elt<T>::V, NL = Elt<T>::NL;
    const int64_t r = row_of(t, task, ntask);
    const int slot = (int)(task - r * t.S), l = level_of(t, slot), n = t.start[l + 1] - t.start[l];
    const int v0 = (slot - t.first[l]) * t.vpr[l], nv = min(t.vpr[l], (n + V - 1) / V - v0);
    const T* zl = z + r * ld + t.start[l];
    T* gl = dz + r * ldg + t.start[l];
    int64_t y = -1;
    float c = 0.0f;
    if (lane < t.G) {
      const int64_t e = (r * t.G + lane) * t.L + l;
      y = paths[e];
      const float ce = coef[e];
      if (y < 0) y = -1;
      else c = y < n ? ce * scale : __builtin_nanf("");
    }
    const float A = group_sum<64>(c);
    const bool live = A != 0.0f;                                                  // (true for NaN)
    float2 ms = make_float2(0.0f, 1.0f);
    Run<T> run;
    if (live) {
      run.load(zl, v0, nv, n, lane);
      ms = merge_runs_wave(partials + r * t.S + t.first[l], t.first[l + 1] - t.first[l], lane);
    }
    const ExpAt ex(ms.x);
    const float k = -A / ms.y * ex.unit;
    const bool mine = y >= (int64_t)v0 * V && y < (int64_t)(v0 + nv) * V && y < n;
    const bool named = __ballot(mine) != 0;                                       // a path names a class of this run
    float zy = 0.0f;
    if (live && mine) zy = Elt<T>::load(zl + y);
    auto write = [&](auto value) {
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int i = j * 64 + lane, e0 = (v0 + i) * V;
        if (j * 64 >= nv) break;
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = value(j, e);
        if (i < nv) {
          if (e0 + V <= n) store16(gl + e0, Elt<T>::pack(f));
          else {
#pragma unroll
            for (int e = 0; e < V; ++e) if (e0 + e < n) gl[e0 + e] = Elt<T>::cvt(f[e]);
          }
        }
      }
    };
    if (!live) write([&](int, int) { return 0.0f; });
    else if (ex.plain) write([&](int j, int e) { return k * ex.template at<true>(run.get(j, e)); });
    else write([&](int j, int e) { return k * ex.template at<false>(run.get(j, e)); });
    if (named) {
      float tot = 0.0f;
      bool leader = mine;
      for (int g = 0; g < t.G; ++g) {
        const int yg = __builtin_amdgcn_readlane((int)(y > n ? n : y), g);
        const float cg = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(c), g));
        if (yg == (int)y) { tot += cg; if (g < lane) leader = false; }
      }
      const float soft = !live ? 0.0f : k * (ex.plain ? ex.template at<true>(zy) : ex.template at<false>(zy));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                            // the vector stores above are in the cache before the same bytes are written again
      if (leader) gl[y] = Elt<T>::cvt(tot + soft);
    }
  }
}

static int build_table(PathTable& t, const int32_t* sizes, int L, int C, int G, int V, int NL) {
  t.L = L; t.G = G; t.start[0] = 0; t.first[0] = 0;
  int64_t s = 0;
  for (int l = 0; l < L; ++l) {
    if (sizes[l] <= 0) { set_error("path loss: empty level %d", l); return LEC_E_ARG; }
    s += sizes[l];
    if (s > C) break;
    const int64_t nvec = ((int64_t)sizes[l] + V - 1) / V, cap = (int64_t)64 * NL, np = (nvec + cap - 1) / cap;
    t.vpr[l] = (int)((nvec + np - 1) / np);
    t.start[l + 1] = (int)s;
    t.first[l + 1] = t.first[l] + (int)((nvec + t.vpr[l] - 1) / t.vpr[l]);
  }
  if (s != C) { set_error("path loss: level sizes sum to %lld or more, expected C=%d", (long long)s, C); return LEC_E_ARG; }
  t.S = t.first[L];
  t.byS = make_fastdiv(t.S); t.byG = make_fastdiv(G);
  return LEC_OK;
}

static int64_t wave_grid(int64_t waves) { const int64_t b = (waves + 3) / 4; return b > (1 << 22) ? (1 << 22) : b; }
constexpr int64_t kMaxSumBlocks = 2048;

// workspace: the arrival counters, 33 lines of 128 bytes | block sums (2048 x 4 doubles)
constexpr int64_t kCounterBytes = 33 * 128, kWorkBytes = kCounterBytes + kMaxSumBlocks * 4 * 8;

static bool aligned8(const void* a, const void* b = nullptr) { return (((uintptr_t)a | (uintptr_t)b) & 7) == 0; }       // partials: pairs of floats; workspace: atomic doubles

template <typename F> static int by_type(int dtype, F&& f) {
  switch (dtype) {
    case LEC_DTYPE_F32: f((const float*)nullptr); return LEC_OK;
    case LEC_DTYPE_BF16: f((const __hip_bfloat16*)nullptr); return LEC_OK;
    case LEC_DTYPE_F16: f((const _Float16*)nullptr); return LEC_OK;
  }
  set_error("path loss: unknown dtype %d", dtype);
  return LEC_E_ARG;
}

static int table_for(PathTable& t, int dtype, int64_t R, int C, const int32_t* sizes, int L, int G) {
  LEC_CHECK_ARG(dtype == LEC_DTYPE_F32 || dtype == LEC_DTYPE_BF16 || dtype == LEC_DTYPE_F16, "path loss: unknown dtype %d", dtype);
  LEC_CHECK_ARG(sizes && L > 0 && L <= kMaxLevels && C > 0 && C <= kMaxClasses, "path loss: bad levels L=%d (1..%d) C=%d (1..%d)", L, kMaxLevels, C, kMaxClasses);
  LEC_CHECK_ARG(R >= 0 && R <= (int64_t)1 << 31 && G > 0 && G <= 64, "path loss: bad sizes rows=%lld paths per row=%d (1..64)", (long long)R, G);
  return dtype == LEC_DTYPE_F32 ? build_table(t, sizes, L, C, G, Elt<float>::V, Elt<float>::NL) : build_table(t, sizes, L, C, G, Elt<_Float16>::V, Elt<_Float16>::NL);
}

static int run_stats(const void* z, int dtype, int64_t ld, int64_t R, const PathTable& t, float2* partials, unsigned int* counters, hipStream_t st, const int64_t* paths = nullptr,
                     float* logp = nullptr) {
  const int rc = by_type(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const auto kernel = logp ? path_stats_kernel<T, true> : path_stats_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)wave_grid(R * t.S)), dim3(256), 0, st, (const T*)z, ld, R, t, partials, counters, paths, logp);
  });
  if (rc != LEC_OK) return rc;
  LEC_CHECK_LAUNCH("path_stats_kernel");
  return LEC_OK;
}

}  // namespace lec

extern "C" int64_t lec_path_partials_bytes(int dtype, int64_t R, int C, const int32_t* level_sizes, int L) {
  using namespace lec;
  PathTable t;
  const int rc = table_for(t, dtype, R, C, level_sizes, L, 1);
  return rc != LEC_OK ? rc : R * t.S * (int64_t)sizeof(float2);
}

extern "C" int64_t lec_path_workspace_bytes(void) { return lec::kWorkBytes; }

extern "C" int lec_path_logp_fwd(const void* logits, int dtype, int64_t ld, int64_t R, int C, const int32_t* level_sizes, int L, const int64_t* paths, int G,
                                 float* logp, void* partials, lec_stream_t stream) {
  using namespace lec;
  PathTable t;
  const int rc = table_for(t, dtype, R, C, level_sizes, L, G);
  if (rc != LEC_OK) return rc;
  LEC_CHECK_ARG(R > 0 && logits && paths && logp && partials && ld >= C, "path_logp_fwd: null pointer or ld=%lld < C=%d or no rows", (long long)ld, C);
  LEC_CHECK_ARG(aligned8(partials), "path_logp_fwd: partials have to be 8-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const bool one_launch = t.S == t.L;                            // every level fits one wave's run: the wave that has its sum also has what its entries need
  const int rs = run_stats(logits, dtype, ld, R, t, (float2*)partials, nullptr, st, paths, one_launch ? logp : nullptr);
  if (rs != LEC_OK || one_launch) return rs;
  const int64_t n = R * G * L, blocks = (n + 255) / 256;
  by_type(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    hipLaunchKernelGGL((path_logp_kernel<T>), dim3((unsigned)(blocks > (1 << 20) ? (1 << 20) : blocks)), dim3(256), 0, st, (const T*)logits, ld, n, t, paths, (const float2*)partials, logp);
  });
  LEC_CHECK_LAUNCH("path_logp_kernel");
  return LEC_OK;
}

extern "C" int lec_path_logp_bwd(const void* logits, int dtype, int64_t ld, int64_t R, int C, const int32_t* level_sizes, int L, const int64_t* paths, int G,
                                 const void* partials, const float* coef, const float* up, const float* norm, void* dlogits, int64_t ldg, lec_stream_t stream) {
  using namespace lec;
  PathTable t;
  const int rc = table_for(t, dtype, R, C, level_sizes, L, G);
  if (rc != LEC_OK) return rc;
  LEC_CHECK_ARG(R > 0 && logits && paths && partials && coef && dlogits && ld >= C && ldg >= C, "path_logp_bwd: null pointer or ld < C or no rows");
  LEC_CHECK_ARG(aligned8(partials), "path_logp_bwd: partials have to be 8-byte aligned");
  by_type(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    hipLaunchKernelGGL((path_grad_kernel<T>), dim3((unsigned)wave_grid(R * t.S)), dim3(256), 0, (hipStream_t)stream, (const T*)logits, ld, R, t, paths,
                       (const float2*)partials, coef, up, norm, (T*)dlogits, ldg);
  });
  LEC_CHECK_LAUNCH("path_grad_kernel");
  return LEC_OK;
}

extern "C" int lec_preference_loss_fwd(const void* logits, int dtype, int64_t ld, int64_t P, int shared, int C, const int32_t* level_sizes, int L, const int64_t* paths,
                                       const float* ref, float beta, float label_smoothing, float* loss, float* rewards, float* coef, void* partials, void* workspace,
                                       int64_t workspace_bytes, lec_stream_t stream) {
  using namespace lec;
  PathTable t;
  const int64_t R = shared ? P : 2 * P;
  const int rc = table_for(t, dtype, R, C, level_sizes, L, shared ? 2 : 1);
  if (rc != LEC_OK) return rc;
  LEC_CHECK_ARG(P > 0 && logits && paths && ref && loss && rewards && coef && partials && ld >= C, "preference_loss: null pointer or ld=%lld < C=%d or no pairs", (long long)ld, C);
  LEC_CHECK_ARG(workspace && workspace_bytes >= kWorkBytes, "preference_loss: workspace needs %lld bytes", (long long)kWorkBytes);
  LEC_CHECK_ARG(aligned8(partials, workspace), "preference_loss: partials and workspace have to be 8-byte aligned");
  LEC_CHECK_ARG(label_smoothing >= 0.0f && label_smoothing <= 1.0f, "preference_loss: label_smoothing %g is not in [0, 1]", (double)label_smoothing);
  hipStream_t st = (hipStream_t)stream;
  unsigned int* counters = (unsigned int*)workspace;
  const int rs = run_stats(logits, dtype, ld, R, t, (float2*)partials, counters, st);
  if (rs != LEC_OK) return rs;
  int LW = 1;
  while (LW < L) LW <<= 1;
  const int64_t per = 128 / LW, blocks = (P + per - 1) / per;
  by_type(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    hipLaunchKernelGGL((preference_kernel<T>), dim3((unsigned)(blocks > kMaxSumBlocks ? kMaxSumBlocks : blocks)), dim3(256), 0, st, (const T*)logits, ld, P, shared, LW, t, paths, ref,
                       beta, label_smoothing, (const float2*)partials, coef, rewards, loss, (double*)((char*)workspace + kCounterBytes), counters);
  });
  LEC_CHECK_LAUNCH("preference_kernel");
  return LEC_OK;
}

extern "C" int lec_policy_loss_fwd(const void* logits, int dtype, int64_t ld, int64_t R, int C, const int32_t* level_sizes, int L, const int64_t* paths, int G, const float* adv,
                                   const float* old_logp, const float* ref_logp, double clip_low, double clip_high, float kl_coef, int per_path, float* loss, float* stats, float* norm, float* coef,
                                   void* partials, void* workspace, int64_t workspace_bytes, lec_stream_t stream) {
  using namespace lec;
  PathTable t;
  const int rc = table_for(t, dtype, R, C, level_sizes, L, G);
  if (rc != LEC_OK) return rc;
  LEC_CHECK_ARG(R > 0 && logits && paths && adv && loss && stats && norm && coef && partials && ld >= C, "policy_loss: null pointer or ld=%lld < C=%d or no rows", (long long)ld, C);
  LEC_CHECK_ARG(workspace && workspace_bytes >= kWorkBytes, "policy_loss: workspace needs %lld bytes", (long long)kWorkBytes);
  LEC_CHECK_ARG(aligned8(partials, workspace), "policy_loss: partials and workspace have to be 8-byte aligned");
  LEC_CHECK_ARG(clip_low >= 0.0 && clip_high >= 0.0, "policy_loss: clip bounds %g, %g are negative", clip_low, clip_high);
  LEC_CHECK_ARG(kl_coef == 0.0f || ref_logp, "policy_loss: a KL coefficient needs the reference's log-probabilities");
  hipStream_t st = (hipStream_t)stream;
  unsigned int* counters = (unsigned int*)workspace;
  const int rs = run_stats(logits, dtype, ld, R, t, (float2*)partials, counters, st);
  if (rs != LEC_OK) return rs;
  int LW = 1;
  while (LW < L) LW <<= 1;
  const int64_t n = R * G, per = 256 / LW, blocks = (n + per - 1) / per;
  const int units = (int)std::min<int64_t>((per + G - 2) / G + 1, per) * L;           // levels of the rows that a block's paths belong to, and the lanes to each (policy_kernel)
  int lanes = 64;
  while (lanes * units > 256) lanes >>= 1;
  SumErrors off{};
  for (int l = 0; l < L; ++l) {
    const double e = sum_error(level_sizes[l], dtype == LEC_DTYPE_F32 ? Elt<float>::V : Elt<_Float16>::V, t.vpr[l], t.first[l + 1] - t.first[l], lanes);
    off.of[l] = std::nextafter((float)e, 1.0f); off.most = std::max(off.most, (double)off.of[l]);
  }
  by_type(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    hipLaunchKernelGGL((policy_kernel<T>), dim3((unsigned)(blocks > kMaxSumBlocks ? kMaxSumBlocks : blocks)), dim3(256), 0, st, (const T*)logits, ld, n, LW, t, paths, adv, old_logp,
                       ref_logp, off, clip_low, clip_high, kl_coef, per_path, (const float2*)partials, coef, loss, stats, norm, (double*)((char*)workspace + kCounterBytes), counters);
  });
  LEC_CHECK_LAUNCH("policy_kernel");
  return LEC_OK;
}
