// Microscaled 4-bit floating point: quantisation, its inverse, and the product of a classifier head held in it.
//
// Form (OCP microscaling, MXFP4): blocks of 32 elements along a row share a power of two X = 2^(clamp(floor(log2 max|v|) - 2, -127, 127)), kept as the byte
// log2 X + 127; an element is v / X rounded to nearest, ties to even, into {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign, saturating at 6.  A block that holds a NaN or an
// infinity has the byte 255 and stands for NaN.  17/32 bytes an element.
//
// Layout: the matrix instruction's own.  v_mfma_scale_f32_16x16x128_f8f6f4 takes from lane l the 32 codes (16 bytes) of row l % 16, elements 32 (l / 16) .. + 32 of a
// 128-element stretch, and one scale byte for them.  So a tile of 16 rows x 128 elements is 1 KB in lane order (codes[row tile][k tile][lane][16]): a wave's operand
// load is one contiguous 1 KB, from memory or from LDS, with no bank conflict and no shuffle.  The scale bytes of four consecutive k tiles sit in one 32-bit word a
// lane (scales[row tile][k tile / 4][lane][4]), which the instruction selects a byte of.  Rows are padded to 16 and elements to 128 with zeros.
#include "lec_common.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>

namespace lec {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t codes_bytes(int64_t rows, int64_t k) { return ceil_div(rows, 16) * ceil_div(k, 128) * 1024; }
static int64_t scales_bytes(int64_t rows, int64_t k) { return ceil_div(rows, 16) * ceil_div(k, 512) * 256; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __uint_as_float((unsigned int)*(const unsigned short*)&v << 16); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __hip_bfloat16 from_f32<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }

// 8 elements at x (n of them exist), one load of 16 or 32 bytes at element alignment
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ x, int n, float (&v)[8]) {
  if (n >= 8) {
    T raw[8];
    __builtin_memcpy(raw, (const void*)x, sizeof(raw));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(x[i]) : 0.0f;
  }
}

// Four neighbouring lanes hold a block, 8 elements each -> the lane's 8 codes and the block's scale byte.  The conversion instruction rounds to nearest even and
// saturates; it is given v / X (a product with a power of two, exact or far below the first threshold) and the scale 1, so that X = 2^-127 needs no special case.
__device__ __forceinline__ unsigned int quantize8(const float (&v)[8], unsigned int& scale) {
  int top = 0;                                                   // as integers: a NaN is above infinity, infinity above every number
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, (int)(__float_as_uint(v[i]) & 0x7fffffffu));
  top = max(top, __builtin_amdgcn_update_dpp(0, top, 0xB1, 0xf, 0xf, false));       // quad_perm: lane xor 1
  top = max(top, __builtin_amdgcn_update_dpp(0, top, 0x4E, 0xf, 0xf, false));       // lane xor 2
  const int e = top >> 23;                                       // floor(log2 max) = e - 127 (0 for subnormals, whose byte is clamped to 0 anyway)
  scale = e == 255 ? 255u : (unsigned int)max(e - 2, 0);
  const float inv = __uint_as_float(e == 255 ? 0u : (254u - scale) << 23);          // 1 / X
  unsigned int w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inv, v[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inv, v[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inv, v[5] * inv, 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inv, v[7] * inv, 1.0f, 3);
  return e == 255 ? 0u : w;
}

// A block takes a row tile and a group of four k tiles (16 rows x 512 elements, one scale word a lane of the layout); a wave reads 512 consecutive elements of a row at
// a time, 16 bytes a lane, so memory sees contiguous kilobytes; the codes of 16 rows meet in the L2.
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int K, int KT, int KG, int64_t ntask, unsigned int* __restrict__ codes,
                                                             unsigned int* __restrict__ scales) {
  __shared__ unsigned char s_scale[256];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int ktl = lane >> 4, kb = (lane >> 2) & 3, sub = lane & 3;
  for (int64_t task = blockIdx.x; task < ntask; task += gridDim.x) {
    const int64_t rt = task / KG;
    const int kg = (int)(task - rt * KG), k = kg * 512 + lane * 8, kt = kg * 4 + ktl;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = rt * 16 + wave * 4 + i;
      load8(x + row * ld + k, row < rows ? K - k : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = wave * 4 + i;
      unsigned int sc;
      const unsigned int w = quantize8(v[i], sc);
      if (kt < KT) codes[((rt * KT + kt) * 64 + kb * 16 + r) * 4 + sub] = w;
      if (sub == 0) s_scale[(kb * 16 + r) * 4 + ktl] = (unsigned char)sc;
    }
    __syncthreads();
    if (t < 64) scales[(rt * KG + kg) * 64 + t] = ((const unsigned int*)s_scale)[t];
    __syncthreads();                                             // (the next task writes s_scale)
  }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const unsigned int* __restrict__ codes, const unsigned char* __restrict__ scales, int64_t rows, int K, int KT, int KG,
                                                               int64_t ntask, T* __restrict__ out, int64_t ld) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int ktl = lane >> 4, kb = (lane >> 2) & 3, sub = lane & 3;
  for (int64_t task = blockIdx.x; task < ntask; task += gridDim.x) {
    const int64_t rt = task / KG;
    const int kg = (int)(task - rt * KG), k = kg * 512 + lane * 8, kt = kg * 4 + ktl;
    if (k >= K) continue;
    unsigned int w[4], sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = wave * 4 + i;                                // (rows past the end are padding of the same tile)
      w[i] = codes[((rt * KT + kt) * 64 + kb * 16 + r) * 4 + sub];
      sc[i] = scales[((rt * KG + kg) * 64 + kb * 16 + r) * 4 + ktl];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = rt * 16 + wave * 4 + i;
      if (row >= rows) continue;
      const float X = sc[i] == 255u ? __builtin_nanf("") : (sc[i] == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(sc[i] << 23));      // 2^(byte - 127); byte 0: subnormal
      T v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 f = j == 0 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 0) : j == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 1)
                      : j == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 2) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 3);
        v[2 * j] = from_f32<T>(f.x * X); v[2 * j + 1] = from_f32<T>(f.y * X);
      }
      T* o = out + row * ld + k;
      if (k + 8 <= K) __builtin_memcpy((void*)o, v, sizeof(v));
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (k + j < K) o[j] = v[j];
      }
    }
  }
}

__device__ __forceinline__ f32x4 mfma4(const uint4& a, const uint4& b, f32x4 c, int which, unsigned int sa, unsigned int sb) {
  i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  switch (which) {                                               // (the selected byte is part of the instruction)
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 1, (int)sa, 1, (int)sb);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 2, (int)sa, 2, (int)sb);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 3, (int)sa, 3, (int)sb);
  }
}

// y[m, n] = sum_k x[m, k] w[n, k] + bias[n].  The weights are the A operand: a lane's four accumulators are four consecutive classes n of one row m.
template <typename T>
__device__ __forceinline__ void store4(T* __restrict__ y, int64_t ldy, int64_t M, int N, int64_t m, int n, const f32x4& acc, const float (&bv)[4]) {
  if (m >= M || n >= N) return;
  T o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(acc[e] + bv[e]);
  T* p = y + m * ldy + n;
  if (n + 4 <= N) __builtin_memcpy((void*)p, o, sizeof(o));
  else {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (n + e < N) p[e] = o[e];
  }
}
__device__ __forceinline__ void load_bias(const float* __restrict__ bias, int N, int n, float (&bv)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) bv[e] = bias && n + e < N ? bias[n + e] : 0.0f;
}

// At most 16 rows (one tile of x): the time is the weights' way from memory.  A wave owns one tile of 16 classes and asks for 16 k tiles of its weights at once; while
// they are under way the block quantises x into LDS (each block again: x is small and comes from the L2, a launch of its own would cost more).  x has to fit 64 KB of LDS: K <= 7680.
template <typename TX, typename T>
__global__ __launch_bounds__(256) void mxfp4_linear_rows_kernel(const TX* __restrict__ x, int64_t ldx, int M, const uint4* __restrict__ wc, const unsigned int* __restrict__ wsc, int N, int K,
                                                                int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned int* xcodes = (unsigned int*)smem;                    // [KT][64][4] words
  unsigned char* xscale = smem + (size_t)KT * 1024;              // [KG][64][4] bytes
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int nt = min((int)blockIdx.x * 4 + wave, ((N + 15) >> 4) - 1);
  const bool mine = (int)blockIdx.x * 4 + wave == nt;            // (a wave past the last tile repeats it and stores nothing)
  constexpr int CH = 16;
  uint4 w[CH];
  unsigned int sw[CH / 4];
  auto fetch = [&](int kt0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) if (kt0 + i < KT) w[i] = wc[((int64_t)nt * KT + kt0 + i) * 64 + lane];
#pragma unroll
    for (int i = 0; i < CH / 4; ++i) if (kt0 / 4 + i < KG) sw[i] = wsc[((int64_t)nt * KG + kt0 / 4 + i) * 64 + lane];
  };
  fetch(0);
  for (int i = t; i < KT * 64; i += 256) ((uint4*)xcodes)[i] = make_uint4(0u, 0u, 0u, 0u);       // rows that do not exist
  for (int i = t; i < KG * 64; i += 256) ((unsigned int*)xscale)[i] = 0u;
  __syncthreads();
  const int per_row = KG * 64;                                   // 8-element pieces of a row, padded to whole groups of 512
  for (int i = t; i < M * per_row; i += 256) {
    const int r = i / per_row, q = i - r * per_row, k = q * 8, kt = k >> 7, kb = (k >> 5) & 3, sub = (k >> 3) & 3;
    float v[8];
    load8(x + (int64_t)r * ldx + k, K - k, v);
    unsigned int sc;
    const unsigned int c = quantize8(v, sc);
    if (kt < KT) xcodes[(kt * 64 + kb * 16 + r) * 4 + sub] = c;
    if (sub == 0) xscale[((kt >> 2) * 64 + kb * 16 + r) * 4 + (kt & 3)] = (unsigned char)sc;
  }
  __syncthreads();
  f32x4 acc[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};                // two chains: an MFMA need not wait for the one before
  for (int kt0 = 0; kt0 < KT; kt0 += CH) {
    if (kt0) fetch(kt0);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (kt0 + i < KT) {
        const uint4 b = ((const uint4*)xcodes)[(kt0 + i) * 64 + lane];
        const unsigned int sb = ((const unsigned int*)xscale)[((kt0 + i) >> 2) * 64 + lane];
        acc[i & 1] = mfma4(w[i], b, acc[i & 1], i & 3, sw[i >> 2], sb);
      }
    }
  }
  if (!mine) return;
  const int n = nt * 16 + 4 * (lane >> 4);
  float bv[4];
  load_bias(bias, N, n, bv);
  store4(y, ldy, M, N, lane & 15, n, acc[0] + acc[1], bv);
}

// A block of WN x WM waves, a wave NT x MT tiles, operands straight from memory (every load is a contiguous kilobyte): few tiles, or shapes too small for the ring below.
template <typename T, int WN, int WM, int NT, int MT>
__global__ __launch_bounds__(64 * WN * WM) void mxfp4_linear_small_kernel(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                                          const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y,
                                                                          int64_t ldy) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nt0 = ((int)blockIdx.x * WN + wave % WN) * NT, ntn = (N + 15) >> 4;
  const int64_t mt0 = ((int64_t)blockIdx.y * WM + wave / WN) * MT, mtn = (M + 15) >> 4;
  if (nt0 >= ntn || mt0 >= mtn) return;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kg = 0; kg < KG; ++kg) {
    unsigned int sa[NT], sb[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) sa[i] = wsc[((int64_t)min(nt0 + i, ntn - 1) * KG + kg) * 64 + lane];       // (tiles past the end repeat the last one; they are not stored)
#pragma unroll
    for (int j = 0; j < MT; ++j) sb[j] = xs[(min(mt0 + j, mtn - 1) * KG + kg) * 64 + lane];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int kt = kg * 4 + q;
      if (kt >= KT) break;
      uint4 a[NT], b[MT];
#pragma unroll
      for (int i = 0; i < NT; ++i) a[i] = wc[((int64_t)min(nt0 + i, ntn - 1) * KT + kt) * 64 + lane];
#pragma unroll
      for (int j = 0; j < MT; ++j) b[j] = xc[(min(mt0 + j, mtn - 1) * KT + kt) * 64 + lane];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma4(a[i], b[j], acc[i][j], q, sa[i], sb[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int n = (nt0 + i) * 16 + 4 * (lane >> 4);
    float bv[4];
    load_bias(bias, N, n, bv);
#pragma unroll
    for (int j = 0; j < MT; ++j) store4(y, ldy, M, N, (mt0 + j) * 16 + (lane & 15), n, acc[i][j], bv);
  }
}

// Large products.  A block of 2 x 2 waves owns 256 x 256 of y, a wave 128 x 128 (8 x 8 tiles, 256 accumulators: one wave a SIMD, one block a CU).  A k tile of both operands is
// 32 KB; a ring of four stages in LDS is filled by LDS-DMA (a wave's request is one contiguous kilobyte = one operand tile in lane order, so there is nothing to swizzle), three stages
// ahead.  Per k tile a wave issues 64 MFMAs of 16 cycles and reads 16 KB of LDS: 96 KB of LDS traffic per 1024 cycles a CU, under its 128 B / clk.
typedef __attribute__((address_space(3))) void lds_ptr;
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t make_rsrc(const void* p, unsigned bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00020000); }
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); __builtin_amdgcn_s_barrier(); asm volatile("" ::: "memory"); }

// (A body with restrict parameters, inlined into the kernel: its memory accesses then carry alias scopes, without which the compiler waits for every outstanding
// LDS-DMA before any read of LDS -- the ring would be one stage deep.)
template <typename T>
__device__ __forceinline__ void mxfp4_linear_big_body(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                                  const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy,
                                                                  int nbn, int nbm, int per_xcd) {
  constexpr int STAGE = 32 * 1024, IPW = 8;                      // bytes of a stage; LDS-DMA instructions a wave issues for one
  constexpr int PIN = (int)0x80000000;                           // a volatile load: it stays where it is written, ahead of the requests behind it
  constexpr int OOB = 0x40000000;                                // past any operand buffer (KT <= 32 768: at most 2^29 bytes)
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1;
  // consecutive blocks land on the eight XCDs in turn: give each XCD a contiguous run of tiles, four tiles of rows by all tiles of classes at a time, so that a run's
  // operands stay in its L2
  const int64_t g = (int64_t)((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (g >= (int64_t)nbn * nbm) return;
  const int band = (int)(g / (4 * (int64_t)nbn)), inb = (int)(g - (int64_t)band * 4 * nbn), bw = min(4, nbm - band * 4);
  const int bn = __builtin_amdgcn_readfirstlane(inb / bw), bm = __builtin_amdgcn_readfirstlane(band * 4 + inb % bw);      // (the division leaves them in vector registers)
  const int ntn = (N + 15) >> 4, mtn = (int)((M + 15) >> 4);
  // The block's operand tiles of each side and their scales as buffers that end with the last of them; a tile past the matrix repeats the last one (and is not stored).
  const int na_ = min(16, ntn - bn * 16), nb_ = min(16, mtn - bm * 16);
  const rsrc_t ra = make_rsrc(wc + (int64_t)bn * 16 * KT * 64, (unsigned)na_ * KT * 1024), rb = make_rsrc(xc + (int64_t)bm * 16 * KT * 64, (unsigned)nb_ * KT * 1024);
  const rsrc_t rsa = make_rsrc(wsc + (int64_t)bn * 16 * KG * 64, (unsigned)na_ * KG * 256), rsb = make_rsrc(xs + (int64_t)bm * 16 * KG * 64, (unsigned)nb_ * KG * 256);
  auto issue = [&](int kt) {                                     // this wave's tiles of stage kt: 4 of the weights, 4 of x.  Past the last stage: no traffic, zeros in LDS
    unsigned char* base = smem + (kt & 3) * STAGE + wave * 1024;
    const int voff = lane * 16 + (kt < KT ? 0 : OOB), kc = min(kt, KT - 1);
#pragma unroll
    for (int u = 0; u < 4; ++u) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr*)(base + u * 4096), 16, voff, (min(wave + 4 * u, na_ - 1) * KT + kc) * 1024, 0, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u) __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr*)(base + 16384 + u * 4096), 16, voff, (min(wave + 4 * u, nb_ - 1) * KT + kc) * 1024, 0, 0);
  };
  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  int sa[8], sb[8], na[8], nb[8];                                // scale words: of this group of four k tiles, of the next one
  auto fetch_scales = [&](int kg) {                              // (a group past the end: the last one again)
    const int kc = min(kg, KG - 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      na[i] = __builtin_amdgcn_raw_buffer_load_b32(rsa, lane * 4, (min(wn * 8 + i, na_ - 1) * KG + kc) * 256, PIN);
      nb[i] = __builtin_amdgcn_raw_buffer_load_b32(rsb, lane * 4, (min(wm * 8 + i, nb_ - 1) * KG + kc) * 256, PIN);
    }
  };
  const uint4* A = (const uint4*)smem + wn * 512 + lane;         // this wave's operand tiles of slot 0
  const uint4* B = (const uint4*)(smem + 16384) + wm * 512 + lane;
  fetch_scales(0);
  issue(0); issue(1); issue(2); issue(3);
  wait_vm<3 * IPW>();                                            // stage 0 has landed for this wave ...
  meet();                                                        // ... and for every wave
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sa[i] = na[i]; sb[i] = nb[i];
    asm volatile("" : "+v"(sa[i]), "+v"(sb[i]));                  // in registers before the loop: its own waits then count the loop's requests only
  }
  uint4 a = A[0], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = B[j * 64];
  // One k tile: rows 0 .. 3 of the products run while the wave reads its other weights of the stage; then everybody is done reading stage kt, whose slot takes stage kt + 4, and
  // stage kt + 1 has landed once at most the two younger stages' requests are outstanding (scale loads in between only make the wait stricter); rows 4 .. 7 run while
  // stage kt + 1's first operands are read.  The order is pinned: left alone the scheduler puts every read before the first product.  Groups of four k tiles, the last one
  // filled up with stages of zeros, so that the body has no branch.
  auto tile = [&](int kt, auto qc) {
    constexpr int q = decltype(qc)::value;
    const uint4* Ao = A + q * (STAGE / 16);
    const uint4* An = A + ((q + 1) & 3) * (STAGE / 16);
    const uint4* Bn = B + ((q + 1) & 3) * (STAGE / 16);
    uint4 ar[8], bx[8];
    ar[0] = a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ar[i + 1] = Ao[(i + 1) * 64];
      if (i > 0) ar[i + 4] = Ao[(i + 4) * 64];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = mfma4(ar[i], b[j], acc[i][j], q, sa[i], sb[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_vm<2 * IPW>();
    meet();
    if (q == 0) fetch_scales((kt >> 2) + 1);
    issue(kt + 4);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 4; i < 8; ++i) {
      if (i == 4) a = An[0];
      bx[2 * (i - 4)] = Bn[2 * (i - 4) * 64];
      bx[2 * (i - 4) + 1] = Bn[(2 * (i - 4) + 1) * 64];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = mfma4(ar[i], b[j], acc[i][j], q, sa[i], sb[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = bx[j];
  };
  for (int kt = 0; kt < KT; kt += 4) {
    tile(kt, std::integral_constant<int, 0>{});
    tile(kt + 1, std::integral_constant<int, 1>{});
    tile(kt + 2, std::integral_constant<int, 2>{});
    tile(kt + 3, std::integral_constant<int, 3>{});
#pragma unroll
    for (int i = 0; i < 8; ++i) { sa[i] = na[i]; sb[i] = nb[i]; }
  }
  wait_vm<0>();                                                  // (the stages of zeros past the end still write LDS)
  const rsrc_t rbias = make_rsrc(bias, bias ? (unsigned)N * 4u : 0u);
  const bool inside = (bn + 1) * 256 <= N && (int64_t)(bm + 1) * 256 <= M;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = (bn * 16 + wn * 8 + i) * 16 + 4 * (lane >> 4);
    float bv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bv[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rbias, (n + e) * 4, 0, 0));       // (past the end: 0)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t m = (int64_t)(bm * 16 + wm * 8 + j) * 16 + (lane & 15);
      if (inside) {
        T o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(acc[i][j][e] + bv[e]);
        __builtin_memcpy((void*)(y + m * ldy + n), o, sizeof(o));
      } else {
        store4(y, ldy, M, N, m, n, acc[i][j], bv);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256, 1) void mxfp4_linear_big_kernel(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                                  const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy,
                                                                  int nbn, int nbm, int per_xcd) {
  mxfp4_linear_big_body<T>(xc, xs, M, wc, wsc, N, KT, KG, bias, y, ldy, nbn, nbm, per_xcd);
}

template <typename F> static int by_dtype(int dtype, const char* what, F&& f) {
  switch (dtype) {
    case LEC_DTYPE_F32: f((float*)nullptr); return LEC_OK;
    case LEC_DTYPE_BF16: f((__hip_bfloat16*)nullptr); return LEC_OK;
    case LEC_DTYPE_F16: f((_Float16*)nullptr); return LEC_OK;
  }
  set_error("%s: unknown dtype %d", what, dtype);
  return LEC_E_ARG;
}
static unsigned grid_of(int64_t blocks) { return (unsigned)(blocks > (1 << 22) ? (1 << 22) : blocks); }

static int quantize(const void* x, int dtype, int64_t ld, int64_t rows, int K, void* codes, void* scales, hipStream_t st) {
  const int KT = (int)ceil_div(K, 128), KG = (int)ceil_div(K, 512);
  const int64_t ntask = ceil_div(rows, 16) * KG;
  const int rc = by_dtype(dtype, "mxfp4_quantize", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL((mxfp4_quantize_kernel<T>), dim3(grid_of(ntask)), dim3(256), 0, st, (const T*)x, ld, rows, K, KT, KG, ntask, (unsigned int*)codes, (unsigned int*)scales);
  });
  if (rc != LEC_OK) return rc;
  LEC_CHECK_LAUNCH("mxfp4_quantize_kernel");
  return LEC_OK;
}

}  // namespace lec

static bool sizes_ok(int64_t rows, int64_t k) { return rows > 0 && rows <= ((int64_t)1 << 31) - 16 && k > 0 && k <= (1 << 24); }

extern "C" int64_t lec_mxfp4_codes_bytes(int64_t rows, int64_t k) { return sizes_ok(rows, k) ? lec::codes_bytes(rows, k) : LEC_E_ARG; }
extern "C" int64_t lec_mxfp4_scales_bytes(int64_t rows, int64_t k) { return sizes_ok(rows, k) ? lec::scales_bytes(rows, k) : LEC_E_ARG; }

extern "C" int lec_mxfp4_quantize(const void* x, int dtype, int64_t ld, int64_t rows, int64_t k, void* codes, void* scales, lec_stream_t stream) {
  using namespace lec;
  LEC_CHECK_ARG(sizes_ok(rows, k), "mxfp4_quantize: bad sizes rows=%lld k=%lld", (long long)rows, (long long)k);
  LEC_CHECK_ARG(x && codes && scales && ld >= k, "mxfp4_quantize: null pointer or ld=%lld < k=%lld", (long long)ld, (long long)k);
  return quantize(x, dtype, ld, rows, (int)k, codes, scales, (hipStream_t)stream);
}

extern "C" int lec_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t k, void* out, int dtype, int64_t ld, lec_stream_t stream) {
  using namespace lec;
  LEC_CHECK_ARG(sizes_ok(rows, k), "mxfp4_dequantize: bad sizes rows=%lld k=%lld", (long long)rows, (long long)k);
  LEC_CHECK_ARG(out && codes && scales && ld >= k, "mxfp4_dequantize: null pointer or ld=%lld < k=%lld", (long long)ld, (long long)k);
  LEC_CHECK_ARG(dtype == LEC_DTYPE_F32 || dtype == LEC_DTYPE_BF16, "mxfp4_dequantize: dtype %d does not hold every value (fp32 or bf16)", dtype);
  const int KT = (int)ceil_div(k, 128), KG = (int)ceil_div(k, 512);
  const int64_t ntask = ceil_div(rows, 16) * KG;
  if (dtype == LEC_DTYPE_F32)
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<float>), dim3(grid_of(ntask)), dim3(256), 0, (hipStream_t)stream, (const unsigned int*)codes, (const unsigned char*)scales, rows, (int)k, KT, KG,
                       ntask, (float*)out, ld);
  else
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<__hip_bfloat16>), dim3(grid_of(ntask)), dim3(256), 0, (hipStream_t)stream, (const unsigned int*)codes, (const unsigned char*)scales, rows, (int)k,
                       KT, KG, ntask, (__hip_bfloat16*)out, ld);
  LEC_CHECK_LAUNCH("mxfp4_dequantize_kernel");
  return LEC_OK;
}

extern "C" int64_t lec_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t k) {
  return sizes_ok(M, k) && sizes_ok(N, k) ? lec::codes_bytes(M, k) + lec::scales_bytes(M, k) : LEC_E_ARG;
}

extern "C" int lec_mxfp4_linear(const void* x, int xdtype, int64_t ldx, int64_t M, const void* wcodes, const void* wscales, int64_t N, int64_t k, const float* bias, void* y, int ydtype,
                                int64_t ldy, void* workspace, int64_t workspace_bytes, lec_stream_t stream) {
  using namespace lec;
  LEC_CHECK_ARG(sizes_ok(M, k) && sizes_ok(N, k), "mxfp4_linear: bad sizes M=%lld N=%lld k=%lld", (long long)M, (long long)N, (long long)k);
  LEC_CHECK_ARG(x && wcodes && wscales && y && ldx >= k && ldy >= N, "mxfp4_linear: null pointer or ldx=%lld < k or ldy=%lld < N", (long long)ldx, (long long)ldy);
  const int64_t need = codes_bytes(M, k) + scales_bytes(M, k);
  LEC_CHECK_ARG(workspace && workspace_bytes >= need, "mxfp4_linear: workspace needs %lld bytes", (long long)need);
  LEC_CHECK_ARG(ydtype == LEC_DTYPE_F32 || ydtype == LEC_DTYPE_BF16 || ydtype == LEC_DTYPE_F16, "mxfp4_linear: unknown dtype %d", ydtype);
  LEC_CHECK_ARG(xdtype == LEC_DTYPE_F32 || xdtype == LEC_DTYPE_BF16 || xdtype == LEC_DTYPE_F16, "mxfp4_linear: unknown dtype %d", xdtype);
  hipStream_t st = (hipStream_t)stream;
  const int KT = (int)ceil_div(k, 128), KG = (int)ceil_div(k, 512), K = (int)k;
  const int64_t ntn = ceil_div(N, 16), mtn = ceil_div(M, 16);
  const size_t lds = (size_t)KT * 1024 + (size_t)KG * 256;       // x in 4 bits
  if (mtn == 1 && lds <= 64 * 1024) {
    by_dtype(xdtype, "", [&](auto* xtag) {
      by_dtype(ydtype, "", [&](auto* ytag) {
        using TX = std::remove_pointer_t<decltype(xtag)>;
        using T = std::remove_pointer_t<decltype(ytag)>;
        hipLaunchKernelGGL((mxfp4_linear_rows_kernel<TX, T>), dim3((unsigned)ceil_div(ntn, 4)), dim3(256), lds, st, (const TX*)x, ldx, (int)M, (const uint4*)wcodes,
                           (const unsigned int*)wscales, (int)N, K, KT, KG, bias, (T*)y, ldy);
      });
    });
    LEC_CHECK_LAUNCH("mxfp4_linear_rows_kernel");
    return LEC_OK;
  }
  void* xs = (char*)workspace + codes_bytes(M, k);
  const int rc = quantize(x, xdtype, ldx, M, K, workspace, xs, st);
  if (rc != LEC_OK) return rc;
  const int64_t nbn = ceil_div(N, 256), nbm = ceil_div(M, 256);
  if (nbn * nbm >= 128 && KT <= 32768) {
    const int64_t per = ceil_div(nbn * nbm, 8);
    LEC_CHECK_ARG(per <= (1 << 20), "mxfp4_linear: y has %lld tiles, too many for one call", (long long)(nbn * nbm));
    int rl = LEC_OK;
    by_dtype(ydtype, "", [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      static const hipError_t set = hipFuncSetAttribute((const void*)mxfp4_linear_big_kernel<T>, hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
      if (set != hipSuccess) { rl = hip_fail(set, "mxfp4_linear_big_kernel"); return; }
      hipLaunchKernelGGL((mxfp4_linear_big_kernel<T>), dim3((unsigned)(per * 8)), dim3(256), 128 * 1024, st, (const uint4*)workspace, (const unsigned int*)xs, M, (const uint4*)wcodes,
                         (const unsigned int*)wscales, (int)N, KT, KG, bias, (T*)y, ldy, (int)nbn, (int)nbm, (int)per);
    });
    if (rl != LEC_OK) return rl;
    LEC_CHECK_LAUNCH("mxfp4_linear_big_kernel");
    return LEC_OK;
  }
  int rl = LEC_OK;
  by_dtype(ydtype, "", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto run = [&](auto kernel, int WN, int WM, int NT, int MT) {
      const int64_t gy = ceil_div(mtn, WM * MT);
      if (gy > 65535) { set_error("mxfp4_linear: %lld rows in one call of %lld classes, too many", (long long)M, (long long)N); rl = LEC_E_ARG; return; }
      hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(ntn, WN * NT), (unsigned)gy), dim3(64 * WN * WM), 0, st, (const uint4*)workspace, (const unsigned int*)xs, M, (const uint4*)wcodes,
                         (const unsigned int*)wscales, (int)N, KT, KG, bias, (T*)y, ldy);
    };
    if (mtn <= 4) run(mxfp4_linear_small_kernel<T, 4, 1, 1, 4>, 4, 1, 1, 4);
    else if (ntn * mtn <= 4096) run(mxfp4_linear_small_kernel<T, 2, 2, 1, 2>, 2, 2, 1, 2);
    else run(mxfp4_linear_small_kernel<T, 2, 2, 4, 4>, 2, 2, 4, 4);
  });
  if (rl != LEC_OK) return rl;
  LEC_CHECK_LAUNCH("mxfp4_linear_small_kernel");
  return LEC_OK;
}
