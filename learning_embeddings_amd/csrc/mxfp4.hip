// Microscaled 4-bit floating point: quantisation, its inverse, and the product of a classifier head held in it.
//
// Form (OCP microscaling, MXFP4): blocks of 32 elements along a row share a power of two X = 2^(clamp(floor(log2 max|v|) - 2, -127, 127)), kept as the byte
// log2 X + 127; an element is v / X rounded to nearest, ties to even, into {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign, saturating at 6.  A block that holds a NaN or an
// infinity has the byte 255 and stands for NaN.  17/32 bytes an element.
//
// Layout: the matrix instruction's own.  v_mfma_scale_f32_32x32x64_f8f6f4 takes from lane l the 32 codes (16 bytes) of row l % 32, elements 32 (l / 32) .. + 32 of a
// 64-element stretch, and one scale byte for them.  So a tile of 32 rows x 64 elements is 1 KB in lane order (codes[row tile][k tile][lane][16]): a wave's operand load is
// one contiguous kilobyte, from memory or from LDS, with no bank conflict and no shuffle.  The scale bytes of four consecutive k tiles sit in one 32-bit word a lane
// (scales[row tile][k tile / 4][lane][4]), which the instruction selects a byte of.  Rows are padded to 32 and elements to 64 with zeros.
// (The 16x16x128 form does the same work per instruction in half the cycles, but its issue -- two words for the scales, two for the product -- then takes longer than the
// product: measured alone 5.4 PFLOP/s with one wave a SIMD and 6.7 with two, against 9.2 and 9.3 for 32x32x64.)
#include "lec_common.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <atomic>

namespace lec {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t codes_bytes(int64_t rows, int64_t k) { return ceil_div(rows, 32) * ceil_div(k, 64) * 1024; }
static int64_t scales_bytes(int64_t rows, int64_t k) { return ceil_div(rows, 32) * ceil_div(k, 256) * 256; }

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

// A block takes a row tile and a group of four k tiles (32 rows x 256 elements, one scale word a lane of the layout): half a wave reads 256 consecutive elements of a row,
// 16 bytes a lane (32 of fp32), and the block writes its 4 KB of codes in one piece through LDS (a tile's half is padded by 8 words: the eight halves a wave writes to at
// once start in different banks).  50 000 x 2 048 bf16: 54 - 63 us = 4.1 - 4.8 TB/s, and 39 us = 6.6 TB/s back (a copy: 5.1).
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int K, int KT, int KG, int64_t ntask, uint4* __restrict__ codes,
                                                             unsigned int* __restrict__ scales) {
  __shared__ __attribute__((aligned(16))) unsigned int s_code[8 * 136];
  __shared__ unsigned char s_scale[256];
  const int t = threadIdx.x, c = t & 31, r0 = t >> 5;            // eight half waves, four rows each
  const int ktl = c >> 3, kh = (c >> 2) & 1, sub = c & 3;
  for (int64_t task = blockIdx.x; task < ntask; task += gridDim.x) {
    const int64_t rt = task / KG;
    const int kg = (int)(task - rt * KG), k = kg * 256 + c * 8;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = rt * 32 + r0 + 8 * i;
      load8(x + row * ld + k, row < rows ? K - k : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 8 * i;
      unsigned int sc;
      s_code[(ktl * 2 + kh) * 136 + r * 4 + sub] = quantize8(v[i], sc);
      if (sub == 0) s_scale[(kh * 32 + r) * 4 + ktl] = (unsigned char)sc;
    }
    __syncthreads();
    const int kt = kg * 4 + (t >> 6);
    if (kt < KT) codes[(rt * KT + kt) * 64 + (t & 63)] = *(const uint4*)&s_code[(t >> 5) * 136 + (t & 31) * 4];
    if (t < 64) scales[(rt * KG + kg) * 64 + t] = ((const unsigned int*)s_scale)[t];
    __syncthreads();                                             // (the next task writes both images)
  }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const unsigned int* __restrict__ codes, const unsigned char* __restrict__ scales, int64_t rows, int K, int KT, int KG,
                                                               int64_t ntask, T* __restrict__ out, int64_t ld) {
  const int t = threadIdx.x, c = t & 31, r0 = t >> 5;
  const int ktl = c >> 3, kh = (c >> 2) & 1, sub = c & 3;
  for (int64_t task = blockIdx.x; task < ntask; task += gridDim.x) {
    const int64_t rt = task / KG;
    const int kg = (int)(task - rt * KG), k = kg * 256 + c * 8, kt = kg * 4 + ktl;
    if (k >= K) continue;
    unsigned int w[4], sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 8 * i;                                  // (rows past the end are padding of the same tile)
      w[i] = codes[((rt * KT + kt) * 64 + kh * 32 + r) * 4 + sub];
      sc[i] = scales[((rt * KG + kg) * 64 + kh * 32 + r) * 4 + ktl];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = rt * 32 + r0 + 8 * i;
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

__device__ __forceinline__ f32x16 mfma4(const uint4& a, const uint4& b, f32x16 c, int which, unsigned int sa, unsigned int sb) {
  i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  switch (which) {                                               // (the selected byte is part of the instruction)
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 1, (int)sa, 1, (int)sb);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 2, (int)sa, 2, (int)sb);
    default: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, 3, (int)sa, 3, (int)sb);
  }
}
__device__ __forceinline__ f32x16 zero16() { return f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}; }

// y[m, n] = sum_k x[m, k] w[n, k] + bias[n].  The weights are the A operand: of a tile of 32 classes x 32 rows a lane holds row m = lane % 32 and, in registers
// 4 g .. 4 g + 3, the classes 8 g + 4 (lane / 32) .. + 4.
template <typename T>
__device__ __forceinline__ void store4(T* __restrict__ y, int64_t ldy, int64_t M, int N, int64_t m, int n, const float (&v)[4]) {
  if (m >= M || n >= N) return;
  T o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(v[e]);
  T* p = y + m * ldy + n;
  if (n + 4 <= N) __builtin_memcpy((void*)p, o, sizeof(o));
  else {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (n + e < N) p[e] = o[e];
  }
}
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t make_rsrc(const void* p, unsigned bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00020000); }
__device__ __forceinline__ float bias_at(const rsrc_t& r, int n) { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, n * 4, 0, 0)); }      // past the end, or no bias: 0

template <typename T>
__device__ __forceinline__ void store_tile(T* __restrict__ y, int64_t ldy, int64_t M, int N, int64_t m0, int n0, int lane, const rsrc_t& rbias, const f32x16& acc) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = n0 + 8 * g + 4 * (lane >> 5);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[4 * g + e] + bias_at(rbias, n + e);
    store4(y, ldy, M, N, m0 + (lane & 31), n, v);
  }
}

// Two waves share a tile of 32 classes, each about half of its k tiles, in whole scale words: this wave's are [lo, hi).
__device__ __forceinline__ void half_of(int KT, int half, int& lo, int& hi) {
  const int mid = min((((KT + 1) >> 1) + 3) & ~3, KT);
  lo = half ? mid : 0; hi = half ? KT : mid;
}
// Up to CH of a wave's weight tiles and their scale words, all asked for at once
constexpr int CH = 16;
struct WeightTiles {
  uint4 w[CH];
  unsigned int s[CH / 4];
  __device__ __forceinline__ void fetch(const uint4* __restrict__ wc, const unsigned int* __restrict__ wsc, int64_t nt, int KT, int KG, int kt0, int hi, int lane) {
#pragma unroll
    for (int i = 0; i < CH; ++i) if (kt0 + i < hi) w[i] = wc[(nt * KT + kt0 + i) * 64 + lane];
#pragma unroll
    for (int i = 0; i < CH / 4; ++i) if (kt0 + 4 * i < hi) s[i] = wsc[(nt * KG + (kt0 >> 2) + i) * 64 + lane];
  }
};
// The second half's sums, joined in a fixed order; true for the wave that then holds the whole of them.  All threads of the block call it.
__device__ __forceinline__ bool join_halves(f32x16& acc, f32x4 (*s_half)[4][64], int pair, int half, int lane) {
  if (half) {
#pragma unroll
    for (int g = 0; g < 4; ++g) s_half[pair][g][lane] = f32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
  }
  __syncthreads();
  if (half) return false;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 o = s_half[pair][g][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[4 * g + e] += o[e];
  }
  return true;
}

// A few rows: the time is the weights' way from memory (1 x 50 000 x 2 048: 13.4 us for 54.4 MB = 4.1 TB/s), and a launch to quantise x would cost more than x is worth, so every block quantises it into LDS while its weights
// are under way.  x has to fit LDS beside the join: K <= 3 328.  Columns of x's tile that are no row of x are never written: a column of the product depends on its own
// column only, and those are not stored.
template <typename TX, typename T>
__global__ __launch_bounds__(256) void mxfp4_linear_few_kernel(const TX* __restrict__ x, int64_t ldx, int M, const uint4* __restrict__ wc, const unsigned int* __restrict__ wsc, int N, int K,
                                                               int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ f32x4 s_half[2][4][64];
  unsigned int* xcodes = (unsigned int*)smem;                    // [KT][64][4] words
  unsigned char* xscale = smem + (size_t)KT * 1024;              // [KG][64][4] bytes
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = wave & 1;
  const int ntn = (N + 31) >> 5, nt_ = (int)blockIdx.x * 2 + (wave >> 1), nt = min(nt_, ntn - 1);        // (a pair past the last tile repeats it and stores nothing)
  int lo, hi;
  half_of(KT, half, lo, hi);
  WeightTiles W;
  W.fetch(wc, wsc, nt, KT, KG, lo, hi, lane);
  const int per_row = KG * 32;                                   // 8-element pieces of a row, padded to whole groups of 256
  for (int i = t; i < M * per_row; i += 256) {
    const int r = i / per_row, q = i - r * per_row, k = q * 8, kt = k >> 6, kh = (k >> 5) & 1, sub = (k >> 3) & 3;
    float v[8];
    load8(x + (int64_t)r * ldx + k, K - k, v);
    unsigned int sc;
    const unsigned int c = quantize8(v, sc);
    if (kt < KT) xcodes[(kt * 64 + kh * 32 + r) * 4 + sub] = c;
    if (sub == 0) xscale[((kt >> 2) * 64 + kh * 32 + r) * 4 + (kt & 3)] = (unsigned char)sc;
  }
  __syncthreads();
  f32x16 acc = zero16();
  for (int kt0 = lo; kt0 < hi; kt0 += CH) {
    if (kt0 > lo) W.fetch(wc, wsc, nt, KT, KG, kt0, hi, lane);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int kt = kt0 + i;
      if (kt < hi) acc = mfma4(W.w[i], ((const uint4*)xcodes)[kt * 64 + lane], acc, i & 3, W.s[i >> 2], ((const unsigned int*)xscale)[(kt >> 2) * 64 + lane]);
    }
  }
  if (join_halves(acc, s_half, wave >> 1, half, lane) && nt_ == nt) store_tile(y, ldy, M, N, 0, nt * 32, lane, make_rsrc(bias, bias ? (unsigned)N * 4u : 0u), acc);
}

// Up to 32 rows, and products too small for the ring below: a wave pair a tile of 32 classes x 32 rows, the weights asked for all at once, x (in 4 bits, from the L2) four k
// tiles at a time.
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_linear_rows_kernel(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                                const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy) {
  __shared__ f32x4 s_half[2][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave & 1;
  const int ntn = (N + 31) >> 5, nt_ = (int)blockIdx.x * 2 + (wave >> 1), nt = min(nt_, ntn - 1);        // (a pair past the last tile repeats it and stores nothing)
  const int64_t mt = blockIdx.y;
  int lo, hi;
  half_of(KT, half, lo, hi);
  f32x16 acc = zero16();
  WeightTiles W;
  for (int kt0 = lo; kt0 < hi; kt0 += CH) {
    W.fetch(wc, wsc, nt, KT, KG, kt0, hi, lane);
#pragma unroll
    for (int h = 0; h < CH / 4; ++h) {
      if (kt0 + 4 * h >= hi) break;
      uint4 b[4];
      const unsigned int sb = xs[(mt * KG + (kt0 >> 2) + h) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) if (kt0 + 4 * h + i < hi) b[i] = xc[(mt * KT + kt0 + 4 * h + i) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) if (kt0 + 4 * h + i < hi) acc = mfma4(W.w[4 * h + i], b[i], acc, i, W.s[h], sb);
    }
  }
  if (join_halves(acc, s_half, wave >> 1, half, lane) && nt_ == nt) store_tile(y, ldy, M, N, mt * 32, nt * 32, lane, make_rsrc(bias, bias ? (unsigned)N * 4u : 0u), acc);
}

// Large products.  A block of 2 x 2 waves owns 192 x 192 of y, a wave 96 x 96 (3 x 3 tiles, 144 accumulators), two blocks a CU: while one drains its output to memory -- 7424 x
// 50000 in bf16 are 742 MB, as long on the way as the products take -- the other one multiplies.  A stage of the ring is two k tiles (128 elements) of both operands, 24 KB;
// three stages in LDS are filled by LDS-DMA (a wave's request is one contiguous kilobyte = one operand tile in lane order, so there is nothing to swizzle), two stages ahead.
// Per stage a wave issues 18 MFMAs of 32 cycles and reads 12 KB of LDS: with the fills 144 KB of LDS traffic per 1152 cycles a CU, just under its 128 B / clk.
// The output leaves through LDS in rows, marked as streaming: it then does not push the operands out of the L2.
// Measured, 7 424 x 50 000 x 2 048 to bf16, quantisation of x (10 us) included:  256 x 256 tiles, one block a CU, stores straight from the registers 638 us;  192 x 192, two blocks
// a CU 581;  stores in rows 560;  marked as streaming 460;  biases from LDS 424 - 444 on five machines = 3.5 PFLOP/s.  Without any stores 342, without stores and operand
// traffic 285; the matrix cores alone, on random operands, run at 6.1 PFLOP/s under their power limit: 250.  Counters: matrix cores busy 52 % of the time at 1.9 GHz, 816 MB
// written for 742 (rows of 100 000 bytes start inside cache lines), 145 MB fetched.  Deeper operand look-ahead in the body, a wave priority around the products, other
// widths of the XCDs' bands and staggered starts of a CU's two blocks changed nothing; one image of the block instead of one a wave gained 1 % in 16 bits and lost 1 % in fp32.
// Blocks that stay and fetch their next tile's first stages ahead of the output were slower, in turn on one machine 487 us and this 456: a later stage's arrival is counted behind the stores.
// W = 3 as described; W = 2 (128 x 128 of y, 64 x 64 a wave, three blocks a CU) where the larger tiles would leave CUs without work.
template <int W> struct Ring {
  static constexpr int TILE = 64 * W, RT = 2 * W;                // classes and rows of a block; row tiles of a side
  static constexpr int SIDE = RT * 2048, STAGE = 2 * SIDE, NS = 3;      // bytes of a stage's operand, of a stage; stages
  static constexpr int ROW = 64 * W, PITCH = ROW + 16;           // bytes of an output image's row (32 W classes in 16 bits, half of them in fp32), and with its padding:
                                                                 // sixteen rows start in different banks
  static constexpr int IMAGES = 4 * 32 * W * PITCH;
  static constexpr int LDS = (NS * STAGE > IMAGES ? NS * STAGE : IMAGES) + TILE * 4;      // the ring and, after it, the waves' images in the same place; the biases
};
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef __attribute__((address_space(3))) void lds_ptr;
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); __builtin_amdgcn_s_barrier(); asm volatile("" ::: "memory"); }

// (A body with restrict parameters, inlined into the kernel: its memory accesses then carry alias scopes, without which the compiler waits for every outstanding
// LDS-DMA before any read of LDS -- the ring would be one stage deep.)
template <typename T, int W>
__device__ __forceinline__ void mxfp4_linear_big_body(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                      const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy, int nbn,
                                                      int nbm, int per_xcd) {
  using R = Ring<W>;
  constexpr int RT = R::RT, SIDE = R::SIDE, STAGE = R::STAGE, NS = R::NS, TILE = R::TILE;
  constexpr int IPW = 2 * W;                                     // LDS-DMA instructions a wave issues for a stage
  constexpr int PIN = (int)0x80000000;                           // a volatile load: it stays where it is written, ahead of the requests behind it
  constexpr int OOB = 0x40000000;                                // past any operand buffer (KT <= 32 768: below 2^28 bytes)
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1;
  // consecutive blocks land on the eight XCDs in turn: give each XCD a contiguous run of tiles, eight tiles of rows by all tiles of classes at a time, so that a run's
  // operands stay in its L2
  const int64_t g = (int64_t)((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (g >= (int64_t)nbn * nbm) return;
  const int band = (int)(g / (8 * (int64_t)nbn)), inb = (int)(g - (int64_t)band * 8 * nbn), bw = min(8, nbm - band * 8);
  const int bn = __builtin_amdgcn_readfirstlane(inb / bw), bm = __builtin_amdgcn_readfirstlane(band * 8 + inb % bw);      // (the division leaves them in vector registers)
  const int ntn = (N + 31) >> 5, mtn = (int)((M + 31) >> 5);
  // The block's operand tiles of each side and their scales as buffers that end with the last of them; a tile past the matrix repeats the last one (and is not stored).
  const int na_ = min(RT, ntn - bn * RT), nb_ = min(RT, mtn - bm * RT);
  const rsrc_t ra = make_rsrc(wc + (int64_t)bn * RT * KT * 64, (unsigned)na_ * KT * 1024), rb = make_rsrc(xc + (int64_t)bm * RT * KT * 64, (unsigned)nb_ * KT * 1024);
  const rsrc_t rsa = make_rsrc(wsc + (int64_t)bn * RT * KG * 64, (unsigned)na_ * KG * 256), rsb = make_rsrc(xs + (int64_t)bm * RT * KG * 64, (unsigned)nb_ * KG * 256);
  // Stage st in slot `slot`: [weights: RT row tiles x 2 k tiles | x: the same], a kilobyte each.  Wave w takes k tile w % 2 of the row tiles w / 2 + 2 u.  Past the last k tile:
  // no traffic, zeros in LDS.
  auto issue = [&](int st, int slot) {
    unsigned char* base = smem + slot * STAGE + wave * 1024;
    const int kt = 2 * st + (wave & 1), kc = min(kt, KT - 1), voff = lane * 16 + (kt < KT ? 0 : OOB);
#pragma unroll
    for (int u = 0; u < W; ++u) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr*)(base + u * 4096), 16, voff, (min((wave >> 1) + 2 * u, na_ - 1) * KT + kc) * 1024, 0, 0);
#pragma unroll
    for (int u = 0; u < W; ++u) __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr*)(base + SIDE + u * 4096), 16, voff, (min((wave >> 1) + 2 * u, nb_ - 1) * KT + kc) * 1024, 0, 0);
  };
  f32x16 acc[W][W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = zero16();
  int sa[W], sb[W], na[W], nb[W];                                // scale words: of this group of four k tiles, of the next one
  auto fetch_scales = [&](int kg) {                              // (a group past the end: the last one again)
    const int kc = min(kg, KG - 1);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      na[i] = __builtin_amdgcn_raw_buffer_load_b32(rsa, lane * 4, (min(wn * W + i, na_ - 1) * KG + kc) * 256, PIN);
      nb[i] = __builtin_amdgcn_raw_buffer_load_b32(rsb, lane * 4, (min(wm * W + i, nb_ - 1) * KG + kc) * 256, PIN);
    }
  };
  const uint4* A = (const uint4*)smem + wn * W * 128 + lane;     // this wave's operand tiles of slot 0: [W row tiles][2 k tiles]
  const uint4* B = (const uint4*)(smem + SIDE) + wm * W * 128 + lane;
  float* s_bias = (float*)(smem + R::LDS - TILE * 4);                 // behind the ring and the image
  const rsrc_t rbias = make_rsrc(bias, bias ? (unsigned)N * 4u : 0u);
  const float bias_here = threadIdx.x < TILE ? bias_at(rbias, bn * TILE + (int)threadIdx.x) : 0.0f;      // (past the end: 0)
  fetch_scales(0);
  issue(0, 0); issue(1, 1); issue(2, 2);
  if (threadIdx.x < TILE) s_bias[threadIdx.x] = bias_here;
  wait_vm<2 * IPW>();                                            // stage 0 has landed for this wave ...
  meet();                                                        // ... and for every wave
#pragma unroll
  for (int i = 0; i < W; ++i) {
    sa[i] = na[i]; sb[i] = nb[i];
    asm volatile("" : "+v"(sa[i]), "+v"(sb[i]));                  // in registers before the loop: its own waits then count the loop's requests only
  }
  uint4 a = A[0], b[W];
#pragma unroll
  for (int j = 0; j < W; ++j) b[j] = B[j * 128];
  // One stage: its first k tile's products run while the wave reads the rest of the stage; then everybody is done reading stage st, whose slot takes stage st + 3, and stage
  // st + 1 has landed once at most the younger stage's requests are outstanding (scale loads in between only make the wait stricter); the second k tile's products run while
  // stage st + 1's first operands are read.  The order is pinned: left alone the scheduler puts every read before the first product.  Groups of two stages, the last one filled
  // up with zeros, so that the body has no branch.
  int slot = 0;
  auto stage = [&](int st, auto qc) {
    constexpr int q = decltype(qc)::value;
    const int next = slot == NS - 1 ? 0 : slot + 1;
    const int o = slot * (STAGE / 16), on = next * (STAGE / 16);
    uint4 a0[W], a1[W], b1[W], bx[W];
    a0[0] = a;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i + 1 < W) a0[i + 1] = A[o + (i + 1) * 128];
      b1[i] = B[o + i * 128 + 64];
      a1[i] = A[o + i * 128 + 64];
#pragma unroll
      for (int j = 0; j < W; ++j) acc[i][j] = mfma4(a0[i], b[j], acc[i][j], q, sa[i], sb[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_vm<IPW>();
    meet();
    if (q == 0) fetch_scales((st >> 1) + 1);
    issue(st + 3, slot);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i == 0) a = A[on];
      bx[i] = B[on + i * 128];
#pragma unroll
      for (int j = 0; j < W; ++j) acc[i][j] = mfma4(a1[i], b1[j], acc[i][j], q + 1, sa[i], sb[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < W; ++j) b[j] = bx[j];
    slot = next;
  };
  for (int st = 0; 2 * st < KT; st += 2) {
    stage(st, std::integral_constant<int, 0>{});
    stage(st + 1, std::integral_constant<int, 2>{});
#pragma unroll
    for (int i = 0; i < W; ++i) { sa[i] = na[i]; sb[i] = nb[i]; }
  }
  wait_vm<0>();                                                  // (the stages of zeros past the end still write LDS)
  const bool inside = (int64_t)(bn + 1) * TILE <= N && (int64_t)(bm + 1) * TILE <= M;
  const int64_t m0 = (int64_t)bm * TILE + wm * 32 * W;
  const int n0 = bn * TILE + wn * 32 * W;
  if (inside) {
    // Through LDS, a wave's 32 W x 32 W as an image of its own (fp32: in two halves of the classes), so that memory sees runs of 64 W bytes of a row instead of 32.
    // Lanes l and l + 32 hold the two halves of eight classes: one exchange of half waves between two groups of registers gives every lane eight consecutive classes.
    meet();                                                      // everybody is done with the ring
    constexpr int NW = sizeof(T), PITCH = R::PITCH, PARTS = NW / 2;      // words of four elements; halves of the classes
    constexpr int CW = W * 32 / PARTS;                           // classes of a half
    unsigned char* img = smem + wave * (32 * W * PITCH);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int nn = i * 32 + 16 * h - part * CW;            // (16 classes lie in one half: CW is a multiple of 16)
          if (nn < 0 || nn >= CW) continue;
          float bl[4], bh[4];
          const float* pb = s_bias + wn * 32 * W + i * 32 + 16 * h + 4 * (lane >> 5);
#pragma unroll
          for (int e = 0; e < 4; ++e) { bl[e] = pb[e]; bh[e] = pb[8 + e]; }
#pragma unroll
          for (int j = 0; j < W; ++j) {
            __attribute__((aligned(16))) T lo[4], hi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) { lo[e] = from_f32<T>(acc[i][j][8 * h + e] + bl[e]); hi[e] = from_f32<T>(acc[i][j][8 * h + 4 + e] + bh[e]); }
            unsigned int ul[NW], uh[NW];
            __builtin_memcpy(ul, lo, sizeof(ul)); __builtin_memcpy(uh, hi, sizeof(uh));
#pragma unroll
            for (int k = 0; k < NW; ++k) {
              const auto s = __builtin_amdgcn_permlane32_swap(ul[k], uh[k], false, false);      // (ul low | uh low) , (ul high | uh high) by halves of the wave
              ul[k] = s[0]; uh[k] = s[1];
            }
            uint4* p = (uint4*)(img + (j * 32 + (lane & 31)) * PITCH + (nn + 8 * (lane >> 5)) * (int)sizeof(T));
            if constexpr (NW == 2) p[0] = make_uint4(ul[0], ul[1], uh[0], uh[1]);
            else { p[0] = make_uint4(ul[0], ul[1], ul[2], ul[3]); p[1] = make_uint4(uh[0], uh[1], uh[2], uh[3]); }
          }
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // (the image is this wave's own)
#pragma unroll
      for (int it = 0; it < 2 * W * W; ++it) {                   // 32 W rows of 4 W pieces of 16 bytes
        const int id = it * 64 + lane, r = id / (4 * W), c = id - r * (4 * W);
        __builtin_nontemporal_store(*(const u32x4*)(img + r * PITCH + c * 16), (u32x4_at2*)(y + (m0 + r) * ldy + n0 + part * CW + c * (16 / (int)sizeof(T))));
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) store_tile(y, ldy, M, N, m0 + j * 32, n0 + i * 32, lane, rbias, acc[i][j]);
  }
}

template <typename T, int W>
__global__ __launch_bounds__(256, W == 3 ? 2 : 3) void mxfp4_linear_big_kernel(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                                  const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy,
                                                                  int nbn, int nbm, int per_xcd) {
  mxfp4_linear_big_body<T, W>(xc, xs, M, wc, wsc, N, KT, KG, bias, y, ldy, nbn, nbm, per_xcd);
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

// Dynamic LDS beyond 64 KB has to be allowed, once a kernel and device; `done` = the kernel's devices, a bit each
static hipError_t allow_lds(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Which product (us of a captured call, K = 2048, bf16; `few` | `rows` | ring of 128 x 128 | ring of 192 x 192):
//   N = 50 000:  M = 1: 14.0 | 16.9    2: 16.2 | 16.9    4: 18.1 | 17.0    32: - | 18.1 | 18.5 | 25.2     64: - | 26.3 | 20.7 | 28.2    256: - | 71.3 | 28.6 | 41.7
//                2 048: - | 499 | 140 | 144    4 096: - | 988 | 271 | 258    7 424: - | 1 783 | 478 | 442
//   N = 10 000:  M = 1: 5.6 | 8.7    4: 7.0 | 8.7    64: - | 11.1 | 13.7 | 19.0    128: - | 15.3 | 12.0 | 21.5    4 096: - | 207 | 66.8 | 69.4    7 424: - | 368 | 109.3 | 107.8
//   N = 2 000:   M = 4: 6.9 | 8.6    256: - | 9.1 | 14.3    512: - | 10.9 | 14.7    1 024: - | 14.3 | 15.6    2 048: - | 23.0 | 17.6
// `few` quantises x in every block: up to four rows -- at four it loses 1 us of 17 with 50 000 classes and gains 1.7 of 8.7 with 10 000 and with 2 000, which more heads have.  `rows` starts the most waves but reads the weights once for every tile of rows: one tile of rows, or few tiles in all --
// some more of them where the weights stay in an XCD's 4 MB of L2.
constexpr int kFewRows = 4;
enum class Form { rows, ring2, ring3 };
static Form form_of(int64_t M, int64_t N, int64_t K) {
  const int64_t ntn = ceil_div(N, 32), mtn = ceil_div(M, 32), tiles = ntn * mtn;
  if (mtn == 1 || tiles <= 1024 || (tiles <= 2048 && codes_bytes(N, K) <= (4 << 20)) || ceil_div(K, 64) > 32768) return Form::rows;
  return ceil_div(N, Ring<3>::TILE) * ceil_div(M, Ring<3>::TILE) >= 3000 ? Form::ring3 : Form::ring2;
}

static int quantize(const void* x, int dtype, int64_t ld, int64_t rows, int K, void* codes, void* scales, hipStream_t st) {
  const int KT = (int)ceil_div(K, 64), KG = (int)ceil_div(K, 256);
  const int64_t ntask = ceil_div(rows, 32) * KG;
  const int rc = by_dtype(dtype, "mxfp4_quantize", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL((mxfp4_quantize_kernel<T>), dim3(grid_of(ntask)), dim3(256), 0, st, (const T*)x, ld, rows, K, KT, KG, ntask, (uint4*)codes, (unsigned int*)scales);
  });
  if (rc != LEC_OK) return rc;
  LEC_CHECK_LAUNCH("mxfp4_quantize_kernel");
  return LEC_OK;
}

}  // namespace lec

static bool aligned16(const void* a, const void* b) { return (((uintptr_t)a | (uintptr_t)b) & 15) == 0; }
static bool sizes_ok(int64_t rows, int64_t k) { return rows > 0 && rows <= ((int64_t)1 << 31) - 32 && k > 0 && k <= (1 << 24); }

extern "C" int64_t lec_mxfp4_codes_bytes(int64_t rows, int64_t k) { return sizes_ok(rows, k) ? lec::codes_bytes(rows, k) : LEC_E_ARG; }
extern "C" int64_t lec_mxfp4_scales_bytes(int64_t rows, int64_t k) { return sizes_ok(rows, k) ? lec::scales_bytes(rows, k) : LEC_E_ARG; }

extern "C" int lec_mxfp4_quantize(const void* x, int dtype, int64_t ld, int64_t rows, int64_t k, void* codes, void* scales, lec_stream_t stream) {
  using namespace lec;
  LEC_CHECK_ARG(sizes_ok(rows, k), "mxfp4_quantize: bad sizes rows=%lld k=%lld", (long long)rows, (long long)k);
  LEC_CHECK_ARG(x && codes && scales && ld >= k, "mxfp4_quantize: null pointer or ld=%lld < k=%lld", (long long)ld, (long long)k);
  LEC_CHECK_ARG(aligned16(codes, scales), "mxfp4_quantize: codes and scales have to be 16-byte aligned");
  return quantize(x, dtype, ld, rows, (int)k, codes, scales, (hipStream_t)stream);
}

extern "C" int lec_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t k, void* out, int dtype, int64_t ld, lec_stream_t stream) {
  using namespace lec;
  LEC_CHECK_ARG(sizes_ok(rows, k), "mxfp4_dequantize: bad sizes rows=%lld k=%lld", (long long)rows, (long long)k);
  LEC_CHECK_ARG(out && codes && scales && ld >= k, "mxfp4_dequantize: null pointer or ld=%lld < k=%lld", (long long)ld, (long long)k);
  LEC_CHECK_ARG(aligned16(codes, scales), "mxfp4_dequantize: codes and scales have to be 16-byte aligned");
  LEC_CHECK_ARG(dtype == LEC_DTYPE_F32 || dtype == LEC_DTYPE_BF16, "mxfp4_dequantize: dtype %d does not hold every value (fp32 or bf16)", dtype);
  const int KT = (int)ceil_div(k, 64), KG = (int)ceil_div(k, 256);
  const int64_t ntask = ceil_div(rows, 32) * KG;
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
  LEC_CHECK_ARG(N <= (1 << 28), "mxfp4_linear: %lld classes (at most 2^28)", (long long)N);
  LEC_CHECK_ARG(x && wcodes && wscales && y && ldx >= k && ldy >= N, "mxfp4_linear: null pointer or ldx=%lld < k or ldy=%lld < N", (long long)ldx, (long long)ldy);
  const int64_t need = codes_bytes(M, k) + scales_bytes(M, k);
  LEC_CHECK_ARG(workspace && workspace_bytes >= need, "mxfp4_linear: workspace needs %lld bytes", (long long)need);
  LEC_CHECK_ARG(aligned16(wcodes, wscales) && aligned16(workspace, nullptr), "mxfp4_linear: codes, scales and workspace have to be 16-byte aligned");
  LEC_CHECK_ARG(ydtype == LEC_DTYPE_F32 || ydtype == LEC_DTYPE_BF16 || ydtype == LEC_DTYPE_F16, "mxfp4_linear: unknown dtype %d", ydtype);
  LEC_CHECK_ARG(xdtype == LEC_DTYPE_F32 || xdtype == LEC_DTYPE_BF16 || xdtype == LEC_DTYPE_F16, "mxfp4_linear: unknown dtype %d", xdtype);
  hipStream_t st = (hipStream_t)stream;
  const int KT = (int)ceil_div(k, 64), KG = (int)ceil_div(k, 256), K = (int)k;
  const int64_t ntn = ceil_div(N, 32), mtn = ceil_div(M, 32);
  const size_t lds = (size_t)KT * 1024 + (size_t)KG * 256;       // x in 4 bits
  if (M <= kFewRows && lds <= 64 * 1024 - 8192) {
    by_dtype(xdtype, "", [&](auto* xtag) {
      by_dtype(ydtype, "", [&](auto* ytag) {
        using TX = std::remove_pointer_t<decltype(xtag)>;
        using T = std::remove_pointer_t<decltype(ytag)>;
        hipLaunchKernelGGL((mxfp4_linear_few_kernel<TX, T>), dim3((unsigned)ceil_div(ntn, 2)), dim3(256), lds, st, (const TX*)x, ldx, (int)M, (const uint4*)wcodes,
                           (const unsigned int*)wscales, (int)N, K, KT, KG, bias, (T*)y, ldy);
      });
    });
    LEC_CHECK_LAUNCH("mxfp4_linear_few_kernel");
    return LEC_OK;
  }
  void* xs = (char*)workspace + codes_bytes(M, k);
  const int rc = quantize(x, xdtype, ldx, M, K, workspace, xs, st);
  if (rc != LEC_OK) return rc;
  int rl = LEC_OK;
  by_dtype(ydtype, "", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto ring = [&](auto w) {
      constexpr int W = decltype(w)::value;
      const int64_t nbn = ceil_div(N, Ring<W>::TILE), nbm = ceil_div(M, Ring<W>::TILE), per = ceil_div(nbn * nbm, 8);
      if (per > (1 << 20)) { set_error("mxfp4_linear: y has %lld tiles, too many for one call", (long long)(nbn * nbm)); rl = LEC_E_ARG; return; }
      static std::atomic<unsigned long long> done{0};
      const hipError_t e = allow_lds((const void*)mxfp4_linear_big_kernel<T, W>, Ring<W>::LDS, done);
      if (e != hipSuccess) { rl = hip_fail(e, "mxfp4_linear_big_kernel"); return; }
      hipLaunchKernelGGL((mxfp4_linear_big_kernel<T, W>), dim3((unsigned)(per * 8)), dim3(256), Ring<W>::LDS, st, (const uint4*)workspace, (const unsigned int*)xs, M,
                         (const uint4*)wcodes, (const unsigned int*)wscales, (int)N, KT, KG, bias, (T*)y, ldy, (int)nbn, (int)nbm, (int)per);
    };
    switch (form_of(M, N, k)) {
      case Form::ring3: ring(std::integral_constant<int, 3>{}); break;
      case Form::ring2: ring(std::integral_constant<int, 2>{}); break;
      case Form::rows:
        if (mtn > 65535) { set_error("mxfp4_linear: %lld rows of %d elements in one call, too many", (long long)M, K); rl = LEC_E_ARG; break; }
        hipLaunchKernelGGL((mxfp4_linear_rows_kernel<T>), dim3((unsigned)ceil_div(ntn, 2), (unsigned)mtn), dim3(256), 0, st, (const uint4*)workspace, (const unsigned int*)xs, M,
                           (const uint4*)wcodes, (const unsigned int*)wscales, (int)N, KT, KG, bias, (T*)y, ldy);
    }
  });
  if (rl != LEC_OK) return rl;
  LEC_CHECK_LAUNCH("mxfp4_linear");
  return LEC_OK;
}
