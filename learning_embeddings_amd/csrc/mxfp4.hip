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

// 32 elements at x (n of them exist) -> 32 codes and the scale byte
template <typename T>
__device__ __forceinline__ uint4 quantize_block(const T* __restrict__ x, int n, unsigned int& scale) {
  float v[32];
  if (n >= 32) {
    T raw[32];
    __builtin_memcpy(raw, (const void*)x, sizeof(raw));          // 16-byte loads at element alignment
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = to_f32(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = i < n ? to_f32(x[i]) : 0.0f;
  }
  unsigned int top = 0;                                          // as integers: a NaN is above infinity, infinity above every number
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const int e = (int)(top >> 23);                                // floor(log2 max) = e - 127 (0 for subnormals, whose byte is clamped to 0 anyway)
  if (e == 255) { scale = 255u; return make_uint4(0u, 0u, 0u, 0u); }
  scale = (unsigned int)max(e - 2, 0);
  const float inv = __uint_as_float((254u - scale) << 23);       // 1 / X, exact
  unsigned int w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[q] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = v[q * 8 + j];
      const float a = fabsf(f) * inv;                            // exact (or far below the first threshold), < 8
      const float magic = a < 2.0f ? 6291456.0f : (a < 4.0f ? 12582912.0f : 25165824.0f);      // 1.5 * 2^23 * the spacing: the sum rounds to a multiple of it, ties to even
      const float r = (a + magic) - magic;
      const int code = min(r < 2.0f ? (int)(2.0f * r) : (r < 4.0f ? (int)r + 2 : (int)(0.5f * r) + 4), 7);
      w[q] |= (unsigned int)(code | ((__float_as_uint(f) >> 28) & 8u)) << (4 * j);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One wave a row tile and a group of four k tiles (a scale word).
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int K, int KT, int KG, int64_t ntask, uint4* __restrict__ codes,
                                                             unsigned int* __restrict__ scales) {
  const int lane = threadIdx.x & 63, r = lane & 15, kb = lane >> 4;
  const int64_t nwave = (int64_t)gridDim.x * 4;
  for (int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); task < ntask; task += nwave) {
    const int64_t rt = task / KG;
    const int kg = (int)(task - rt * KG);
    const int64_t row = rt * 16 + r;
    unsigned int word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int kt = kg * 4 + i;
      if (kt >= KT) break;
      const int k = kt * 128 + kb * 32;
      unsigned int s = 0;
      uint4 c = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows && k < K) c = quantize_block(x + row * ld + k, K - k, s);
      codes[(rt * KT + kt) * 64 + lane] = c;
      word |= s << (8 * i);
    }
    scales[(rt * KG + kg) * 64 + lane] = word;
  }
}

__device__ __forceinline__ float decode(unsigned int code, int scale) {
  const float mag[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
  const float v = ldexpf(mag[code & 7u], scale - 127);
  return scale == 255 ? __builtin_nanf("") : ((code & 8u) ? -v : v);
}

template <typename T>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint4* __restrict__ codes, const unsigned char* __restrict__ scales, int64_t rows, int K, int KT, int KG,
                                                               int64_t ntask, T* __restrict__ out, int64_t ld) {
  const int lane = threadIdx.x & 63, r = lane & 15, kb = lane >> 4;
  const int64_t nwave = (int64_t)gridDim.x * 4;
  for (int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); task < ntask; task += nwave) {
    const int64_t rt = task / KT;
    const int kt = (int)(task - rt * KT);
    const int64_t row = rt * 16 + r;
    const int k = kt * 128 + kb * 32;
    if (row >= rows || k >= K) continue;
    const uint4 c = codes[(rt * KT + kt) * 64 + lane];
    const int s = scales[((rt * KG + (kt >> 2)) * 64 + lane) * 4 + (kt & 3)];
    const unsigned int w[4] = {c.x, c.y, c.z, c.w};
    T v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = from_f32<T>(decode(w[i >> 3] >> (4 * (i & 7)), s));
    T* o = out + row * ld + k;
    if (k + 32 <= K) __builtin_memcpy((void*)o, v, sizeof(v));
    else {
#pragma unroll
      for (int i = 0; i < 32; ++i) if (k + i < K) o[i] = v[i];
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
// A wave owns NT x MT tiles, a block 2 x 2 waves; operands straight from memory (every load is a contiguous kilobyte).
template <typename T, int NT, int MT>
__global__ __launch_bounds__(256) void mxfp4_linear_kernel(const uint4* __restrict__ xc, const unsigned int* __restrict__ xs, int64_t M, const uint4* __restrict__ wc,
                                                           const unsigned int* __restrict__ wsc, int N, int KT, int KG, const float* __restrict__ bias, T* __restrict__ y, int64_t ldy) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nt0 = ((int)blockIdx.x * 2 + (wave & 1)) * NT, ntn = (N + 15) >> 4;
  const int64_t mt0 = ((int64_t)blockIdx.y * 2 + (wave >> 1)) * MT, mtn = (M + 15) >> 4;
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
#pragma unroll
    for (int e = 0; e < 4; ++e) bv[e] = bias && n + e < N ? bias[n + e] : 0.0f;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int64_t m = (mt0 + j) * 16 + (lane & 15);
      if (m >= M || n >= N) continue;
      T o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(acc[i][j][e] + bv[e]);
      T* p = y + m * ldy + n;
      if (n + 4 <= N) __builtin_memcpy((void*)p, o, sizeof(o));
      else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e < N) p[e] = o[e];
      }
    }
  }
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
static unsigned grid_of(int64_t waves) { const int64_t b = ceil_div(waves, 4); return (unsigned)(b > (1 << 22) ? (1 << 22) : b); }

static int quantize(const void* x, int dtype, int64_t ld, int64_t rows, int K, void* codes, void* scales, hipStream_t st) {
  const int KT = (int)ceil_div(K, 128), KG = (int)ceil_div(K, 512);
  const int64_t ntask = ceil_div(rows, 16) * KG;
  const int rc = by_dtype(dtype, "mxfp4_quantize", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL((mxfp4_quantize_kernel<T>), dim3(grid_of(ntask)), dim3(256), 0, st, (const T*)x, ld, rows, K, KT, KG, ntask, (uint4*)codes, (unsigned int*)scales);
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
  const int64_t ntask = ceil_div(rows, 16) * KT;
  if (dtype == LEC_DTYPE_F32)
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<float>), dim3(grid_of(ntask)), dim3(256), 0, (hipStream_t)stream, (const uint4*)codes, (const unsigned char*)scales, rows, (int)k, KT, KG,
                       ntask, (float*)out, ld);
  else
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<__hip_bfloat16>), dim3(grid_of(ntask)), dim3(256), 0, (hipStream_t)stream, (const uint4*)codes, (const unsigned char*)scales, rows, (int)k,
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
  hipStream_t st = (hipStream_t)stream;
  void* xs = (char*)workspace + codes_bytes(M, k);
  const int rc = quantize(x, xdtype, ldx, M, (int)k, workspace, xs, st);
  if (rc != LEC_OK) return rc;
  const int KT = (int)ceil_div(k, 128), KG = (int)ceil_div(k, 512);
  const int64_t gy = ceil_div(M, 128);
  LEC_CHECK_ARG(gy <= 65535, "mxfp4_linear: %lld rows in one call (at most %d)", (long long)M, 65535 * 128);
  by_dtype(ydtype, "mxfp4_linear", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL((mxfp4_linear_kernel<T, 4, 4>), dim3((unsigned)ceil_div(N, 128), (unsigned)gy), dim3(256), 0, st, (const uint4*)workspace, (const unsigned int*)xs, M,
                       (const uint4*)wcodes, (const unsigned int*)wscales, (int)N, KT, KG, bias, (T*)y, ldy);
  });
  LEC_CHECK_LAUNCH("mxfp4_linear_kernel");
  return LEC_OK;
}
