// Rows held in 8 bits, and scores as products of them.
//
//   top = max |x|, code = rint(x (127 / top)), scale = top / 127          out_ij = scale_i scale_j sum_k code_ik code_jk + biases
//
// Codes lie in rows of nncf_int8_pitch(k) bytes, zeros behind the k-th: whole steps of the integer matrix instruction, 16-byte
// aligned.  The integer sum is exact (k <= 131,072: 127^2 k < 2^31), so nothing depends on the order of a sum.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "devutil.h"

namespace nncf {
namespace {

constexpr int kMaxDepth = 131072;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

__host__ __device__ inline int64_t pitch_of(int64_t k) { return k <= 64 ? 64 : (k + 127) / 128 * 128; }

template <class E>
__device__ __forceinline__ void load8(const E* row, int64_t c0, int64_t k, bool vec, float* x) {
  if (vec && c0 + 8 <= k) {   // rows start on a multiple of 4 elements
    typedef E E4 __attribute__((ext_vector_type(4)));
    const E4 a = *reinterpret_cast<const E4*>(row + c0), b = *reinterpret_cast<const E4*>(row + c0 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = (float)a[e];
      x[4 + e] = (float)b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = c0 + e < k ? (float)row[c0 + e] : 0.f;
  }
}

// what a row's codes are made with: the factor, the scale; pre: a power of two that keeps 127 / top finite for tiny rows
struct Coder {
  float pre, inv, scale;
};
__device__ __forceinline__ Coder coder_for(float top, bool finite, float sum2, int normalize) {
  Coder c;
  c.pre = top < 0x1p-100f ? 0x1p64f : 1.f;
  const float t = top * c.pre;
  c.inv = finite && t > 0.f ? 127.f / t : 0.f;
  c.scale = finite ? top / 127.f : NAN;
  if (normalize) c.scale *= rsqrtf(fmaxf(sum2, kNormEps));
  return c;
}
__device__ __forceinline__ uint64_t codes8(const float* x, Coder c) {
  uint64_t r = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int q = c.inv > 0.f ? (int)rintf((x[e] * c.pre) * c.inv) : 0;
    r |= (uint64_t)(uint8_t)(int8_t)q << (8 * e);
  }
  return r;
}

// One row per LR lanes, 8 columns a lane and step.  Rows of one step (LR = 8, 16) stay in registers between the two uses of a
// value; longer ones are read twice, the second time from a cache.
template <class E, int LR, bool ONE>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const E* __restrict__ x, int64_t stride, int64_t n, int64_t k, int vec,
                                                            int normalize, int8_t* __restrict__ q, float* __restrict__ scale) {
  const int64_t row = (int64_t)blockIdx.x * (256 / LR) + threadIdx.x / LR;
  if (row >= n) return;
  const int lane = threadIdx.x % LR;
  const E* src = x + row * stride;
  const int64_t pitch = pitch_of(k);
  float v[8];
  float top = 0.f, sum2 = 0.f;
  bool finite = true;
  for (int64_t c0 = 8 * lane; c0 < pitch; c0 += 8 * LR) {
    load8(src, c0, k, vec != 0, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(v[e]);
      finite = finite && a < INFINITY;
      top = fmaxf(top, a);
      sum2 = fmaf(v[e], v[e], sum2);
    }
    if (ONE) break;
  }
  int ok = finite;
#pragma unroll
  for (int o = LR / 2; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor(top, o));
    sum2 += __shfl_xor(sum2, o);
    ok &= __shfl_xor(ok, o);
  }
  const Coder c = coder_for(top, ok != 0, sum2, normalize);
  for (int64_t c0 = 8 * lane; c0 < pitch; c0 += 8 * LR) {
    if (!ONE) load8(src, c0, k, vec != 0, v);
    *reinterpret_cast<uint64_t*>(q + row * pitch + c0) = codes8(v, c);
    if (ONE) break;
  }
  if (lane == 0) scale[row] = c.scale;
}

template <class E>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, int64_t n,
                                                              int64_t k, int64_t groups, E* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // groups of 8 columns
  if (i >= n * groups) return;
  const int64_t row = i / groups, c0 = (i - row * groups) * 8;
  const uint64_t v = *reinterpret_cast<const uint64_t*>(q + row * pitch_of(k) + c0);
  const float s = scale[row];
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(v >> (8 * e)) * s;
  E* dst = out + row * k + c0;
  if (k % 8 == 0) {
    typedef E E4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      E4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (E)f[4 * h + e];
      *reinterpret_cast<E4*>(dst + 4 * h) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < k) dst[e] = (E)f[e];
  }
}

struct Scores {
  const int8_t *qx, *qt;
  const float *sx, *st, *rb, *cb;
  void* out;
  int64_t m, c, out_stride, pitch;
};

// ---- many rows: 128 x 128 outputs per workgroup, 64 x 64 per wave, k in steps of KB bytes through LDS ------------------------------
constexpr int kMT = 128;

template <int KB>
__device__ __forceinline__ int tile_at(int row, int chunk) {   // 16-byte chunks; see the bank note at the reads
  if (KB == 128) return row * 128 + ((chunk ^ (row >> 1 & 7)) << 4);
  return row * 64 + ((chunk ^ (row >> 2 & 3)) << 4);
}

template <class E, int KB>
__global__ void __launch_bounds__(256, 2) int8_scores_kernel(Scores a, int64_t m_tiles) {
  __shared__ __attribute__((aligned(16))) char s_x[kMT * KB], s_t[kMT * KB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  const int64_t m0 = (int64_t)(blockIdx.x % m_tiles) * kMT, c0 = (int64_t)(blockIdx.x / m_tiles) * kMT;
  const int wm = (wave >> 1) * 64, wc = (wave & 1) * 64;
  i32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = 0;
  for (int64_t k0 = 0; k0 < a.pitch; k0 += KB) {
    __syncthreads();
    for (int i = tid; i < kMT * KB / 16; i += 256) {
      const int row = i / (KB / 16), chunk = i % (KB / 16);
      const int64_t rx = std::min(m0 + row, a.m - 1), rt = std::min(c0 + row, a.c - 1);
      *reinterpret_cast<int4*>(s_x + tile_at<KB>(row, chunk)) = *reinterpret_cast<const int4*>(a.qx + rx * a.pitch + k0 + chunk * 16);
      *reinterpret_cast<int4*>(s_t + tile_at<KB>(row, chunk)) = *reinterpret_cast<const int4*>(a.qt + rt * a.pitch + k0 + chunk * 16);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KB / 32; ++k) {
      i32x4 x[2], t[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = *reinterpret_cast<const i32x4*>(s_x + tile_at<KB>(wm + 32 * i + col, 2 * k + half));
        t[i] = *reinterpret_cast<const i32x4*>(s_t + tile_at<KB>(wc + 32 * i + col, 2 * k + half));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[i], t[j], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t item = c0 + wc + 32 * j + col;
    if (item >= a.c) continue;
    const float st = a.st[item], cb = a.cb ? a.cb[item] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t row = m0 + wm + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
        if (row < a.m) {
          const float v = ((float)acc[i][j][r] * a.sx[row]) * st + (a.rb ? a.rb[row] + cb : cb);
          reinterpret_cast<E*>(a.out)[row * a.out_stride + item] = (E)v;
        }
      }
  }
}

// ---- up to 32 rows: the table is read once, 32 items per wave straight into the operands ------------------------------------------
template <class E>
__global__ void __launch_bounds__(256) int8_scores_few_kernel(Scores a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
  const int64_t c0 = ((int64_t)blockIdx.x * 4 + wave) * 32;
  if (c0 >= a.c) return;
  const int8_t* t = a.qt + std::min(c0 + col, a.c - 1) * a.pitch + half * 16;
  const int8_t* x = a.qx + std::min<int64_t>(col, a.m - 1) * a.pitch + half * 16;
  i32x16 acc = 0;
  for (int64_t k0 = 0; k0 < a.pitch; k0 += 64) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*reinterpret_cast<const i32x4*>(t + k0 + 32 * k),
                                                  *reinterpret_cast<const i32x4*>(x + k0 + 32 * k), acc, 0, 0, 0);
  }
  if (col >= a.m) return;
  const float sx = a.sx[col], rb = a.rb ? a.rb[col] : 0.f;
  E* out = reinterpret_cast<E*>(a.out) + (int64_t)col * a.out_stride;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t item = c0 + 8 * (r >> 2) + 4 * half + (r & 3);
    if (item < a.c) out[item] = (E)(((float)acc[r] * sx) * a.st[item] + (a.cb ? rb + a.cb[item] : rb));
  }
}

template <class E>
int run_quantize(const void* x, int64_t stride, int64_t n, int64_t k, int normalize, int8_t* q, float* scale, hipStream_t st) {
  const E* p = reinterpret_cast<const E*>(x);
  const int vec = (uintptr_t)x % (4 * sizeof(E)) == 0 && stride % 4 == 0;
  const int64_t pitch = pitch_of(k);
  ProfScope ps("quantize_rows_kernel", st);
  if (pitch == 64)
    hipLaunchKernelGGL((quantize_rows_kernel<E, 8, true>), dim3((unsigned)((n + 31) / 32)), dim3(256), 0, st, p, stride, n, k, vec, normalize, q, scale);
  else if (pitch == 128)
    hipLaunchKernelGGL((quantize_rows_kernel<E, 16, true>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, st, p, stride, n, k, vec, normalize, q, scale);
  else
    hipLaunchKernelGGL((quantize_rows_kernel<E, 64, false>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, p, stride, n, k, vec, normalize, q, scale);
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

template <class E>
int run_scores(const Scores& a, hipStream_t st) {
  ProfScope ps("int8_scores_kernel", st);
  if (a.m <= 32) {
    hipLaunchKernelGGL((int8_scores_few_kernel<E>), dim3((unsigned)((a.c + 127) / 128)), dim3(256), 0, st, a);
  } else {
    const int64_t mt = (a.m + kMT - 1) / kMT, ct = (a.c + kMT - 1) / kMT;
    NNCF_REQUIRE(mt * ct < (1LL << 31), "%lld x %lld scores in one call", (long long)a.m, (long long)a.c);
    if (a.pitch == 64)
      hipLaunchKernelGGL((int8_scores_kernel<E, 64>), dim3((unsigned)(mt * ct)), dim3(256), 0, st, a, mt);
    else
      hipLaunchKernelGGL((int8_scores_kernel<E, 128>), dim3((unsigned)(mt * ct)), dim3(256), 0, st, a, mt);
  }
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

bool known(int32_t dtype) { return dtype == NNCF_F32 || dtype == NNCF_F16 || dtype == NNCF_BF16; }
uintptr_t size_of(int32_t dtype) { return dtype == NNCF_F32 ? 4 : 2; }
}  // namespace
}  // namespace nncf

extern "C" int64_t nncf_int8_pitch(int32_t k) { return k > 0 && k <= nncf::kMaxDepth ? nncf::pitch_of(k) : -1; }

extern "C" int nncf_quantize_rows(const void* d_x, int64_t x_stride, int32_t dtype, int64_t n, int32_t k, int32_t normalize, int8_t* d_q,
                                  float* d_scale, void* stream) {
  using namespace nncf;
  NNCF_REQUIRE(n >= 0 && n <= (1LL << 31), "n = %lld rows out of range (0..2^31)", (long long)n);
  NNCF_REQUIRE(k > 0 && k <= kMaxDepth, "k = %d out of range (1..%d)", k, kMaxDepth);
  NNCF_REQUIRE(known(dtype), "dtype = %d unknown", dtype);
  if (n == 0) return NNCF_OK;
  NNCF_REQUIRE(d_x && d_q && d_scale, "NULL argument");
  NNCF_REQUIRE(x_stride >= k, "row stride %lld is below k = %d", (long long)x_stride, k);
  NNCF_REQUIRE((uintptr_t)d_x % size_of(dtype) == 0, "rows are not aligned to their elements");
  NNCF_REQUIRE(((uintptr_t)d_q & 15) == 0, "codes must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  if (dtype == NNCF_F32) return run_quantize<float>(d_x, x_stride, n, k, normalize, d_q, d_scale, st);
  if (dtype == NNCF_F16) return run_quantize<_Float16>(d_x, x_stride, n, k, normalize, d_q, d_scale, st);
  return run_quantize<__bf16>(d_x, x_stride, n, k, normalize, d_q, d_scale, st);
}

extern "C" int nncf_dequantize_rows(const int8_t* d_q, const float* d_scale, int64_t n, int32_t k, void* d_out, int32_t dtype, void* stream) {
  using namespace nncf;
  NNCF_REQUIRE(n >= 0 && n <= (1LL << 31), "n = %lld rows out of range (0..2^31)", (long long)n);
  NNCF_REQUIRE(k > 0 && k <= kMaxDepth, "k = %d out of range (1..%d)", k, kMaxDepth);
  NNCF_REQUIRE(known(dtype), "dtype = %d unknown", dtype);
  if (n == 0) return NNCF_OK;
  NNCF_REQUIRE(d_q && d_scale && d_out, "NULL argument");
  NNCF_REQUIRE(((uintptr_t)d_q & 15) == 0 && ((uintptr_t)d_out & 15) == 0, "codes and output must be 16-byte aligned");
  const int64_t groups = (k + 7) / 8, blocks = (n * groups + 255) / 256;
  NNCF_REQUIRE(blocks < (1LL << 31), "%lld x %d values in one call", (long long)n, k);
  hipStream_t st = as_stream(stream);
  {
    ProfScope ps("dequantize_rows_kernel", st);
    const dim3 grid((unsigned)blocks);
    if (dtype == NNCF_F32)
      hipLaunchKernelGGL((dequantize_rows_kernel<float>), grid, dim3(256), 0, st, d_q, d_scale, n, (int64_t)k, groups, (float*)d_out);
    else if (dtype == NNCF_F16)
      hipLaunchKernelGGL((dequantize_rows_kernel<_Float16>), grid, dim3(256), 0, st, d_q, d_scale, n, (int64_t)k, groups, (_Float16*)d_out);
    else
      hipLaunchKernelGGL((dequantize_rows_kernel<__bf16>), grid, dim3(256), 0, st, d_q, d_scale, n, (int64_t)k, groups, (__bf16*)d_out);
  }
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

extern "C" int nncf_int8_scores(const int8_t* d_qx, const float* d_sx, int64_t m, const int8_t* d_qt, const float* d_st, int64_t c, int32_t k,
                                const float* d_row_bias, const float* d_col_bias, void* d_out, int64_t out_stride, int32_t dtype, void* stream) {
  using namespace nncf;
  NNCF_REQUIRE(m >= 0 && c >= 0 && m <= (1LL << 31) && c <= (1LL << 31), "%lld x %lld scores out of range", (long long)m, (long long)c);
  NNCF_REQUIRE(k > 0 && k <= kMaxDepth, "k = %d out of range (1..%d)", k, kMaxDepth);
  NNCF_REQUIRE(known(dtype), "dtype = %d unknown", dtype);
  if (m == 0 || c == 0) return NNCF_OK;
  NNCF_REQUIRE(d_qx && d_sx && d_qt && d_st && d_out, "NULL argument");
  NNCF_REQUIRE(((uintptr_t)d_qx & 15) == 0 && ((uintptr_t)d_qt & 15) == 0, "codes must be 16-byte aligned");
  NNCF_REQUIRE((uintptr_t)d_out % size_of(dtype) == 0, "output is not aligned to its elements");
  NNCF_REQUIRE(out_stride >= c, "output stride %lld is below c = %lld", (long long)out_stride, (long long)c);
  const Scores a{d_qx, d_qt, d_sx, d_st, d_row_bias, d_col_bias, d_out, m, c, out_stride, pitch_of(k)};
  hipStream_t st = as_stream(stream);
  if (dtype == NNCF_F32) return run_scores<float>(a, st);
  if (dtype == NNCF_F16) return run_scores<_Float16>(a, st);
  return run_scores<__bf16>(a, st);
}
