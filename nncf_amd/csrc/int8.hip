// Rows held in 8 bits, and scores as products of them.
//
//   top = max |x|, code = rint(x (127 / top)), scale = top / 127          out_ij = scale_i scale_j sum_k code_ik code_jk + biases
//
// Codes lie in rows of nncf_int8_pitch(k) bytes, zeros behind the k-th: whole steps of the integer matrix instruction, 16-byte
// aligned.  The integer sum is exact (codes of -127 .. 127, k <= 131,072: 127^2 k < 2^31), so nothing depends on the order of a sum.
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

// Bound by its bytes: 1M x 128 fp32 135 us, 644 MB at 4.8 TB/s (a copy of 1 GiB: 5.2); back to fp32 125 us, 5.2 TB/s.
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

// ---- many rows ---------------------------------------------------------------------------------------------------------------
// (32 WM) x (32 WC) outputs per wave, RW x 2 waves; KB codes of every row a stage, two stages in turn, filled from global memory without a
// register (1 KB per wave and instruction).  Chunks of 16 bytes are placed so that the 32 rows of an operand read meet every bank alike.
// 128 codes a stage are whole lines: 2,000 x 16,384 x 4,096 took 165 us in halves of lines with tiles of 128 x 256, whether one stage lay
// ahead or two, and takes 154 (best of 40: 132) in whole ones with 256 x 256: 1.7-2.0 POP/s, the pipe busy in 57% of its cycles (44% before).
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

template <int KB>
__device__ __forceinline__ int code_at(int row, int chunk) {
  return KB == 128 ? row * 128 + ((chunk ^ (row >> 1 & 7)) << 4) : row * 64 + ((chunk ^ (row >> 2 & 3)) << 4);
}

template <int XR, int TR, int KB>
struct __attribute__((aligned(16))) CodeStage {
  char x[XR * KB], t[TR * KB];
};

template <class E, int WM, int WC, int RW, int KB>
__global__ void __launch_bounds__(128 * RW, 2) int8_scores_kernel(Scores a, int64_t m_tiles, int64_t tiles, int vec) {
  constexpr int MT = 32 * WM * RW, CT = 64 * WC, kPer = 1024 / KB;   // kPer rows of one fill
  constexpr int NX = MT / kPer / (2 * RW), NT = CT / kPer / (2 * RW);
  typedef CodeStage<MT, CT, KB> Stage;
  __shared__ Stage s_a, s_b;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  // Workgroups of an XCD (ids of one residue mod 8) take neighbouring tiles, all row tiles of a column of tiles after one another: its
  // L2 reads an eighth of the table and the rows.
  const int64_t share = (tiles + 7) / 8, tile = (int64_t)(blockIdx.x % 8) * share + blockIdx.x / 8;
  if (tile >= tiles) return;
  const int64_t m0 = tile % m_tiles * MT, c0 = tile / m_tiles * CT;
  const int8_t *gx = a.qx + m0 * a.pitch, *gt = a.qt + c0 * a.pitch;
  const int mrows = (int)min((int64_t)MT, a.m - m0), crows = (int)min((int64_t)CT, a.c - c0);
  // rows behind the last are read as the last
  uint32_t ox[NX], ot[NT];
  const int frow = lane / (KB / 16);
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int r = (wave * NX + i) * kPer + frow;
    ox[i] = (uint32_t)min(r, mrows - 1) * (uint32_t)a.pitch + code_at<KB>(r, lane % (KB / 16)) % KB;
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int r = (wave * NT + i) * kPer + frow;
    ot[i] = (uint32_t)min(r, crows - 1) * (uint32_t)a.pitch + code_at<KB>(r, lane % (KB / 16)) % KB;
  }
  auto fill = [&](Stage& st, int64_t k0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NX; ++i) __builtin_amdgcn_global_load_lds((gptr_t)(gx + k0 + ox[i]), (lptr_t)(st.x + (wave * NX + i) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < NT; ++i) __builtin_amdgcn_global_load_lds((gptr_t)(gt + k0 + ot[i]), (lptr_t)(st.t + (wave * NT + i) * 1024), 16, 0, 0);
    __builtin_amdgcn_sched_barrier(0);   // asked for before the products of the stage, not among them
  };
  auto filled = [] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  const int wm = (wave >> 1) * 32 * WM, wc = (wave & 1) * 32 * WC;   // of RW x 2 waves
  i32x16 acc[WM][WC];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WC; ++j) acc[i][j] = 0;
  auto work = [&](const Stage& st) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < KB / 32; ++k) {
      i32x4 x[WM], t[WC];
#pragma unroll
      for (int i = 0; i < WM; ++i) x[i] = *reinterpret_cast<const i32x4*>(st.x + code_at<KB>(wm + 32 * i + col, 2 * k + half));
#pragma unroll
      for (int j = 0; j < WC; ++j) t[j] = *reinterpret_cast<const i32x4*>(st.t + code_at<KB>(wc + 32 * j + col, 2 * k + half));
#pragma unroll
      for (int j = 0; j < WC; ++j)
#pragma unroll
        for (int i = 0; i < WM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[i], t[j], acc[i][j], 0, 0, 0);
    }
    // one step's operands are read among the products of the step before
    if (WM * WC > 1) {
      __builtin_amdgcn_sched_group_barrier(0x100, WM + WC, 0);
#pragma unroll
      for (int k = 1; k < KB / 32; ++k) {
#pragma unroll
        for (int i = 0; i < WM + WC; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, WM * WC - WM - WC, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, WM * WC, 0);
    }
  };
  const int stages = (int)(a.pitch / KB);
  fill(s_a, 0);
  filled();
  int k = 0;
  for (; k + 2 <= stages; k += 2) {
    fill(s_b, (int64_t)(k + 1) * KB);
    work(s_a);
    filled();
    if (k + 2 < stages) fill(s_a, (int64_t)(k + 2) * KB);
    work(s_b);
    filled();
  }
  if (k < stages) {
    work(s_a);
    __syncthreads();
  }
  // A wave's 32 x 32 blocks: to rows of 4 adjacent values per lane by way of LDS (8 x 128 bytes per store instruction), where the
  // output allows it.
  float* turn = reinterpret_cast<float*>(s_a.x) + wave * (32 * 40);
  static_assert(sizeof(s_a) >= 2 * RW * 32 * 40 * 4 || WM * WC == 1, "room to turn a block per wave");
#pragma unroll
  for (int i = 0; i < WM; ++i) {
    float sx[16], rb[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t row = min(m0 + wm + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3), a.m - 1);
      sx[r] = a.sx[row];
      rb[r] = a.rb ? a.rb[row] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < WC; ++j) {
      __builtin_amdgcn_sched_barrier(0);   // block by block: the next one's scales would take the registers of its sums
      const int64_t item = c0 + wc + 32 * j + col, safe = min(item, a.c - 1);
      const float st = a.st[safe], cb = a.cb ? a.cb[safe] : 0.f;
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = ((float)acc[i][j][r] * sx[r]) * st + (rb[r] + cb);
      if (vec && WM * WC > 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) turn[(8 * (r >> 2) + 4 * half + (r & 3)) * 40 + col] = v[r];
        __builtin_amdgcn_wave_barrier();
        const int64_t c4 = c0 + wc + 32 * j + 4 * (lane & 7);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int in = 8 * q + (lane >> 3);
          const int64_t row = m0 + wm + 32 * i + in;
          const float4 f = *reinterpret_cast<const float4*>(turn + in * 40 + 4 * (lane & 7));
          if (row < a.m && c4 < a.c) {   // c is a multiple of 4 here
            typedef E E4 __attribute__((ext_vector_type(4)));
            E4 o;
            o[0] = (E)f.x;
            o[1] = (E)f.y;
            o[2] = (E)f.z;
            o[3] = (E)f.w;
            *reinterpret_cast<E4*>(reinterpret_cast<E*>(a.out) + row * a.out_stride + c4) = o;
          }
        }
        __builtin_amdgcn_wave_barrier();
      } else if (item < a.c) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t row = m0 + wm + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
          if (row < a.m) reinterpret_cast<E*>(a.out)[row * a.out_stride + item] = (E)v[r];
        }
      }
    }
  }
}

// ---- many rows of up to 128 codes ----------------------------------------------------------------------------------------------
// The output is all there is to do: 4 bytes a value against 128 codes.  Its rows start anywhere in a line, and tiles cut at whole columns
// wrote every 128-byte line that two of them share in parts (16,000 x 16,980 fp32: 370 us, 235 with c = 16,960, whose rows are whole
// lines).  So a tile computes 256 columns (32 x 256 per wave) and writes, row by row, the 224 that begin with its first whole line; the
// values go through LDS in a ring of two 32-column blocks, from which each line is taken as soon as its second block is there.  A line is 32
// values: 128 bytes in fp32; 16-bit outputs are written in half lines, and values one by one where rows start between groups of four.
constexpr int kWideRows = 128, kWideCols = 256, kWideStep = 224;

template <int P>
__device__ __forceinline__ int wide_at(int row, int chunk) {
  return code_at<P>(row, chunk);
}

template <class E, int P, int VEC>
__global__ void __launch_bounds__(256, 2) int8_scores_wide_kernel(Scores a, int64_t c_tiles, int64_t tiles) {
  constexpr int kPitch = 72;      // of the ring, in floats: the two halves of a wave write different banks
  constexpr int kCodes = (kWideRows + kWideCols) * P, kRing = 4 * 32 * kPitch * 4;
  __shared__ __attribute__((aligned(16))) char s_mem[kCodes > kRing ? kCodes : kRing];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int64_t share = (tiles + 7) / 8, tile = (int64_t)(blockIdx.x % 8) * share + blockIdx.x / 8;   // neighbours on one XCD
  if (tile >= tiles) return;
  const int64_t m0 = tile / c_tiles * kWideRows, c0 = tile % c_tiles * kWideStep;
  const int mrows = (int)min((int64_t)kWideRows, a.m - m0), crows = (int)min((int64_t)kWideCols, a.c - c0);
  char *s_x = s_mem, *s_t = s_mem + kWideRows * P;
  constexpr int kPer = 1024 / P;     // rows of one fill
  const int frow = lane / (P / 16);
#pragma unroll
  for (int i = 0; i < kWideRows / kPer / 4; ++i) {
    const int r = (i * 4 + wave) * kPer + frow, chunk = (wide_at<P>(r, lane % (P / 16)) >> 4) % (P / 16);
    __builtin_amdgcn_global_load_lds((gptr_t)(a.qx + (m0 + min(r, mrows - 1)) * P + chunk * 16), (lptr_t)(s_x + (i * 4 + wave) * 1024), 16, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kWideCols / kPer / 4; ++i) {
    const int r = (i * 4 + wave) * kPer + frow, chunk = (wide_at<P>(r, lane % (P / 16)) >> 4) % (P / 16);
    __builtin_amdgcn_global_load_lds((gptr_t)(a.qt + (c0 + min(r, crows - 1)) * P + chunk * 16), (lptr_t)(s_t + (i * 4 + wave) * 1024), 16, 0, 0);
  }
  const int64_t r0 = m0 + wave * 32;
  float sx[16], rb[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t row = min(r0 + 8 * (r >> 2) + 4 * half + (r & 3), a.m - 1);
    sx[r] = a.sx[row];
    rb[r] = a.rb ? a.rb[row] : 0.f;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  i32x16 acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0;
#pragma unroll
  for (int k = 0; k < P / 32; ++k) {
    const i32x4 x = *reinterpret_cast<const i32x4*>(s_x + wide_at<P>(wave * 32 + col, 2 * k + half));
#pragma unroll
    for (int j = 0; j < 8; ++j)
      acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x, *reinterpret_cast<const i32x4*>(s_t + wide_at<P>(32 * j + col, 2 * k + half)), acc[j], 0, 0, 0);
  }
  __syncthreads();
  float* ring = reinterpret_cast<float*>(s_mem) + wave * (32 * kPitch);
  const uint32_t phase = (uint32_t)((uintptr_t)a.out / sizeof(E) + c0);      // of a row's first value, with its row's offset, mod 32
  constexpr int kLanes = 32 / VEC, kRowsPer = 64 / kLanes, kTurns = 32 / kRowsPer;
  const int in = lane / kLanes, e0 = lane % kLanes * VEC;
  auto emit = [&](int line) __attribute__((always_inline)) {
#pragma unroll 4
    for (int q = 0; q < kTurns; ++q) {
      const int r = kRowsPer * q + in;
      const int64_t row = r0 + r;
      const int first = (int)(-(phase + (uint32_t)row * (uint32_t)a.out_stride) & 31);   // columns before the first whole line
      const int x = first + 32 * line + e0;
      if (row < a.m && x >= 0 && c0 + x < a.c) {
        E* dst = reinterpret_cast<E*>(a.out) + row * a.out_stride + c0 + x;
        if constexpr (VEC == 4) {
          const float4 f = *reinterpret_cast<const float4*>(ring + r * kPitch + (x & 63));
          typedef E E4 __attribute__((ext_vector_type(4)));
          E4 o;
          o[0] = (E)f.x;
          o[1] = (E)f.y;
          o[2] = (E)f.z;
          o[3] = (E)f.w;
          *reinterpret_cast<E4*>(dst) = o;
        } else {
          *dst = (E)ring[r * kPitch + (x & 63)];
        }
      }
    }
  };
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    __builtin_amdgcn_sched_barrier(0);   // block by block: the next one's scales would take the registers of its sums
    const int64_t item = min(c0 + 32 * j + col, a.c - 1);
    const float st = a.st[item], cb = a.cb ? a.cb[item] : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      ring[(8 * (r >> 2) + 4 * half + (r & 3)) * kPitch + (j & 1) * 32 + col] = ((float)acc[j][r] * sx[r]) * st + (rb[r] + cb);
    __builtin_amdgcn_wave_barrier();
    if (j == 0) {
      if (c0 == 0) emit(-1);
    } else {
      emit(j - 1);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- up to 32 rows: the table is read once, straight into the operands -------------------------------------------------------------
// Bound by the table's bytes: 1M x 128 codes 26 us, 5.1 TB/s where the last-level cache holds them, 33 from memory; with four blocks of 32
// items a wave instead of two it was 35 (half the waves in flight).
// A wave takes 32 items at a time, twice (8 reads of 1 KB in flight for rows of 128 codes), against all rows, which it holds.
// FUSED: the rows come as floating point values, and every workgroup codes them for itself (m k <= kFused values) instead of waiting
// for a launch that does it once.
constexpr int kFused = 4096;

struct FloatRows {
  const void* x;
  int64_t stride, k;
  int vec;
};

constexpr int kItems = 2;   // blocks of 32 items of a wave
template <class E, class X, bool FUSED>
__global__ void __launch_bounds__(256) int8_scores_few_kernel(Scores a, FloatRows f) {
  __shared__ __attribute__((aligned(16))) int8_t s_q[FUSED ? kFused : 16];
  __shared__ float s_sx[32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
  const int8_t* qx = a.qx;
  const float* sx = a.sx;
  // the table's first 128 codes are asked for before anything else
  const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * (32 * kItems);
  const int8_t* t[kItems];
  i32x4 ahead[kItems][4];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    t[j] = a.qt + min(first + 32 * j + col, a.c - 1) * a.pitch + half * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < 2 || a.pitch > 64) ahead[j][k] = *reinterpret_cast<const i32x4*>(t[j] + 32 * k);
  }
  if constexpr (FUSED) {
    for (int r = wave; r < a.m; r += 4) {
      const X* src = reinterpret_cast<const X*>(f.x) + r * f.stride;
      float v[8], top = 0.f, sum2 = 0.f;
      bool finite = true;
      for (int64_t c0 = 8 * lane; c0 < a.pitch; c0 += 512) {
        load8(src, c0, f.k, f.vec != 0, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          finite = finite && fabsf(v[e]) < INFINITY;
          top = fmaxf(top, fabsf(v[e]));
        }
      }
      int ok = finite;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor(top, o));
        ok &= __shfl_xor(ok, o);
      }
      const Coder c = coder_for(top, ok != 0, sum2, 0);
      for (int64_t c0 = 8 * lane; c0 < a.pitch; c0 += 512) {
        if (a.pitch > 512) load8(src, c0, f.k, f.vec != 0, v);
        *reinterpret_cast<uint64_t*>(s_q + r * a.pitch + c0) = codes8(v, c);
      }
      if (lane == 0) s_sx[r] = c.scale;
    }
    __syncthreads();
    qx = s_q;
    sx = s_sx;
  }
  const int8_t* x = qx + min((int64_t)col, a.m - 1) * a.pitch + half * 16;
  if (first >= a.c) return;
  i32x16 acc[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) acc[j] = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < 2 || a.pitch > 64) {
      const i32x4 xk = *reinterpret_cast<const i32x4*>(x + 32 * k);
#pragma unroll
      for (int j = 0; j < kItems; ++j) acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xk, ahead[j][k], acc[j], 0, 0, 0);
    }
  for (int64_t k0 = 128; k0 < a.pitch; k0 += 64) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const i32x4 xk = *reinterpret_cast<const i32x4*>(x + k0 + 32 * k);
#pragma unroll
      for (int j = 0; j < kItems; ++j) acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xk, *reinterpret_cast<const i32x4*>(t[j] + k0 + 32 * k), acc[j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t item = first + 32 * j + col;
    if (item >= a.c) continue;
    const float st = a.st[item], cb = a.cb ? a.cb[item] : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 8 * (r >> 2) + 4 * half + (r & 3);
      if (row < a.m) reinterpret_cast<E*>(a.out)[row * a.out_stride + item] = (E)(((float)acc[j][r] * sx[row]) * st + (a.rb ? a.rb[row] + cb : cb));
    }
  }
}

// A launch holds fewer than 2^32 work items: this many workgroups of 256 at most, longer calls in pieces.
constexpr int64_t kMostBlocks = 1LL << 23;

template <class E, int LR, bool ONE>
void launch_quantize(const E* x, int64_t stride, int64_t n, int64_t k, int vec, int normalize, int8_t* q, float* scale, hipStream_t st) {
  constexpr int kRows = 256 / LR;      // of a workgroup
  const int64_t pitch = pitch_of(k);
  for (int64_t at = 0; at < n; at += kMostBlocks * kRows) {
    const int64_t rows = std::min(n - at, kMostBlocks * kRows);
    hipLaunchKernelGGL((quantize_rows_kernel<E, LR, ONE>), dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(256), 0, st, x + at * stride, stride,
                       rows, k, vec, normalize, q + at * pitch, scale + at);
  }
}

template <class E>
int run_quantize(const void* x, int64_t stride, int64_t n, int64_t k, int normalize, int8_t* q, float* scale, hipStream_t st) {
  const E* p = reinterpret_cast<const E*>(x);
  const int vec = (uintptr_t)x % (4 * sizeof(E)) == 0 && stride % 4 == 0;
  const int64_t pitch = pitch_of(k);
  ProfScope ps("quantize_rows_kernel", st);
  if (pitch == 64) launch_quantize<E, 8, true>(p, stride, n, k, vec, normalize, q, scale, st);
  else if (pitch == 128) launch_quantize<E, 16, true>(p, stride, n, k, vec, normalize, q, scale, st);
  else launch_quantize<E, 64, false>(p, stride, n, k, vec, normalize, q, scale, st);
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

template <class E>
int run_dequantize(const int8_t* q, const float* scale, int64_t n, int64_t k, void* out, hipStream_t st) {
  const int64_t groups = (k + 7) / 8, most = kMostBlocks * 256 / groups;     // rows of a piece: at least 131,072
  ProfScope ps("dequantize_rows_kernel", st);
  for (int64_t at = 0; at < n; at += most) {
    const int64_t rows = std::min(n - at, most);
    hipLaunchKernelGGL((dequantize_rows_kernel<E>), dim3((unsigned)((rows * groups + 255) / 256)), dim3(256), 0, st, q + at * pitch_of(k), scale + at,
                       rows, k, groups, reinterpret_cast<E*>(out) + at * k);
  }
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

template <class E, class X, bool FUSED>
int run_few(const Scores& a, const FloatRows& f, hipStream_t st) {
  ProfScope ps("int8_scores_kernel", st);
  hipLaunchKernelGGL((int8_scores_few_kernel<E, X, FUSED>), dim3((unsigned)((a.c + 128 * kItems - 1) / (128 * kItems))), dim3(256), 0, st, a, f);
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

template <class E, int WM, int WC, int RW, int KB>
int run_many(const Scores& a, hipStream_t st) {
  const int64_t mt = (a.m + 32 * WM * RW - 1) / (32 * WM * RW), ct = (a.c + 64 * WC - 1) / (64 * WC);
  NNCF_REQUIRE(mt * ct <= kMostBlocks - 8, "%lld x %lld scores in one call", (long long)a.m, (long long)a.c);      // (of up to 512 threads)
  const int vec = a.c % 4 == 0 && a.out_stride % 4 == 0 && (uintptr_t)a.out % (4 * sizeof(E)) == 0;
  const dim3 grid((unsigned)((mt * ct + 7) / 8 * 8));
  ProfScope ps("int8_scores_kernel", st);
  hipLaunchKernelGGL((int8_scores_kernel<E, WM, WC, RW, KB>), grid, dim3(128 * RW), 0, st, a, mt, mt * ct, vec);
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

template <class E>
int run_scores(Scores a, hipStream_t st) {
  constexpr int64_t kRows = 1LL << 22;      // of a piece: few columns of very many rows are more workgroups than a launch takes
  while (a.m > kRows) {
    Scores piece = a;
    piece.m = kRows;
    const int rc = run_scores<E>(piece, st);
    if (rc) return rc;
    a.qx += kRows * a.pitch;
    a.sx += kRows;
    if (a.rb) a.rb += kRows;
    a.out = reinterpret_cast<E*>(a.out) + kRows * a.out_stride;
    a.m -= kRows;
  }
  if (a.m <= 32) return run_few<E, float, false>(a, FloatRows{}, st);
  const int64_t wide_c = (a.c + kWideStep - 1) / kWideStep, wide = (a.m + kWideRows - 1) / kWideRows * wide_c;
  if (a.pitch <= 128 && wide >= 256) {
    NNCF_REQUIRE(wide <= kMostBlocks - 8, "%lld x %lld scores in one call", (long long)a.m, (long long)a.c);
    const bool vec = a.c % 4 == 0 && a.out_stride % 4 == 0 && (uintptr_t)a.out % (4 * sizeof(E)) == 0;
    const dim3 grid((unsigned)((wide + 7) / 8 * 8));
    ProfScope ps("int8_scores_kernel", st);
    if (a.pitch == 64 && vec)
      hipLaunchKernelGGL((int8_scores_wide_kernel<E, 64, 4>), grid, dim3(256), 0, st, a, wide_c, wide);
    else if (a.pitch == 64)
      hipLaunchKernelGGL((int8_scores_wide_kernel<E, 64, 1>), grid, dim3(256), 0, st, a, wide_c, wide);
    else if (vec)
      hipLaunchKernelGGL((int8_scores_wide_kernel<E, 128, 4>), grid, dim3(256), 0, st, a, wide_c, wide);
    else
      hipLaunchKernelGGL((int8_scores_wide_kernel<E, 128, 1>), grid, dim3(256), 0, st, a, wide_c, wide);
    NNCF_HIP_CHECK(hipGetLastError());
    return NNCF_OK;
  }
  // large tiles once they are enough for every CU
  const int64_t large = (a.m + 255) / 256 * ((a.c + 255) / 256);
  return large >= 256 && a.pitch >= 128 ? run_many<E, 2, 4, 4, 128>(a, st) : run_many<E, 1, 1, 2, 64>(a, st);
}

template <class E>
int run_fused(const Scores& a, const FloatRows& f, int32_t x_dtype, hipStream_t st) {
  if (x_dtype == NNCF_F32) return run_few<E, float, true>(a, f, st);
  if (x_dtype == NNCF_F16) return run_few<E, _Float16, true>(a, f, st);
  return run_few<E, __bf16, true>(a, f, st);
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
  hipStream_t st = as_stream(stream);
  if (dtype == NNCF_F32) return run_dequantize<float>(d_q, d_scale, n, k, d_out, st);
  if (dtype == NNCF_F16) return run_dequantize<_Float16>(d_q, d_scale, n, k, d_out, st);
  return run_dequantize<__bf16>(d_q, d_scale, n, k, d_out, st);
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

extern "C" int32_t nncf_int8_scores_fused(int64_t m, int32_t k) {
  return m > 0 && m <= 32 && k > 0 && k <= nncf::kMaxDepth && m * nncf::pitch_of(k) <= nncf::kFused;
}

extern "C" int nncf_int8_scores_rows(const void* d_x, int64_t x_stride, int32_t x_dtype, int64_t m, const int8_t* d_qt, const float* d_st,
                                     int64_t c, int32_t k, const float* d_row_bias, const float* d_col_bias, void* d_out, int64_t out_stride,
                                     int32_t dtype, void* stream) {
  using namespace nncf;
  NNCF_REQUIRE(nncf_int8_scores_fused(m, k), "%lld rows of %d columns are coded by nncf_quantize_rows first", (long long)m, k);
  NNCF_REQUIRE(c >= 0 && c <= (1LL << 31), "c = %lld out of range", (long long)c);
  NNCF_REQUIRE(known(dtype) && known(x_dtype), "dtype = %d or %d unknown", dtype, x_dtype);
  if (c == 0) return NNCF_OK;
  NNCF_REQUIRE(d_x && d_qt && d_st && d_out, "NULL argument");
  NNCF_REQUIRE(x_stride >= k, "row stride %lld is below k = %d", (long long)x_stride, k);
  NNCF_REQUIRE(((uintptr_t)d_qt & 15) == 0, "codes must be 16-byte aligned");
  NNCF_REQUIRE((uintptr_t)d_x % size_of(x_dtype) == 0 && (uintptr_t)d_out % size_of(dtype) == 0, "a tensor is not aligned to its elements");
  NNCF_REQUIRE(out_stride >= c, "output stride %lld is below c = %lld", (long long)out_stride, (long long)c);
  const Scores a{nullptr, d_qt, nullptr, d_st, d_row_bias, d_col_bias, d_out, m, c, out_stride, pitch_of(k)};
  const FloatRows f{d_x, x_stride, k, (uintptr_t)d_x % (4 * size_of(x_dtype)) == 0 && x_stride % 4 == 0};
  hipStream_t st = as_stream(stream);
  if (dtype == NNCF_F32) return run_fused<float>(a, f, x_dtype, st);
  if (dtype == NNCF_F16) return run_fused<_Float16>(a, f, x_dtype, st);
  return run_fused<__bf16>(a, f, x_dtype, st);
}
