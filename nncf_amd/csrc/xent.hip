// Softmax cross entropy over the whole item table, with its gradients, without the logits.
//
//   z_ij = scale u_i . v_j + bias_j        loss_i = weight_i (log sum_j e^z_ij - z_i,t_i)
//
// One streaming kernel serves both directions.  It holds 32 OWN rows per wave (columns of the matrix instruction), walks over the
// STREAM rows in tiles, and keeps per own row a a reference exponent M_a, l_a = sum_b 2^(y_ab - M_a) and O_a = sum_b 2^(y_ab - M_a)
// x_b (y in base 2), so that n x c values are formed, used and dropped in registers:
//   forward   own = users, stream = items, y = z log2(e):                     the normaliser and the mean item under p
//   backward  own = items, stream = users, y = z log2(e) - lse + log2 |w|:    the columns of p times the user rows, exactly d_table
// (the mean item is d_rows).  Logits are formed twice instead of being stored: 8 n c d operations where 6 are the least.
//
// The TARGET of a row is left out of the forward sums and joined in fp32: with A = log sum_{j != t} e^z_ij, loss = softplus(A - z_t)
// and 1 - p_t = sigmoid(A - z_t) keep their relative accuracy as p_t -> 1, where 1 - p_t by subtraction keeps none; the gradient is
// weight scale (1 - p_t) (mean_{j != t} v_j - v_t), and the backward pass takes -(1 - p_t) for the target's coefficient.
//
// Products of fp32 tables run on the f16 matrix pipe as two planes, x 2^b = hi + lo, with a power of two per ROW that brings its
// largest value into [2^13, 2^14): hi + lo then hold 22 bits of every value within 2^16 of the row's largest and an absolute 2^-38 of
// it below; three products (hi hi, hi lo, lo hi; lo lo is left out) leave about 6e-8 of sum |a b|, as an fp32 sum does.  Fewer bits than fp32
// arithmetic keeps, place by place:
//   - rows whose largest value is below 2^-80 (the power stops at 2^77), and items whose rows are 2^100 smaller than the largest of the
//     call (their 2^-b rides in the exponent beside the reference, and their terms below 2^-36 of the largest leave the normaliser);
//   - where 16 rows of zeros are neighbours, rows below 2^-27 beside them (see xent_prep_kernel);
//   - rows of more than 2^90 may overflow (a product is brought back by one side's power before the other's);
//   - a coefficient 2^(y - M) of an fp32 table is held in two planes: 22 bits down to 2^-24 of the largest of kAside stages, an absolute 2^-34
//     of that one below: at most 2^-22 of it in all that the 4,096 rows of those stages can lose;
//   - a coefficient of a 16-bit table is rounded to the table's type before it meets the rows, as these are: it moves the sums by less than the
//     rounding of the result (8,192 x 16,980 bf16: both 1.7e-3 from the definition, 2.6e-4 apart in d_rows, 9e-5 in d_table).  The targets',
//     the largest terms of their sums, are held in two planes for every type.
// Sums, normalisers and references are fp32.  The reference exponents M are whole numbers, so every rescaling is exact.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "common.h"
#include "devutil.h"

namespace nncf {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr int kOwn = 128;      // own rows of a workgroup: 4 waves x 32
constexpr int kTile = 64;      // stream rows of a stage
constexpr int kAside = 64;    // stages after which a workgroup's sums of rows are put aside
constexpr float kTop = 10.f;   // a new reference puts the largest exponent of a row at <= 2^10 ...
constexpr float kRaise = 15.f; // ... and is taken again once one passes 2^15 (f16 ends at 2^16)

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct F16 {
  typedef _Float16 E;
  typedef f16x8 V;
  static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
struct BF16 {
  typedef __bf16 E;
  typedef bf16x8 V;
  static __device__ __forceinline__ f32x16 mfma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// One side of the product, in the workspace.  img: [rows_pad][NP][DP] 16-bit values; inv = 2^-b (two planes only); h: what is added to
// the exponent when the side streams; kq: the target coefficient of a user row; tgt: its target.
struct Side {
  const char* img;
  const float* inv;
  const float* h;
  const float* kq;
  const float* sgn;
  const int32_t* tgt;
  const float* bias;  // items
  int64_t rows;       // rows of the call
  int64_t rows_pad;   // a multiple of 128
};
// Where a pass over items that are not split puts its results: the gradients themselves (table NULL: Part).
struct Grad {
  void* table;
  float* bias;
  const int32_t* valid;
  float scale;
  int d, mean, vec;
};
struct Part {   // results of the streaming kernel: [splits][own rows_pad]
  float *o, *m, *l;
};

// 16-byte chunks of a row are stored at chunk ^ g(row): a wave's ds_read_b128 of one chunk of 32 rows and its transposing
// ds_read_b64 of 4 chunks of 4 consecutive rows then both meet every bank once.
template <int NP, int DP>
__device__ __forceinline__ int lds_at(int row, int plane, int chunk) {
  if (DP == 128) {
    const int g = ((row & 3) << 2) | ((row >> 2) & 3);
    return row * (NP * 256) + plane * 256 + ((chunk ^ g) << 4);
  } else {
    const int u = (row >> 1) & 7, g = ((u & 1) << 2) | (u >> 1);
    if (NP == 1) return row * 128 + ((chunk ^ g) << 4);
    return row * 256 + ((plane ^ (row & 1)) << 7) + ((chunk ^ g) << 4);
  }
}

// the inverse: byte offset in a tile of the row-major image of what lies in 16-byte slot i of its LDS form
template <int NP, int DP>
__device__ __forceinline__ int image_at(int i) {
  if (DP == 128) {
    const int row = i / (NP * 16), g = ((row & 3) << 2) | ((row >> 2) & 3);
    return (i & ~15) * 16 + (((i & 15) ^ g) << 4);
  } else {
    const int row = i / (NP * 8), u = (row >> 1) & 7, g = ((u & 1) << 2) | (u >> 1);
    const int plane = NP == 1 ? 0 : (i >> 3 & 1) ^ (row & 1);
    return row * (NP * 128) + plane * 128 + (((i & 7) ^ g) << 4);
  }
}

// A stage of stream rows in LDS, and its asynchronous filling: global memory to LDS without a register, 1 KB per wave and instruction.
template <int NP, int DP>
struct __attribute__((aligned(16))) Stage {
  char img[kTile * NP * DP * 2];
  float h[kTile], inv[kTile], sgn[kTile], kq[kTile];
  int32_t tgt[kTile];
};
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

// The slots a wave fills lie a multiple of 16 rows apart, where the order of chunks is the same: one lane offset (two for rows of 512
// bytes) serves them all.
template <int NP, int DP>
struct Filler {
  static constexpr int kRow = NP * DP * 2, kEach = kTile * kRow / 16 / 256, kOff = kRow == 512 ? 2 : 1;
  int off[kOff];
  static __device__ __forceinline__ int slot(int j, int wave) {   // in units of 64 slots
    return kOff == 2 ? (j & 1) + 2 * wave + 8 * (j >> 1) : wave + 4 * j;
  }
  __device__ __forceinline__ Filler(int wave, int lane) {
#pragma unroll
    for (int j = 0; j < kOff; ++j) off[j] = image_at<NP, DP>(slot(j, wave) * 64 + lane);
  }
};

template <int NP, int DP, bool BWD, bool WT>
__device__ __forceinline__ void fill(Stage<NP, DP>& to, const Filler<NP, DP>& f, const Side& str, int64_t row0, int wave, int lane) {
  typedef Filler<NP, DP> F;
#pragma unroll
  for (int j = 0; j < F::kEach; ++j) {
    constexpr int step = F::kOff == 2 ? 16 * F::kRow : 4096;     // bytes of the image between a wave's equal offsets
    const char* src = str.img + row0 * F::kRow + (j / F::kOff) * step;
    __builtin_amdgcn_global_load_lds((gptr_t)(src + f.off[j % F::kOff]), (lptr_t)(to.img + F::slot(j, wave) * 1024), 16, 0, 0);
  }
  if (wave == 0) __builtin_amdgcn_global_load_lds((gptr_t)(str.h + row0 + lane), (lptr_t)to.h, 4, 0, 0);
  if (NP == 2 && wave == 1) __builtin_amdgcn_global_load_lds((gptr_t)(str.inv + row0 + lane), (lptr_t)to.inv, 4, 0, 0);
  if (BWD && wave == 1) __builtin_amdgcn_global_load_lds((gptr_t)(str.kq + row0 + lane), (lptr_t)to.kq, 4, 0, 0);
  if (WT && wave == 2) __builtin_amdgcn_global_load_lds((gptr_t)(str.sgn + row0 + lane), (lptr_t)to.sgn, 4, 0, 0);
  if (BWD && wave == 3) __builtin_amdgcn_global_load_lds((gptr_t)(str.tgt + row0 + lane), (lptr_t)to.tgt, 4, 0, 0);
}
__device__ __forceinline__ void filled() {   // this wave's part has arrived, and everyone's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// sum + kept += x, with what the addition rounds away in kept (two-sum: any signs and sizes)
__device__ __forceinline__ void add_kept(float& sum, float& kept, float x) {
  const float s = sum + x, b = s - sum;
  kept += (sum - (s - b)) + (x - b);
  sum = s;
}

template <class T, int NP, int DP>
__device__ __forceinline__ typename T::V read_rows(const char* lds, int row, int plane, int chunk) {
  return *reinterpret_cast<const typename T::V*>(lds + lds_at<NP, DP>(row, plane, chunk));
}
// column (32 dt + lane % 32) of rows r0 + 0..3 and r0 + 8 + 0..3, r0 = 16 s + 4 (lane / 32): the k order in which the accumulator
// of the first product holds its rows, so that it is the second product's operand as it stands
template <class T, int NP, int DP>
__device__ __forceinline__ typename T::V read_cols(const char* lds, int plane, int base, int dt, int lane) {
  typedef __attribute__((address_space(3))) s16x4_t* lp_t;
  const int t = lane & 15, half = lane >> 5, sub = (lane >> 4) & 1;
  const int row = base + 4 * half + (t >> 2), chunk = dt * 4 + sub * 2 + ((t & 3) >> 1), off = (t & 1) * 8;
  const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp_t)(const_cast<char*>(lds) + lds_at<NP, DP>(row, plane, chunk) + off));
  const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp_t)(const_cast<char*>(lds) + lds_at<NP, DP>(row + 8, plane, chunk) + off));
  typedef short s16x8_t __attribute__((__vector_size__(8 * sizeof(short))));
  const s16x8_t c = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(typename T::V, c);
}

// What bounds it (measured): 4,096 x 1M x 128 fp32 takes 5.63 + 5.57 ms (best of 40: 5.57 + 5.54; on another box 5.36 + 5.33), 1.12 PFLOP/s of
// issued products: the matrix pipe is busy in 63% and 66% of its cycles, the vector ALU in 50%, at the 1.73 GHz that the card holds under them.
// 8,192 x 16,980 x 100 bf16: forward 85 us (pipe 45%, vector ALU 50%: as many exponentials and conversions as products), backward 106 (pipe 37%,
// vector ALU 45%: the target branch, and its popular items' workgroups).
// Two workgroups of four waves on a CU, 250 registers a wave; a third does not fit.  32 x 32 x 16 products, because their accumulator
// layout is the next product's operand layout (read_cols): the coefficients never leave the registers.  LDS reads meet no bank conflict.
// Tried and left: results of a line of equal pieces instead of splits (5.5 -> 5.9 ms, 8,192: 135 -> 160 us), workgroups of two waves that
// need no splits (512 x 17,000: 77 -> 95 us), references at the top of f16's range (kTop 13 and 15: 8,192 x 16,980 204 -> 209 and 217 us).
//
// The streaming kernel.  DU: the columns in use, rounded up (of rows DP wide in their image).  BWD: own rows are items.  WT: row weights of
// either sign.  MEAN: the O sums are wanted.
template <class T, int NP, int DP, int DU, bool BWD, bool WT, bool MEAN>
__global__ void __launch_bounds__(256, 2) xent_stream_kernel(Side own, Side str, Part part, Grad grad, float scale2, int stages, int stages_per_split) {
  typedef typename T::V V;
  constexpr int kRow = NP * DP * 2;             // bytes of an image row
  constexpr int KS = (DU + 15) / 16, DT = (DU + 31) / 32, RT = NP == 2 || WT ? 1 : 2;   // sub-tiles of 32 stream rows worked on together
  __shared__ Stage<NP, DP> s_a, s_b;            // two objects, so that a read of one does not wait for the filling of the other
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int split = blockIdx.x;
  const int64_t own0 = (int64_t)blockIdx.y * kOwn + wave * 32, own_row = own0 + col;

  V of[NP][KS];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int k = 0; k < KS; ++k)
      of[p][k] = *reinterpret_cast<const V*>(own.img + own_row * kRow + p * (DP * 2) + (2 * k + half) * 16);
  const float c = NP == 2 ? scale2 * own.inv[own_row] : scale2;
  const bool inside = own_row < own.rows;
  const int32_t own_id = (int32_t)own_row;
  const int32_t own_tgt = BWD ? -1 : own.tgt[own_row];
  const float add = BWD && inside && own.bias ? own.bias[own_row] * kLog2e : 0.f;

  f32x16 o[MEAN ? DT : 1];
#pragma unroll
  for (int d = 0; d < (MEAN ? DT : 1); ++d) o[d] = 0.f;
  float m = 0.f, l = 0.f, lc = 0.f;             // the sum is l + lc
  bool seen = false;

  auto work = [&](const Stage<NP, DP>& st, int64_t row0) __attribute__((always_inline)) {
    const char* s_img = st.img;
    const float *s_h = st.h, *s_inv = st.inv, *s_sgn = st.sgn, *s_kq = st.kq;
    const int32_t* s_tgt = st.tgt;
#pragma unroll 1
    for (int r0 = 0; r0 < kTile / 32; r0 += RT) {
      f32x16 s[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const V a = read_rows<T, NP, DP>(s_img, 32 * (r0 + r) + col, 0, 2 * k + half);
          s[r] = T::mfma(a, of[0][k], s[r]);
          if (NP == 2) {
            const V b = read_rows<T, NP, DP>(s_img, 32 * (r0 + r) + col, 1, 2 * k + half);
            s[r] = T::mfma(a, of[NP - 1][k], s[r]);
            s[r] = T::mfma(b, of[0][k], s[r]);
          }
        }
      // Operands three steps (NP == 1: four or eight reads) ahead of their products: left alone, the compiler read, waited and multiplied one
      // by one (4,096 x 1M fp32, forward: 5.55 ms; so 5.47, on one box).
      constexpr int kAhead = NP == 2 ? 6 : BWD ? 4 : 8, kReads = NP * KS * RT;
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int i = kAhead; i < kReads; i += NP) {
        __builtin_amdgcn_sched_group_barrier(0x008, NP == 2 ? 3 : 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NP, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, NP == 2 ? 9 : kAhead, 0);
      float d[RT][16], iv[NP == 2 ? RT : 1][16];
      const float shift = m - add;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at = 32 * (r0 + r) + 8 * g + 4 * half;
          const float4 h4 = *reinterpret_cast<const float4*>(s_h + at);
          const float hv[4] = {h4.x, h4.y, h4.z, h4.w};
          float4 i4 = make_float4(1.f, 1.f, 1.f, 1.f);
          if (NP == 2) i4 = *reinterpret_cast<const float4*>(s_inv + at);
          const float ivv[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (NP == 2) iv[r][4 * g + e] = ivv[e];
            d[r][4 * g + e] = fmaf(NP == 2 ? s[r][4 * g + e] * ivv[e] : s[r][4 * g + e], c, hv[e] - shift);
          }
        }
      float top = d[0][0];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = r ? 0 : 1; i < 16; ++i) top = fmaxf(top, d[r][i]);
      // targets: a wave-uniform branch, then selects: no lane loads or computes by itself
      const int32_t first = (int32_t)(row0 + 32 * r0);
      uint64_t hit_rows = 0;
      if (!BWD) {
        if (__any((uint32_t)(own_tgt - first) < 32u * RT)) {
          top = -INFINITY;
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (first + 32 * r + 8 * (i >> 2) + 4 * half + (i & 3) == own_tgt) d[r][i] = -INFINITY;
              top = fmaxf(top, d[r][i]);
            }
        }
      } else {
        // its own products, below; here a target's place holds nothing, and its size counts for the reference
        hit_rows = __ballot((uint32_t)(s_tgt[32 * r0 + (RT == 2 ? lane : col)] - (int32_t)own0) < 32u);
        if (hit_rows) {
          top = -INFINITY;
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if (!(hit_rows >> (32 * r + 8 * g) & 0xff)) continue;
              const int at = 32 * (r0 + r) + 8 * g + 4 * half;
              const int4 t4 = *reinterpret_cast<const int4*>(s_tgt + at);
              const float4 k4 = *reinterpret_cast<const float4*>(s_kq + at);
              const int32_t tv[4] = {t4.x, t4.y, t4.z, t4.w};
              const float kv[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float& x = d[r][4 * g + e];
                const bool is = tv[e] == own_id;
                // 2^exponent is at or above the coefficient; one that is 0 asks for nothing
                const float need = kv[e] == 0.f ? -INFINITY : (float)__builtin_amdgcn_frexp_expf(kv[e]) - m;
                top = fmaxf(top, is ? need : -INFINITY);
                x = is ? -INFINITY : x;
              }
            }
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, d[r][i]);
        }
      }
      if (__any(top > kRaise || (!seen && top > -INFINITY))) {
        top = fmaxf(top, __shfl_xor(top, 32));   // both halves of a column keep one reference
        const bool move = top > kRaise || (!seen && top > -INFINITY);
        const float by = move ? ceilf(top) - kTop : 0.f;
        const float f = seen ? __builtin_amdgcn_exp2f(-by) : 1.f;
        seen = seen || move;
        m += by;
        l *= f;
        lc *= f;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 16; ++i) d[r][i] -= by;
        if (MEAN) {
#pragma unroll
          for (int t = 0; t < DT; ++t) o[t] *= f;
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) d[r][i] = __builtin_amdgcn_exp2f(d[r][i]);
      if (WT) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 w4 = *reinterpret_cast<const float4*>(s_sgn + 32 * (r0 + r) + 8 * g + 4 * half);
            d[r][4 * g] *= w4.x;
            d[r][4 * g + 1] *= w4.y;
            d[r][4 * g + 2] *= w4.z;
            d[r][4 * g + 3] *= w4.w;
          }
      }
      // The normaliser: a sub-tile's terms in four short sums, and those into a sum that keeps what its rounding loses.  One running fp32 sum
      // of a million equal terms was off by up to 7e-4.
      {
        float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            // 2^b = 1 / 2^-b, by its exponent
            if (NP == 2) t[i & 3] = fmaf(d[r][i], __builtin_bit_cast(float, 0x7F000000 - __builtin_bit_cast(int, iv[r][i])), t[i & 3]);
            else t[i & 3] += d[r][i];
          }
        add_kept(l, lc, (t[0] + t[1]) + (t[2] + t[3]));
      }
      if (MEAN) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            V hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              hi[e] = (typename T::E)d[r][8 * q + e];
              if (NP == 2) lo[e] = (typename T::E)(d[r][8 * q + e] - (float)hi[e]);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
              const V a = read_cols<T, NP, DP>(s_img, 0, 32 * (r0 + r) + 16 * q, t, lane);
              o[t] = T::mfma(a, hi, o[t]);
              if (NP == 2) {
                const V b = read_cols<T, NP, DP>(s_img, NP - 1, 32 * (r0 + r) + 16 * q, t, lane);
                o[t] = T::mfma(a, lo, o[t]);
                o[t] = T::mfma(b, hi, o[t]);
              }
            }
          }
        if (BWD && hit_rows) {   // targets, 16 stream rows at a time: the largest terms of their sums, so two planes for every type
#pragma unroll 1
          for (int w = 0; w < 2 * RT; ++w) {
            if (!(hit_rows >> (16 * w) & 0xffff)) continue;
            V hi, lo;
            float sum = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int at = 32 * r0 + 16 * w + 8 * g + 4 * half;
              const int4 t4 = *reinterpret_cast<const int4*>(s_tgt + at);
              const float4 k4 = *reinterpret_cast<const float4*>(s_kq + at);
              float4 i4 = make_float4(1.f, 1.f, 1.f, 1.f);
              if (NP == 2) i4 = *reinterpret_cast<const float4*>(s_inv + at);
              const int32_t tv[4] = {t4.x, t4.y, t4.z, t4.w};
              const float kv[4] = {k4.x, k4.y, k4.z, k4.w}, ivv[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = tv[e] == own_id ? -ldexpf(kv[e], (int)-m) : 0.f;
                hi[4 * g + e] = (typename T::E)v;
                lo[4 * g + e] = (typename T::E)(v - (float)hi[4 * g + e]);
                sum += NP == 2 ? v * __builtin_bit_cast(float, 0x7F000000 - __builtin_bit_cast(int, ivv[e])) : v;
              }
            }
            add_kept(l, lc, sum);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
              const V a = read_cols<T, NP, DP>(s_img, 0, 32 * r0 + 16 * w, t, lane);
              o[t] = T::mfma(a, hi, o[t]);
              o[t] = T::mfma(a, lo, o[t]);
              if (NP == 2) o[t] = T::mfma(read_cols<T, NP, DP>(s_img, NP - 1, 32 * r0 + 16 * w, t, lane), hi, o[t]);
            }
          }
        }
      }
    }
  };
  const int t0 = split * stages_per_split, t1 = min(stages, t0 + stages_per_split);
  // The sums of kAside stages are put aside in memory, beside their reference, by the lanes that hold them, and begun anew.  Running on, O was
  // one fp32 chain of the matrix pipe (equal terms, 8,192 rows x 1M fp32: the mean item off by 3e-4), and coefficients of 16 bits that are
  // 2^35 below the largest of the whole stream, not of kAside stages, were lost.
  const int64_t aside0 = (int64_t)split * own.rows_pad + own0;      // of the wave
  auto lane_again = [&] {                                           // for addresses that are formed anew each time: not kept in the loop
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  auto join_aside = [&](bool first, auto&& take) __attribute__((always_inline)) {
    const int x = lane_again();
    float* const at_m = part.m + aside0 + (x & 31);                 // both halves of a column, the same values
    float* const at_l = part.l + aside0 + (x & 31);
    float* const at_o = part.o + aside0 * DP + ((x & 31) * DP + 4 * (x >> 5));
    const float before = first ? -INFINITY : *at_m, top = seen ? fmaxf(before, m) : before;
    // nothing seen on either side: zeros, or NaN, which stays
    const float fb = top > -INFINITY ? __builtin_amdgcn_exp2f(before - top) : 1.f, f = seen ? __builtin_amdgcn_exp2f(m - top) : 1.f;
    l += lc;
    l += __shfl_xor(l, 32);
    l *= f;
    if (!first) l = fmaf(fb, *at_l, l);
    if (MEAN) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float4* p = reinterpret_cast<float4*>(at_o + 32 * t + 8 * g);
          float4 v = make_float4(o[t][4 * g] * f, o[t][4 * g + 1] * f, o[t][4 * g + 2] * f, o[t][4 * g + 3] * f);
          if (!first) v = fma4(fb, *p, v);
          take(t, g, v, p);
          if (g & 1) __builtin_amdgcn_sched_barrier(0);             // two reads in flight: more would take registers from the loop
        }
    }
    m = top;
    return std::pair<float*, float*>(at_m, at_l);
  };
  auto put_aside = [&](bool first) {
    const auto at = join_aside(first, [](int, int, float4 v, float4* p) { *p = v; });
    *at.first = m;
    *at.second = l;
#pragma unroll
    for (int t = 0; t < (MEAN ? DT : 1); ++t) o[t] = 0.f;
    m = l = lc = 0.f;
    seen = false;
  };
  if (t0 < t1) {
    const Filler<NP, DP> filler(wave, lane);
    fill<NP, DP, BWD, WT>(s_a, filler, str, (int64_t)t0 * kTile, wave, lane);
    filled();
    for (int tile = t0; tile < t1; tile += 2) {
      if (tile + 1 < t1) fill<NP, DP, BWD, WT>(s_b, filler, str, (int64_t)(tile + 1) * kTile, wave, lane);
      work(s_a, (int64_t)tile * kTile);
      filled();
      if (tile + 1 >= t1) break;
      if (tile + 2 < t1) fill<NP, DP, BWD, WT>(s_a, filler, str, (int64_t)(tile + 2) * kTile, wave, lane);
      work(s_b, (int64_t)(tile + 1) * kTile);
      filled();
      if ((tile + 2 - t0) % kAside == 0 && tile + 2 < t1) put_aside(tile + 2 - t0 == kAside);
    }
  }
  if (t1 - t0 > kAside) {
    join_aside(false, [&](int t, int g, float4 v, float4*) {
      o[t][4 * g] = v.x;
      o[t][4 * g + 1] = v.y;
      o[t][4 * g + 2] = v.z;
      o[t][4 * g + 3] = v.w;
    });
    seen = m > -INFINITY;
    if (!seen) m = 0.f;
  } else {
    l += lc;
    l += __shfl_xor(l, 32);
  }
  const int64_t row = own0 + (lane_again() & 31);
  if (BWD && grad.table) {
    if (row >= own.rows) return;
    typedef typename std::conditional<NP == 2, float, typename T::E>::type E;
    typedef E E4 __attribute__((ext_vector_type(4)));
    const bool none = (!seen && l == l) || add == -INFINITY;   // a column of nothing but NaN stays that
    const float share = grad.mean ? 1.f / (float)max(1, *grad.valid) : 1.f, k = grad.scale * share;
    const int up = none ? 0 : (int)m;
    E* dst = reinterpret_cast<E*>(grad.table) + row * grad.d;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c0 = 32 * t + 8 * g + 4 * half;
        E4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (E)(none ? 0.f : ldexpf(o[t][4 * g + e], up) * k);
        if (grad.vec) {
          if (c0 < grad.d) *reinterpret_cast<E4*>(dst + c0) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c0 + e < grad.d) dst[c0 + e] = v[e];
        }
      }
    if (half == 0 && grad.bias) grad.bias[row] = none ? 0.f : ldexpf(l, up) * share;
    return;
  }
  const int64_t at = (int64_t)split * own.rows_pad + row;
  if (half == 0) {
    part.m[at] = seen ? m : -INFINITY;   // (a column of nothing but NaN too: its l says so)
    part.l[at] = l;
  }
  if (MEAN) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(part.o + at * DP + 32 * t + 8 * g + 4 * half) =
            make_float4(o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]);
  }
  }

// ---- images ------------------------------------------------------------------------------------------------------------------
template <class E>
__device__ __forceinline__ void load8(const E* row, int c0, int d, bool vec, float* x) {
  if (vec) {   // rows start on a multiple of 4 elements
    typedef E E4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = c0 + 4 * q;
      if (at + 4 <= d) {
        const E4 v = *reinterpret_cast<const E4*>(row + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * q + e] = (float)v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * q + e] = at + e < d ? (float)row[at + e] : 0.f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = c0 + e < d ? (float)row[c0 + e] : 0.f;
  }
}

struct PrepSide {
  const void* src;
  int64_t stride, rows, rows_pad;
  const int32_t* keep;    // users: rows with keep < 0 are not used
  const float* bias;      // items: rows at -inf are not used
  char* img;
  float *inv, *h, *sgn;
  int32_t* tgt;
  int vec;
};

// One row per DP / 8 lanes (8 columns each): the row in one or two 16-bit planes, its scale, and for an item what streams with it.
template <class E, int NP, int DP>
__global__ void __launch_bounds__(256) xent_prep_kernel(PrepSide a, PrepSide b, int64_t a_blocks, int d, int32_t* valid, int n) {
  constexpr int LR = DP / 8;
  if (blockIdx.x == gridDim.x - 1) {   // rows that have a target, by one workgroup
    __shared__ int s_cnt[4];
    int cnt = 0;
    for (int i = threadIdx.x; i < n; i += 256) cnt += a.keep[i] >= 0;
    cnt = wave_sum_i(cnt);
    if ((threadIdx.x & 63) == 0) s_cnt[threadIdx.x >> 6] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) *valid = s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3];
    return;
  }
  const bool first = (int64_t)blockIdx.x < a_blocks;
  const PrepSide s = first ? a : b;
  const int64_t row = ((int64_t)blockIdx.x - (first ? 0 : a_blocks)) * (256 / LR) + threadIdx.x / LR;
  if (row >= s.rows_pad) return;      // (of whole workgroups: rows_pad is a multiple of 128)
  const int q = threadIdx.x % LR;
  bool use = row < s.rows;
  float bias = 0.f;
  if (use && s.keep) use = s.keep[row] >= 0;
  if (use && s.bias) {
    bias = s.bias[row];
    use = !(bias == -INFINITY);
  }
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (use) load8(reinterpret_cast<const E*>(s.src) + row * s.stride, 8 * q, d, s.vec != 0, x);
  float inv = 1.f, shift = 0.f;
  char* out = s.img + row * (NP * DP * 2) + q * 16;
  if constexpr (NP == 2) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
    for (int o = LR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    // 2^15 2^77 and 2^23 rows stay below 2^127 in l
    const bool scaled = top > 0.f && top < INFINITY;
    int b = scaled ? min(77, 14 - __builtin_amdgcn_frexp_expf(top)) : 0;
    // A row of zeros adds nothing to O, and its coefficient should not set the reference of rows that do: it goes as one of the smallest row of
    // its workgroup, or of 2^-27 among nothing but zeros.
    __shared__ int s_b[4];
    int most = scaled ? b : INT32_MIN;
#pragma unroll
    for (int o = LR; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
    if ((threadIdx.x & 63) == 0) s_b[threadIdx.x >> 6] = most;
    __syncthreads();
    most = max(max(s_b[0], s_b[1]), max(s_b[2], s_b[3]));
    if (top == 0.f) b = most > INT32_MIN ? most : 40;
    inv = ldexpf(1.f, -b);
    shift = (float)b;
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = ldexpf(x[e], b);
      hi[e] = (_Float16)v;
      lo[e] = (_Float16)(v - (float)hi[e]);
    }
    *reinterpret_cast<f16x8*>(out) = hi;
    *reinterpret_cast<f16x8*>(out + DP * 2) = lo;
  } else {
    typedef E E8 __attribute__((ext_vector_type(8)));
    E8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (E)x[e];
    *reinterpret_cast<E8*>(out) = v;
  }
  if (q == 0) {
    if (NP == 2) s.inv[row] = inv;
    if (s.sgn) {
      s.sgn[row] = 1.f;
      s.tgt[row] = row < s.rows ? s.keep[row] : -1;
    }
    s.h[row] = use && !s.keep ? bias * kLog2e - shift : -INFINITY;   // users: written once their normaliser is known
  }
}

// ---- joining the splits ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int rows_with_target(const int32_t* target, int n) {
  int k = 0;
  for (int i = 0; i < n; ++i) k += target[i] >= 0;
  return k;
}

struct RowsOut {
  const void *rows, *table;
  int64_t rows_stride, table_stride;
  const float *bias, *weight;
  const int32_t *target, *valid;
  float *loss_rows, *lse, *h, *kq, *sgn;
  const float* inv;
  void* d_rows;
  float scale;
  int64_t n, c, rows_pad;
  int d, mean, splits;
};

// W waves per row (1 or 4): joins its splits, adds the target, writes loss, lse, d_rows and what the row streams with in the backward
// pass.  Reading a row's results of 128 splits in turn was a chain of trips to memory (15 us for any n): past 8 splits four waves share
// them, eight reads in flight each.
template <class E, int NP, int DP, bool MEAN, int W>
__global__ void __launch_bounds__(256) xent_rows_kernel(RowsOut a, Part part) {
  __shared__ float s_o[W][DP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part_of = wave % W;
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W;
  if (W == 1 && row >= a.n) return;
  const int32_t t = a.target[row];
  const bool has = t >= 0, bad = has && t >= a.c;
  const E* u = reinterpret_cast<const E*>(a.rows) + row * a.rows_stride;
  const E* v = reinterpret_cast<const E*>(a.table) + (int64_t)(has && !bad ? t : 0) * a.table_stride;
  float top = -INFINITY;
  for (int k = lane; k < a.splits; k += 64) top = fmaxf(top, part.m[(int64_t)k * a.rows_pad + row]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  const bool some = top > -INFINITY;
  if (has) {
    for (int k = lane; k < a.splits; k += 64) {
      const int64_t at = (int64_t)k * a.rows_pad + row;
      const float mk = part.m[at], lk = part.l[at];
      if (mk > -INFINITY || lk != lk) l += mk > -INFINITY ? lk * __builtin_amdgcn_exp2f(mk - top) : lk;
    }
    l = wave_sum(l);
    if (MEAN) {
#pragma unroll 8
      for (int k = part_of; k < a.splits; k += W) {
        const int64_t at = (int64_t)k * a.rows_pad + row;
        const float mk = part.m[at], f = mk > -INFINITY ? __builtin_amdgcn_exp2f(mk - top) : 0.f;
        o0 = fmaf(part.o[at * DP + lane], f, o0);
        if (DP == 128) o1 = fmaf(part.o[at * DP + 64 + lane], f, o1);
      }
    }
  }
  if (W > 1) {
    s_o[part_of][lane] = o0;
    if (DP == 128) s_o[part_of][DP - 64 + lane] = o1;
    __syncthreads();
    if (part_of) return;
    o0 = (s_o[0][lane] + s_o[1 % W][lane]) + (s_o[2 % W][lane] + s_o[3 % W][lane]);
    if (DP == 128) o1 = (s_o[0][DP - 64 + lane] + s_o[1 % W][DP - 64 + lane]) + (s_o[2 % W][DP - 64 + lane] + s_o[3 % W][DP - 64 + lane]);
  }
  float u0 = 0.f, u1 = 0.f, v0 = 0.f, v1 = 0.f;
  const float beta = has && !bad && a.bias ? a.bias[t] : 0.f;
  const bool out = beta == -INFINITY;     // the target itself is left out: nothing to learn from
  if (has && !bad && !out) {
    if (lane < a.d) { u0 = (float)u[lane]; v0 = (float)v[lane]; }
    if (lane + 64 < a.d) { u1 = (float)u[lane + 64]; v1 = (float)v[lane + 64]; }
  }
  const float zt = out ? -INFINITY : fmaf(a.scale, wave_sum(fmaf(u1, v1, u0 * v0)), beta);
  const float rest = l != l ? l : some && !(l == 0.f) ? (top + log2f(l)) * kLn2 : -INFINITY;   // log sum over the other items
  const float apart = rest - zt;
  float each, q, lse;
  if (out) {
    each = INFINITY;
    q = 0.f;
    lse = rest;
  } else {
    const float e = expf(-fabsf(apart));                 // rest = -inf: 0
    each = fmaxf(apart, 0.f) + log1pf(e);
    q = apart >= 0.f ? 1.f / (1.f + e) : e / (1.f + e);
    lse = fmaxf(rest, zt) + log1pf(e);
  }
  float w = a.weight ? a.weight[row] : 1.f;
  if (bad) {
    each = lse = q = NAN;
  }
  if (!has) {
    each = lse = q = w = 0.f;
  }
  const float g = a.mean ? w / (float)max(1, a.valid ? *a.valid : rows_with_target(a.target, (int)a.n)) : w;
  if (lane == 0) {
    // a weight of zero takes the row out of the loss, whatever its loss is
    a.loss_rows[row] = has && !(w == 0.f) ? w * each : 0.f;
    a.lse[row] = lse;
    const float inv = NP == 2 ? a.inv[row] : 1.f;
    if (a.h) {
      const bool dead = !has || out || w == 0.f;
      const float shift = NP == 2 ? (float)(__builtin_amdgcn_frexp_expf(inv) - 1) : 0.f;   // log2 of the power of two
      a.h[row] = dead ? -INFINITY : (__builtin_amdgcn_logf(fabsf(w)) - lse * kLog2e) + shift;
      a.kq[row] = dead ? 0.f : w * q * inv;
      a.sgn[row] = w < 0.f ? -1.f : 1.f;
    }
  }
  if (MEAN) {
    const float k = w == 0.f ? 0.f : a.scale * g * q;
    const bool zero = !has || out || w == 0.f || q == 0.f;
    const float r = l == 0.f ? 0.f : 1.f / l;
    E* dr = reinterpret_cast<E*>(a.d_rows) + row * a.d;
    if (lane < a.d) dr[lane] = (E)(zero ? 0.f : k * fmaf(o0, r, -v0));
    if (lane + 64 < a.d) dr[lane + 64] = (E)(zero ? 0.f : k * fmaf(o1, r, -v1));
  }
}

struct TableOut {
  const float* bias;
  const int32_t* valid;
  const float* loss_rows;
  float* loss;
  void* d_table;
  float* d_bias;
  float scale;
  int64_t n, c, rows_pad;
  int d, mean, reduce, splits;
};

// sum of the rows' losses, in row order per lane: one workgroup
__device__ __forceinline__ void total_loss(const float* rows, int64_t n, int mean, const int32_t* valid, float* out) {
  __shared__ double s_sum[4];
  double sum = 0;
  for (int64_t i = threadIdx.x; i < n; i += 256) sum += (double)rows[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double all = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    *out = (float)(mean ? all / (double)max(1, *valid) : all);
  }
}

__global__ void __launch_bounds__(256) xent_loss_kernel(TableOut a) { total_loss(a.loss_rows, a.n, a.mean, a.valid, a.loss); }

// ---- a few rows --------------------------------------------------------------------------------------------------------------
// Up to N rows live in the registers of every 16-lane group (8 columns a lane); a group takes an item's row as it lies in the table, four
// items at a time, in fp32: no image, no matrix instruction, and the table's bytes are the bound.
struct Few {
  const void *rows, *table;
  int64_t rows_stride, table_stride;
  const int32_t* target;
  const float *bias, *h, *kq, *sgn;
  int64_t c, per;      // items of a workgroup
  float scale;
  int n, d, rows_vec, table_vec, out_vec;
  // backward
  const float* loss_rows;
  float* loss;
  void* d_table;
  float* d_bias;
  int mean, reduce;
};
template <class E, int N>
__device__ __forceinline__ void load_few(const Few& a, int q, float (&u)[N][8], int32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = i < a.n ? a.target[i] : -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) u[i][e] = 0.f;
    if (t[i] >= 0) load8(reinterpret_cast<const E*>(a.rows) + i * a.rows_stride, 8 * q, a.d, a.rows_vec != 0, u[i]);
  }
}
// base-2 logits of an item against the rows, in every lane of the group
template <int N>
__device__ __forceinline__ void few_logits(const float (&u)[N][8], const float (&v)[8], float scale2, float b2, float (&y)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(u[i][e], v[e], s);
    y[i] = fmaf(row16_sum(s), scale2, b2);
  }
}

template <class E, int N, bool MEAN>
__global__ void __launch_bounds__(256) xent_few_forward_kernel(Few a, Part part, int64_t rows_pad) {
  __shared__ float s_m[16][N], s_l[16][N], s_o[MEAN ? 16 : 1][MEAN ? 128 : 1];
  const int q = threadIdx.x & 15, group = threadIdx.x >> 4;
  const float scale2 = a.scale * kLog2e;
  float u[N][8], m[N], l[N], o[MEAN ? N : 1][8];
  int32_t t[N];
  load_few<E, N>(a, q, u, t);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (MEAN) o[i][e] = 0.f;
  }
  const int64_t end = min(a.c, (int64_t)(blockIdx.x + 1) * a.per);
  for (int64_t j0 = (int64_t)blockIdx.x * a.per + group; j0 < end; j0 += 64) {
    float v[4][8], b2[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t j = j0 + 16 * k;
      b2[k] = j < end ? (a.bias ? a.bias[j] * kLog2e : 0.f) : -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
      if (!(b2[k] == -INFINITY)) load8(reinterpret_cast<const E*>(a.table) + j * a.table_stride, 8 * q, a.d, a.table_vec != 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float y[N];
      few_logits<N>(u, v[k], scale2, b2[k], y);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = j0 + 16 * k == t[i] ? -INFINITY : y[i];
        const float to = fmaxf(m[i], z != z ? 0.f : z);     // a NaN has to reach the sums
        if (!(to == -INFINITY)) {
          const float f = __builtin_amdgcn_exp2f(m[i] - to), p = __builtin_amdgcn_exp2f(z - to);
          m[i] = to;
          l[i] = fmaf(l[i], f, p);
          if (MEAN) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[i][e] = fmaf(o[i][e], f, p * v[k][e]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (q == 0) {
      s_m[group][i] = m[i];
      s_l[group][i] = l[i];
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= a.n) break;
    float top = -INFINITY;
    for (int g = 0; g < 16; ++g) top = fmaxf(top, s_m[g][i]);
    const bool some = top > -INFINITY;
    const int64_t at = (int64_t)blockIdx.x * rows_pad + i;
    if (MEAN) {
      const float f = some && m[i] > -INFINITY ? __builtin_amdgcn_exp2f(m[i] - top) : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s_o[group][8 * q + e] = f == 0.f ? 0.f : o[i][e] * f;
      __syncthreads();
      if (threadIdx.x < 128) {
        float sum = 0.f;
#pragma unroll
        for (int g = 0; g < 16; ++g) sum += s_o[g][threadIdx.x];
        part.o[at * 128 + threadIdx.x] = sum;
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      float sum = 0.f;
      for (int g = 0; g < 16; ++g)
        if (some && s_m[g][i] > -INFINITY) sum += s_l[g][i] * __builtin_amdgcn_exp2f(s_m[g][i] - top);
      part.m[at] = top;
      part.l[at] = sum;
    }
  }
}

template <class E, int N>
__global__ void __launch_bounds__(256) xent_few_backward_kernel(Few a) {
  if (a.reduce && blockIdx.x == gridDim.x - 1) {
    const int32_t has = rows_with_target(a.target, a.n);
    total_loss(a.loss_rows, a.n, a.mean, &has, a.loss);
    return;
  }
  const int q = threadIdx.x & 15, group = threadIdx.x >> 4;
  const float scale2 = a.scale * kLog2e;
  const float share = a.mean ? 1.f / (float)max(1, rows_with_target(a.target, a.n)) : 1.f;
  float u[N][8], h[N], kq[N], sg[N];
  int32_t t[N];
  load_few<E, N>(a, q, u, t);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = i < a.n;
    h[i] = in ? a.h[i] : -INFINITY;
    kq[i] = in ? a.kq[i] : 0.f;
    sg[i] = in ? a.sgn[i] : 1.f;
  }
  const int64_t end = min(a.c, (int64_t)(blockIdx.x + 1) * a.per);
  for (int64_t j0 = (int64_t)blockIdx.x * a.per + group; j0 < end; j0 += 64) {
    float v[4][8], b2[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t j = j0 + 16 * k;
      b2[k] = j < end ? (a.bias ? a.bias[j] * kLog2e : 0.f) : -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
      if (!(b2[k] == -INFINITY)) load8(reinterpret_cast<const E*>(a.table) + j * a.table_stride, 8 * q, a.d, a.table_vec != 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t j = j0 + 16 * k;
      if (j >= end) break;
      const bool out = b2[k] == -INFINITY;
      float y[N], x[8] = {}, sum = 0.f;
      few_logits<N>(u, v[k], scale2, b2[k], y);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (out) continue;                    // left out: zeros whatever the rows hold (0 * NaN is none)
        const float w = j == t[i] ? -kq[i] : sg[i] * __builtin_amdgcn_exp2f(y[i] + h[i]);
        sum += w;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(w, u[i][e], x[e]);
      }
      E* dst = reinterpret_cast<E*>(a.d_table) + j * a.d + 8 * q;
      const float s = a.scale * share;
      if (a.out_vec) {
        typedef E E4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (8 * q + 4 * g < a.d) {
            E4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (E)(x[4 * g + e] * s);
            *reinterpret_cast<E4*>(dst + 4 * g) = o;
          }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * q + e < a.d) dst[e] = (E)(x[e] * s);
      }
      if (q == 0 && a.d_bias) a.d_bias[j] = sum * share;
    }
  }
}

__global__ void __launch_bounds__(256) xent_few_loss_kernel(Few a) {
  const int32_t has = rows_with_target(a.target, a.n);
  total_loss(a.loss_rows, a.n, a.mean, &has, a.loss);
}

// One row of the table per DP / 4 lanes: joins its splits, applies the scales; the last workgroup sums the losses.
template <class E, int DP>
__global__ void __launch_bounds__(256) xent_table_kernel(TableOut a, Part part) {
  if (a.reduce && blockIdx.x == gridDim.x - 1) {
    total_loss(a.loss_rows, a.n, a.mean, a.valid, a.loss);
    return;
  }
  constexpr int LR = DP / 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / LR) + threadIdx.x / LR;
  const int q = threadIdx.x % LR;
  if (row >= a.c) return;
  const bool out = a.bias && a.bias[row] == -INFINITY;
  float top = -INFINITY;
  for (int k = 0; k < a.splits; ++k) top = fmaxf(top, part.m[(int64_t)k * a.rows_pad + row]);
  float l = 0.f;
  float4 o = zero4();
  if (!out) {
    if (!(top > -INFINITY)) top = 0.f;       // nothing, or nothing but NaN
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) {
      const int64_t at = (int64_t)k * a.rows_pad + row;
      const float mk = part.m[at], f = mk > -INFINITY ? __builtin_amdgcn_exp2f(mk - top) : 0.f;
      l = fmaf(part.l[at], f, l);            // NaN * 0 is NaN: a split of nothing but NaN is not lost
      o = fma4(f, *reinterpret_cast<const float4*>(part.o + at * DP + 4 * q), o);
    }
    const float share = a.mean ? 1.f / (float)max(1, *a.valid) : 1.f;
    l = ldexpf(l, (int)top) * share;
    const float k = a.scale * share;
    o.x = ldexpf(o.x, (int)top) * k;
    o.y = ldexpf(o.y, (int)top) * k;
    o.z = ldexpf(o.z, (int)top) * k;
    o.w = ldexpf(o.w, (int)top) * k;
  }
  const float v[4] = {o.x, o.y, o.z, o.w};
  E* dst = reinterpret_cast<E*>(a.d_table) + row * a.d;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (4 * q + e < a.d) dst[4 * q + e] = (E)v[e];
  if (q == 0 && a.d_bias) a.d_bias[row] = l;
}
// ---- host --------------------------------------------------------------------------------------------------------------------
inline int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Splits of the stream axis.  A workgroup costs its stages and about three more (operands in, results out and joined); k of them on a CU
// take 0.8 k times as long as one (two at a time overlap a little).  In the backward pass a popular item's workgroup meets a target in
// every stage and takes up to three times as long in it: it may become the launch's long pole.  Measured, whole calls in us.  Forward, 512 x
// 17,000 x 100 fp32 (4 own tiles, 266 stages): 106 / 84 / 74 / 77 / 85 / 90 with 16 / 32 / 54 / 89 / 133 / 256; 1,000 x 50,021 bf16 (8, 782):
// 141 / 113 / 109 / 120 / 145 with 16 / 32 / 64 / 89 / 256.  Backward, the same two (133, 8): 90 / 80 / 74 / 78 / 80 / 89 with 1 / 2 / 3 / 4 /
// 6 / 8; (391, 16): 110 / 105 / 110 / 113 / 142 with 1 / 2 / 3 / 4 / 8; 2,048 x 4,000 fp32 (32, 32): 236 / 153 / 109 / 92 / 87 / 102 with 1 / 2 / 4 /
// 8 / 16 / 32.  These three shapes are all it rests on.
inline int splits_for(int64_t own_tiles, int64_t stages, bool backward) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 256 && s <= stages; ++s) {
    const int64_t per = (stages + s - 1) / s;
    if ((stages + per - 1) / per != s) continue;    // the last split would be empty
    const int64_t k = (own_tiles * s + 255) / 256;
    const int64_t cost = std::max((k == 1 ? 10 : 8 * k) * (per + 3), backward ? 30 * per + 30 : 0);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

struct Layout {
  int np, dp;
  int64_t npad, cpad;
  int fs, bs;                       // splits of the two passes
  int64_t u_img, u_inv, u_h, u_kq, u_sgn, u_tgt, v_img, v_inv, v_h, o, m, l, loss, valid, bytes;
};

Layout layout(int64_t n, int64_t c, int d, int dtype, bool grad) {
  Layout y{};
  y.np = dtype == NNCF_F32 ? 2 : 1;
  y.dp = d <= 64 ? 64 : 128;
  y.npad = up(n, kOwn);
  y.cpad = up(c, kOwn);
  y.fs = splits_for(y.npad / kOwn, up(c, kTile) / kTile, false);
  y.bs = splits_for(y.cpad / kOwn, up(n, kTile) / kTile, true);
  int64_t at = 0;
  auto take = [&at](int64_t b) { const int64_t r = at; at += up(b, 256); return r; };
  const int64_t row = (int64_t)y.np * y.dp * 2;
  // the backward pass needs room where it is split, and where it puts sums aside
  const bool room = grad && (y.bs > 1 || up(n, kTile) / kTile > kAside);
  const int64_t part = std::max((int64_t)y.fs * y.npad, room ? (int64_t)y.bs * y.cpad : 0);
  y.u_img = take(y.npad * row);
  y.u_inv = take(y.npad * 4);
  y.u_h = take(y.npad * 4);
  y.u_kq = take(y.npad * 4);
  y.u_sgn = take(y.npad * 4);
  y.u_tgt = take(y.npad * 4);
  y.v_img = take(y.cpad * row);
  y.v_inv = take(y.cpad * 4);
  y.v_h = take(y.cpad * 4);
  y.o = take(grad ? part * y.dp * 4 : 0);
  y.m = take(part * 4);
  y.l = take(part * 4);
  y.loss = take(n * 4);
  y.valid = take(4);
  y.bytes = at;
  return y;
}

// Up to four rows take the kernels of a few rows: one row of 17,000 x 100 fp32 24 us (47 through images and the matrix pipe), four 35 (48),
// of 1M x 128 330 and 403 (574); in 16 bits, where the table is half the bytes and the matrix pipe needs a third of the products, four
// rows only of a smaller table: 35 (38) at 17,000, but 471 (323) at 1M.  131,072 is a place between these two, not a measured one.
constexpr int kFewRows = 4;
inline bool few_rows(int64_t n, int64_t c, int32_t dtype) { return n == 1 || (n <= kFewRows && (dtype == NNCF_F32 || c < 131072)); }

template <class T, int NP, int DP, int DU>
int run(const nncf_xent* x, const Layout& y, char* ws, hipStream_t st) {
  typedef typename std::conditional<NP == 2, float, typename T::E>::type E;
  const bool grad = x->d_rows != nullptr;
  auto f = [ws](int64_t at) { return reinterpret_cast<float*>(ws + at); };
  int32_t* valid = reinterpret_cast<int32_t*>(ws + y.valid);
  int32_t* tgt = reinterpret_cast<int32_t*>(ws + y.u_tgt);
  auto vec = [](const void* p, int64_t stride) { return ((uintptr_t)p % (4 * sizeof(E)) == 0 && stride % 4 == 0) ? 1 : 0; };
  const PrepSide pu{x->rows, x->rows_stride, x->n, y.npad, x->target, nullptr, ws + y.u_img, f(y.u_inv), f(y.u_h), f(y.u_sgn),
                    tgt, vec(x->rows, x->rows_stride)};
  const PrepSide pv{x->table, x->table_stride, x->c, y.cpad, nullptr, x->bias, ws + y.v_img, f(y.v_inv), f(y.v_h), nullptr, nullptr,
                    vec(x->table, x->table_stride)};
  constexpr int kPrepRows = 256 / (DP / 8);
  const int64_t ub = up(y.npad, kPrepRows) / kPrepRows, vb = up(y.cpad, kPrepRows) / kPrepRows;
  {
    ProfScope ps("xent_prep_kernel", st);
    hipLaunchKernelGGL((xent_prep_kernel<E, NP, DP>), dim3((unsigned)(ub + vb + 1)), dim3(256), 0, st, pu, pv, ub, x->dim, valid,
                       (int)x->n);
  }
  const Side u{ws + y.u_img, f(y.u_inv), f(y.u_h), f(y.u_kq), f(y.u_sgn), tgt, nullptr, x->n, y.npad};
  const Side v{ws + y.v_img, f(y.v_inv), f(y.v_h), nullptr, nullptr, nullptr, x->bias, x->c, y.cpad};
  const Part part{f(y.o), f(y.m), f(y.l)};
  const float scale2 = x->scale * kLog2e;
  {
    const int stages = (int)(up(x->c, kTile) / kTile), per = (stages + y.fs - 1) / y.fs;
    const dim3 grid((unsigned)y.fs, (unsigned)(y.npad / kOwn));
    ProfScope ps("xent_stream_kernel", st);
    if (grad)
      hipLaunchKernelGGL((xent_stream_kernel<T, NP, DP, DU, false, false, true>), grid, dim3(256), 0, st, u, v, part, Grad{}, scale2, stages, per);
    else
      hipLaunchKernelGGL((xent_stream_kernel<T, NP, DP, DU, false, false, false>), grid, dim3(256), 0, st, u, v, part, Grad{}, scale2, stages, per);
  }
  const bool scalar = x->reduction != NNCF_NONE;
  const int mean = x->reduction == NNCF_MEAN;
  float* loss_rows = scalar ? f(y.loss) : x->loss;
  const RowsOut ro{x->rows, x->table, x->rows_stride, x->table_stride, x->bias, x->weight, x->target, valid, loss_rows, x->lse,
                   grad ? f(y.u_h) : nullptr, f(y.u_kq), f(y.u_sgn), f(y.u_inv), x->d_rows, x->scale, x->n, x->c, y.npad, x->dim, mean, y.fs};
  {
    ProfScope ps("xent_rows_kernel", st);
    if (!grad)
      hipLaunchKernelGGL((xent_rows_kernel<E, NP, DP, false, 1>), dim3((unsigned)((x->n + 3) / 4)), dim3(256), 0, st, ro, part);
    else if (y.fs <= 8)
      hipLaunchKernelGGL((xent_rows_kernel<E, NP, DP, true, 1>), dim3((unsigned)((x->n + 3) / 4)), dim3(256), 0, st, ro, part);
    else
      hipLaunchKernelGGL((xent_rows_kernel<E, NP, DP, true, 4>), dim3((unsigned)x->n), dim3(256), 0, st, ro, part);
  }
  TableOut to{x->bias, valid, loss_rows, x->loss, x->d_table, x->d_bias, x->scale, x->n, x->c, y.cpad, x->dim, mean, scalar, y.bs};
  if (!grad) {
    if (scalar) hipLaunchKernelGGL(xent_loss_kernel, dim3(1), dim3(256), 0, st, to);
  } else {
    const int stages = (int)(up(x->n, kTile) / kTile), per = (stages + y.bs - 1) / y.bs;
    // d_table alone needs no joining where the users are not split: 0.5 GB less to write and to read at 1M items of 128
    const Grad direct = y.bs == 1 ? Grad{x->d_table, x->d_bias, valid, x->scale, x->dim, mean, vec(x->d_table, x->dim)} : Grad{};
    const dim3 grid((unsigned)y.bs, (unsigned)(y.cpad / kOwn));
    {
      ProfScope ps("xent_stream_kernel", st);
      if (x->weight)
        hipLaunchKernelGGL((xent_stream_kernel<T, NP, DP, DU, true, true, true>), grid, dim3(256), 0, st, v, u, part, direct, scale2, stages, per);
      else
        hipLaunchKernelGGL((xent_stream_kernel<T, NP, DP, DU, true, false, true>), grid, dim3(256), 0, st, v, u, part, direct, scale2, stages, per);
    }
    if (y.bs == 1) {
      if (scalar) hipLaunchKernelGGL(xent_loss_kernel, dim3(1), dim3(256), 0, st, to);
      NNCF_HIP_CHECK(hipGetLastError());
      return NNCF_OK;
    }
    ProfScope ps("xent_table_kernel", st);
    constexpr int kRows = 256 / (DP / 4);
    hipLaunchKernelGGL((xent_table_kernel<E, DP>), dim3((unsigned)((x->c + kRows - 1) / kRows + (scalar ? 1 : 0))), dim3(256), 0, st, to, part);
  }
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

struct FewLayout {
  int splits;
  int64_t per, o, m, l, h, kq, sgn, loss, bytes;
};
FewLayout few_layout(int64_t n, int64_t c, bool grad) {
  FewLayout y{};
  // more workgroups where there is work for them; their results are joined in turn.  At most 4,096 items: 256 terms of a running sum.
  y.per = std::min<int64_t>(up(c / (c < 131072 ? 256 : 512) + 1, 64), 4096);
  y.splits = (int)((c + y.per - 1) / y.per);
  int64_t at = 0;
  auto take = [&at](int64_t b) { const int64_t r = at; at += up(b, 256); return r; };
  y.o = take(grad ? (int64_t)y.splits * kFewRows * 128 * 4 : 0);
  y.m = take((int64_t)y.splits * kFewRows * 4);
  y.l = take((int64_t)y.splits * kFewRows * 4);
  y.h = take(kFewRows * 4);
  y.kq = take(kFewRows * 4);
  y.sgn = take(kFewRows * 4);
  y.loss = take(kFewRows * 4);
  y.bytes = at;
  return y;
}

template <class E, int N>
int run_few(const nncf_xent* x, char* ws, hipStream_t st) {
  const bool grad = x->d_rows != nullptr;
  const FewLayout y = few_layout(x->n, x->c, grad);
  auto f = [ws](int64_t at) { return reinterpret_cast<float*>(ws + at); };
  auto vec = [](const void* p, int64_t stride) { return ((uintptr_t)p % (4 * sizeof(E)) == 0 && stride % 4 == 0) ? 1 : 0; };
  const bool scalar = x->reduction != NNCF_NONE;
  const int mean = x->reduction == NNCF_MEAN;
  float* loss_rows = scalar ? f(y.loss) : x->loss;
  const Few a{x->rows, x->table, x->rows_stride, x->table_stride, x->target, x->bias, f(y.h), f(y.kq), f(y.sgn), x->c, y.per, x->scale, (int)x->n,
              x->dim, vec(x->rows, x->rows_stride), vec(x->table, x->table_stride), vec(x->d_table, x->dim), loss_rows, x->loss, x->d_table, x->d_bias, mean, scalar};
  const Part part{f(y.o), f(y.m), f(y.l)};
  const RowsOut ro{x->rows, x->table, x->rows_stride, x->table_stride, x->bias, x->weight, x->target, nullptr, loss_rows, x->lse,
                   grad ? f(y.h) : nullptr, f(y.kq), f(y.sgn), nullptr, x->d_rows, x->scale, x->n, x->c, kFewRows, x->dim, mean, y.splits};
  {
    ProfScope ps("xent_few_forward_kernel", st);
    if (grad)
      hipLaunchKernelGGL((xent_few_forward_kernel<E, N, true>), dim3((unsigned)y.splits), dim3(256), 0, st, a, part, (int64_t)kFewRows);
    else
      hipLaunchKernelGGL((xent_few_forward_kernel<E, N, false>), dim3((unsigned)y.splits), dim3(256), 0, st, a, part, (int64_t)kFewRows);
  }
  {
    ProfScope ps("xent_rows_kernel", st);
    if (grad)
      hipLaunchKernelGGL((xent_rows_kernel<E, 1, 128, true, 4>), dim3((unsigned)x->n), dim3(256), 0, st, ro, part);
    else
      hipLaunchKernelGGL((xent_rows_kernel<E, 1, 128, false, 1>), dim3((unsigned)((x->n + 3) / 4)), dim3(256), 0, st, ro, part);
  }
  if (grad) {
    ProfScope ps("xent_few_backward_kernel", st);
    Few b = a;
    b.per = up((x->c + 2047) / 2048, 64);      // as many workgroups as the device holds: nothing is joined behind them
    hipLaunchKernelGGL((xent_few_backward_kernel<E, N>), dim3((unsigned)((x->c + b.per - 1) / b.per + (scalar ? 1 : 0))), dim3(256), 0, st, b);
  } else if (scalar) {
    hipLaunchKernelGGL((xent_few_loss_kernel), dim3(1), dim3(256), 0, st, a);
  }
  NNCF_HIP_CHECK(hipGetLastError());
  return NNCF_OK;
}

template <class E>
int run_few_rows(const nncf_xent* x, char* ws, hipStream_t st) {
  if (x->n == 1) return run_few<E, 1>(x, ws, st);
  return run_few<E, 4>(x, ws, st);
}

// Products over the columns in use: at 96 of 128 a quarter of them less.
template <class T, int NP>
int run_width(const nncf_xent* x, const Layout& y, char* ws, hipStream_t st) {
  if (x->dim <= 64) return run<T, NP, 64, 64>(x, y, ws, st);
  if (x->dim <= 96) return run<T, NP, 128, 96>(x, y, ws, st);
  if (x->dim <= 112) return run<T, NP, 128, 112>(x, y, ws, st);
  return run<T, NP, 128, 128>(x, y, ws, st);
}

int check_shape(int64_t n, int64_t c, int32_t dim, int32_t dtype) {
  NNCF_REQUIRE(n > 0 && n <= (int64_t)kOwn * 65535, "n = %lld rows out of range (1..%lld)", (long long)n, (long long)kOwn * 65535);
  // own tiles of a launch are its grid's second dimension
  NNCF_REQUIRE(c > 0 && c <= (int64_t)kOwn * 65535, "c = %lld items out of range (1..%lld)", (long long)c, (long long)kOwn * 65535);
  NNCF_REQUIRE(dim > 0 && dim <= 128, "dim = %d out of range (1..128)", dim);
  NNCF_REQUIRE(dtype == NNCF_F32 || dtype == NNCF_F16 || dtype == NNCF_BF16, "dtype = %d unknown", dtype);
  return NNCF_OK;
}
}  // namespace
}  // namespace nncf

extern "C" int64_t nncf_softmax_xent_ws_bytes(int64_t n, int64_t c, int32_t dim, int32_t dtype, int32_t with_grad) {
  if (nncf::check_shape(n, c, dim, dtype) != NNCF_OK) return -1;
  if (nncf::few_rows(n, c, dtype)) return nncf::few_layout(n, c, with_grad != 0).bytes;
  return nncf::layout(n, c, dim, dtype, with_grad != 0).bytes;
}

extern "C" int nncf_softmax_xent(const nncf_xent* x, void* d_ws, int64_t ws_bytes, void* stream) {
  using namespace nncf;
  NNCF_REQUIRE(x != nullptr, "NULL argument");
  const int rc = check_shape(x->n, x->c, x->dim, x->dtype);
  if (rc) return rc;
  NNCF_REQUIRE(x->rows && x->table && x->target && x->loss && x->lse && d_ws, "NULL argument");
  NNCF_REQUIRE((x->d_rows != nullptr) == (x->d_table != nullptr), "d_rows and d_table are computed together");
  NNCF_REQUIRE(!x->d_bias || (x->bias && x->d_rows), "d_bias needs a bias and the other gradients");
  NNCF_REQUIRE(x->rows_stride >= x->dim && x->table_stride >= x->dim, "a row stride is below dim = %d", x->dim);
  NNCF_REQUIRE(x->reduction == NNCF_NONE || x->reduction == NNCF_MEAN || x->reduction == NNCF_SUM, "reduction = %d unknown", x->reduction);
  NNCF_REQUIRE(std::isfinite(x->scale), "scale must be finite");
  const uintptr_t es = x->dtype == NNCF_F32 ? 4 : 2;
  NNCF_REQUIRE((uintptr_t)x->rows % es == 0 && (uintptr_t)x->table % es == 0 && (uintptr_t)x->d_rows % es == 0 &&
               (uintptr_t)x->d_table % es == 0, "a tensor is not aligned to its elements");
  const bool few = few_rows(x->n, x->c, x->dtype);
  const Layout y = few ? Layout{} : layout(x->n, x->c, x->dim, x->dtype, x->d_rows != nullptr);
  const int64_t need = few ? few_layout(x->n, x->c, x->d_rows != nullptr).bytes : y.bytes;
  NNCF_REQUIRE(ws_bytes >= need, "workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  NNCF_REQUIRE(((uintptr_t)d_ws & 255) == 0, "workspace must be 256-byte aligned");
  char* ws = reinterpret_cast<char*>(d_ws);
  hipStream_t st = as_stream(stream);
  if (few) {
    if (x->dtype == NNCF_F32) return run_few_rows<float>(x, ws, st);
    if (x->dtype == NNCF_F16) return run_few_rows<_Float16>(x, ws, st);
    return run_few_rows<__bf16>(x, ws, st);
  }
  if (x->dtype == NNCF_F32) return run_width<F16, 2>(x, y, ws, st);
  if (x->dtype == NNCF_F16) return run_width<F16, 1>(x, y, ws, st);
  return run_width<BF16, 1>(x, y, ws, st);
}
