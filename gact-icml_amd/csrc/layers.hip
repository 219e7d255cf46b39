// Layers that train on 8-bit checkpoints, for MI355X (gfx950): checkpoints of rows, layer norm, linear layers with bias, activation
// and residual in the product's epilogue, and the products of the backward pass, one of which reads the checkpoint's codes.
//
// A checkpoint of a matrix of T holds every row in groups of 256 columns, the last one shorter.  Per group: the minimum and a scale,
// both float, scale = float(255 / (double(max - min) + 2e-6)); per value: code = rint(max(fma(x - min, scale, 0.5) - 0.5, 0)).
// That is the 8-bit code of gact_quantize on the values widened to float, rounded to nearest (GACT_NOISE_CONST).
// (A NaN: code 0, and left out of minimum and maximum, as there.)
// A code stands for code / scale + min, computed as fma(code, 1 / scale, min): one division per group and not one per value, which
// differs from the quotient by a rounding of float.
//
// Compiled with -ffp-contract=off: every operation is the one it spells (but for roundings to a half, see rounded()).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gact_hip.h"
#include "layer_cuts.h"

namespace {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kGroup = 256;
constexpr int kVec = 8;   // columns of a lane's piece

// The workgroup's number in a launch of grid_of(): beyond 2^32 threads a launch goes on along y
__device__ __forceinline__ int64_t block_of() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// ---- eight consecutive columns ----
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[kVec]) {
  if constexpr (std::is_same<T, float>::value) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = a[e], v[e + 4] = b[e];
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 a = *(const T8*)p;
#pragma unroll
    for (int e = 0; e < kVec; e++) v[e] = (float)a[e];
  }
}
// A result is a float before it is rounded to T, in every kernel and whichever way it is stored: the empty statement keeps the compiler from making
// one instruction of the last operation and its rounding to a half, which rounds once and differs in one of 2^13 values - of rows at one address and
// not of the same rows at another.
template <typename T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (std::is_same<T, f16>::value) asm("" : "+v"(v));
  return (T)v;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[kVec]) {
  if constexpr (std::is_same<T, float>::value) {
    *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 a;
#pragma unroll
    for (int e = 0; e < kVec; e++) a[e] = rounded<T>(v[e]);
    *(T8*)p = a;
  }
}
// the same of a row of which `n` columns are left; WHOLE: n is 0 or at least 8 and the address a multiple of 16 bytes.  Otherwise whole
// pieces are still one access, at whatever address (value by value a layer norm of 771 halves takes twice as long).
template <typename T>
struct Loose {
  typedef T Eight __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_cols(const T* p, int64_t n, float (&v)[kVec]) {
  if (WHOLE) {
    if (n > 0) {
      load8(p, v);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e++) v[e] = 0.0f;
    }
  } else if (n >= kVec) {
    const typename Loose<T>::Eight a = *(const typename Loose<T>::Eight*)p;
#pragma unroll
    for (int e = 0; e < kVec; e++) v[e] = (float)a[e];
  } else {
#pragma unroll
    for (int e = 0; e < kVec; e++) v[e] = e < n ? (float)p[e] : 0.0f;
  }
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store_cols(T* p, int64_t n, const float (&v)[kVec]) {
  if (WHOLE) {
    if (n > 0) store8(p, v);
  } else if (n >= kVec) {
    typename Loose<T>::Eight a;
#pragma unroll
    for (int e = 0; e < kVec; e++) a[e] = rounded<T>(v[e]);
    *(typename Loose<T>::Eight*)p = a;
  } else {
#pragma unroll
    for (int e = 0; e < kVec; e++)
      if (e < n) p[e] = rounded<T>(v[e]);
  }
}

// ---- reductions over 2^n neighbouring lanes, the result in each of them ----
template <int CTRL>
__device__ __forceinline__ float row_rotated(float v) {
  const int b = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, CTRL, 0xf, 0xf, false));
}
struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Least {
  static __device__ __forceinline__ float of(float a, float b) { return __builtin_fminf(a, b); }
};
struct Most {
  static __device__ __forceinline__ float of(float a, float b) { return __builtin_fmaxf(a, b); }
};
template <typename OP, int LANES>
__device__ __forceinline__ float over_lanes(float v) {
  static_assert(LANES >= 16 && LANES <= 64, "rows of 16 lanes");
  v = OP::of(v, row_rotated<0x128>(v));
  v = OP::of(v, row_rotated<0x124>(v));
  v = OP::of(v, row_rotated<0x122>(v));
  v = OP::of(v, row_rotated<0x121>(v));
  if (LANES >= 32) v = OP::of(v, __shfl_xor(v, 16));
  if (LANES >= 64) v = OP::of(v, __shfl_xor(v, 32));
  return v;
}

// ---- the checkpoint's arithmetic ----
__device__ __forceinline__ float scale_of(float lo, float hi) { return (float)(255.0 / ((double)(hi - lo) + 2e-6)); }
// scales of K groups, of which every row of 16 lanes holds the ends: lane k divides for group k, one division for all of them
template <int LANE>
__device__ __forceinline__ float row_broadcast(float v) {
  const int b = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, 0x150 + LANE, 0xf, 0xf, false));
}
template <int K, int AT = 0>
__device__ __forceinline__ void broadcast_all(float mine, float (&s)[K]) {
  if constexpr (AT < K) {
    s[AT] = row_broadcast<AT>(mine);
    broadcast_all<K, AT + 1>(mine, s);
  }
}
template <int K>
__device__ __forceinline__ void scales_of(const float (&lo)[K], const float (&hi)[K], float (&s)[K]) {
  static_assert(K <= 16, "a row has 16 lanes");
  float l = lo[0], h = hi[0];
#pragma unroll
  for (int k = 1; k < K; k++) {
    const bool mine = (threadIdx.x & 15) == k;
    l = mine ? lo[k] : l;
    h = mine ? hi[k] : h;
  }
  const float q = scale_of(l, h);
  if (K == 1)
    s[0] = q;
  else
    broadcast_all<K>(q, s);
}
// 1 / scale: the hardware's reciprocal and one step of Newton's, within a unit in the last place; NaN for a scale of zero (a range that
// overflowed), which stands for nothing
__device__ __forceinline__ float inverse_of(float scale) {
  const float r = __builtin_amdgcn_rcpf(scale);
  return __builtin_fmaf(__builtin_fmaf(-scale, r, 1.0f), r, r);
}
// [0, 255] and rounded to nearest even by the conversion itself; a NaN becomes 0
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float lo, float scale) {
  uint32_t w = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(a - lo, scale, 0.5f) - 0.5f, 0, 0);
  w = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(b - lo, scale, 0.5f) - 0.5f, 1, w);
  w = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(c - lo, scale, 0.5f) - 0.5f, 2, w);
  return __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(d - lo, scale, 0.5f) - 0.5f, 3, w);
}
__device__ __forceinline__ float code_at(uint32_t w, int e) { return (float)(uint8_t)(w >> (8 * e)); }
// A value is a float before it is rounded to T, in every kernel: the empty statement keeps the compiler from making one instruction of the
// sum and its rounding to a half, which rounds once and differs in one of 2^13 values.
__device__ __forceinline__ float value_of(uint32_t w, int e, float inv, float lo) {
  float v = __builtin_fmaf(code_at(w, e), inv, lo);
  asm("" : "+v"(v));
  return v;
}
__device__ __forceinline__ void eight_values(u32x2 w, float inv, float lo, float (&v)[kVec]) {
#pragma unroll
  for (int e = 0; e < kVec; e++) v[e] = value_of(w[e >> 2], e & 3, inv, lo);
}

// ---- activations: act(z) and act'(z) ----
enum { ACT_UNFINISHED = -1, ACT_NONE = GACT_ACT_NONE, ACT_GELU = GACT_ACT_GELU, ACT_GELU_TANH = GACT_ACT_GELU_TANH, ACT_SILU = GACT_ACT_SILU };
// Exact to float's rounding for float; for 16-bit types, whose own rounding is at least 2^-12, the hardware's exponential and reciprocal and a
// polynomial: log2(2 (1 - Phi(a))), a >= 0, is smooth, and a fit of degree 7 over [0, 6] gives 1 - Phi(a) in float steps to 7e-6 of itself up to 4,
// 1.1e-5 up to 5 and 2.9e-5 up to 6.  Beyond it falls: 1.5e-4 of itself up to 7, 3 % up to 9, of which 1e-19 are left.  Phi is off by 2.8e-6 at
// most, GELU by 8.3e-7.
// In the epilogue of a product of 1024 columns the library's erfc takes as long as the product, a quotient of polynomials a quarter of it.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float x) {
  if (EXACT) return 1.0f / (1.0f + expf(-x));
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}
__device__ __forceinline__ float twice_upper_tail(float a) {
  float p = __builtin_fmaf(a, -1.79147102e-06f, 6.08547037e-05f);
  p = __builtin_fmaf(a, p, -0.000925627672f);
  p = __builtin_fmaf(a, p, 0.00849229447f);
  p = __builtin_fmaf(a, p, -0.0539352561f);
  p = __builtin_fmaf(a, p, -0.458482679f);
  p = __builtin_fmaf(a, p, -1.15124609f);
  return __builtin_amdgcn_exp2f(a * p);
}
// the normal distribution's cumulative function and exp(-z^2/2)
template <bool EXACT>
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& e) {
  if (EXACT) {
    e = expf(-0.5f * z * z);
    cdf = 0.5f * erfcf(-0.70710678118654752f * z);
    return;
  }
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  const float q = 0.5f * twice_upper_tail(__builtin_fabsf(z));
  cdf = z < 0.0f ? q : 1.0f - q;
}
template <bool EXACT>
__device__ __forceinline__ float activated(float z, int act) {
  switch (act) {
    case ACT_GELU: {
      if (!EXACT) {
        // max(z, 0) - |z| (1 - Phi(|z|)), the maximum as z / 2 + |z| / 2, which the largest z do not overflow; the bound keeps an infinite z
        // from meeting a tail of zero
        const float a = __builtin_fabsf(z), h = 0.5f * a;
        return __builtin_fmaf(-__builtin_amdgcn_fmed3f(h, 0.0f, 1.5e38f), twice_upper_tail(a), __builtin_fmaf(0.5f, z, h));
      }
      float cdf, e;
      normal_cdf<EXACT>(z, cdf, e);
      return z * cdf;
    }
    case ACT_GELU_TANH: return z * sigmoid<EXACT>(1.5957691216057308f * (z + 0.044715f * z * z * z));   // 0.5 (1 + tanh u) = sigmoid(2 u)
    case ACT_SILU: return z * sigmoid<EXACT>(z);
    default: return z;
  }
}
template <typename T, int ACT>
__device__ __forceinline__ f32x4 activated4(f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = activated<std::is_same<T, float>::value>(v[e], ACT);
  return v;
}
template <bool EXACT>
__device__ __forceinline__ float slope(float z, int act) {
  switch (act) {
    case ACT_GELU: {
      float cdf, e;
      normal_cdf<EXACT>(z, cdf, e);
      return cdf + z * e * 0.39894228040143268f;
    }
    case ACT_GELU_TANH: {
      const float s = sigmoid<EXACT>(1.5957691216057308f * (z + 0.044715f * z * z * z));
      return s + z * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * z * z);
    }
    case ACT_SILU: {
      const float s = sigmoid<EXACT>(z);
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Checkpoints of rows.  32 lanes (16 of rows of up to 128 columns) own a group: one 16-byte piece each (float: two), its minimum and maximum over
// those lanes.
// ---------------------------------------------------------------------------------------------------------------------------------
// Times, here and of the kernels below up to the products, are of launches one behind the other whose inputs are in no cache; a small tensor that
// the caches hold takes less (the restore of 25088x384 right behind its checkpoint 6 to 7 us, layer norm of 16384x1024 21 each way).
// Bound by memory: 32768x4096 halves 83 us (4.9 TB/s), floats 115 (5.9), 16384x1024 floats 16.9 (5.0), 25088x384 halves 12.1, of which the launch
// and the one load that nothing overlaps are half.  One group at a time: four to a half wave, with their loads together and one division for all of their
// scales, take 84 us instead of 90 for 134 M halves, but 14 instead of 11.5 for 10 M.  A group shorter than 256 leaves lanes idle (771
// columns of halves, 23 us for 25088 rows, 2.6 TB/s).
template <typename T, int LANES, bool WHOLE>
__global__ __launch_bounds__(256) void checkpoint_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ldx, int groups,
                                                         uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale,
                                                         float* __restrict__ mn) {
  const int64_t unit = block_of() * (256 / LANES) + threadIdx.x / LANES;
  const int64_t row = unit / groups;
  const int g = (int)(unit - row * groups), lane = threadIdx.x % LANES;
  if (row >= rows) return;
  const int col = g * kGroup + lane * kVec, n = cols - col;
  float v[kVec];
  load_cols<T, WHOLE>(x + row * ldx + col, n, v);
  float lo = __builtin_inff(), hi = -__builtin_inff();
#pragma unroll
  for (int e = 0; e < kVec; e++)
    if ((WHOLE ? 0 : e) < n) lo = __builtin_fminf(lo, v[e]), hi = __builtin_fmaxf(hi, v[e]);
  lo = over_lanes<Least, LANES>(lo);
  hi = over_lanes<Most, LANES>(hi);
  const float s = scale_of(lo, hi);
  if (n > 0)
    *(u32x2*)(codes + row * ldc + col) = u32x2{four_codes(v[0], v[1], v[2], v[3], lo, s), four_codes(v[4], v[5], v[6], v[7], lo, s)};
  if (lane == 0) {
    scale[unit] = s;
    mn[unit] = lo;
  }
}

// The values again, the same lanes: 32768x4096 halves 73 us (5.5 TB/s), floats 118 (5.7), 16384x1024 halves 12.0 (4.2), 25088x384 8.7.  1 / scale
// is made by every lane: the division is hidden behind the loads.
template <typename T, int LANES, bool WHOLE>
__global__ __launch_bounds__(256) void restore_kernel(const uint8_t* __restrict__ codes, int64_t ldc, const float* __restrict__ scale,
                                                      const float* __restrict__ mn, int64_t rows, int cols, int groups,
                                                      T* __restrict__ out) {
  const int64_t unit = block_of() * (256 / LANES) + threadIdx.x / LANES;
  const int64_t row = unit / groups;
  const int g = (int)(unit - row * groups), lane = threadIdx.x % LANES;
  if (row >= rows) return;
  const int col = g * kGroup + lane * kVec, n = cols - col;
  if (n <= 0) return;
  float v[kVec];
  eight_values(*(const u32x2*)(codes + row * ldc + col), inverse_of(scale[unit]), mn[unit], v);
  store_cols<T, WHOLE>(out + row * cols + col, n, v);
}

// rows copied to a stride that the products can load 16 bytes at a time from, the columns behind the last one zero.  25088x771 halves 18.6 us
// (4.2 TB/s); a product that reads such rows value by value takes several times as long as on whole pieces.
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ldx, T* __restrict__ out,
                                                       int ldo) {
  const int per = ldo / kVec;
  const int64_t unit = block_of() * 256 + threadIdx.x;
  const int64_t row = unit / per;
  if (row >= rows) return;
  const int col = (int)(unit - row * per) * kVec;
  float v[kVec];
  load_cols<T, false>(x + row * ldx + col, cols - col, v);
  store8(out + row * ldo + col, v);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Layer norm.  LPR threads own a row and hold it in registers: NC pieces of 8 columns each, LPR * 8 columns apart, so that a group
// of 256 columns is one piece of 32 neighbouring threads (LPR 16: rows of up to 128 columns, one piece).  LPR up to 64: 256 / LPR rows per workgroup;
// above: a workgroup of LPR threads per row.
// ---------------------------------------------------------------------------------------------------------------------------------
template <int LPR, int THREADS = 256>
struct RowShape {
  static constexpr int kThreads = LPR <= 64 ? THREADS : LPR;
  static constexpr int kRows = kThreads / LPR;            // rows at a time
  static constexpr int kWaves = LPR <= 64 ? 1 : LPR / 64;   // waves of a row
  static constexpr int kSpan = LPR * kVec;                // columns of a piece
};
// the sum of v over the threads of a row; `turn` tells apart the buffers of consecutive sums
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* shared, int turn) {
  v = over_lanes<Sum, (LPR < 64 ? LPR : 64)>(v);
  if constexpr (RowShape<LPR>::kWaves > 1) {
    constexpr int W = RowShape<LPR>::kWaves;
    float* at = shared + (turn & 1) * W;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) v += at[w];
  }
  return v;
}

// mean = sum / cols, var = sum (x - mean)^2 / cols from the row in registers, in floats: one read, one write of x, and the codes.  Bound by memory:
// 401408x96 floats 71 us (5.0 TB/s), 65536x1024 halves 73 (4.6), 16384x4096 halves 67 (5.0), 16384x1024 halves 26 (3.3: half of it launch,
// ramp and the tail).  U consecutive rows at a time: their loads are on the way together, and their scales are one division (see scales_of).
template <typename T, int LPR, int NC, int U, bool WHOLE>
__global__ __launch_bounds__(RowShape<LPR>::kThreads) void norm_forward_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ weight, const T* __restrict__ bias, int64_t rows, int cols, float per_col,
    float eps, T* __restrict__ y, uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale, float* __restrict__ mn,
    float* __restrict__ stats) {
  using Shape = RowShape<LPR>;
  __shared__ float shared[2 * Shape::kWaves];
  const int lane = threadIdx.x % LPR;
  const int64_t row0 = (block_of() * Shape::kRows + threadIdx.x / LPR) * U;
  if (row0 >= rows) return;      // all of the row's threads, so none waits for another
  const int there = U == 1 || rows - row0 >= U ? U : (int)(rows - row0);      // of the U rows
  float v[U][NC][kVec];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int col = c * Shape::kSpan + lane * kVec;
      load_cols<T, WHOLE>(x + (row0 + (u < there ? u : 0)) * ldx + col, cols - col, v[u][c]);
    }
  float mean[U], rstd[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int e = 0; e < kVec; e++) sum += v[u][c][e];
    mean[u] = row_sum<LPR>(sum, shared, 2 * u) * per_col;
    sum = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int left = cols - (c * Shape::kSpan + lane * kVec);
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        const float d = (WHOLE ? 0 : e) < left ? v[u][c][e] - mean[u] : 0.0f;
        sum = __builtin_fmaf(d, d, sum);
      }
    }
    rstd[u] = __builtin_amdgcn_rsqf(__builtin_fmaf(row_sum<LPR>(sum, shared, 2 * u + 1), per_col, eps));
  }
  if (stats && lane == 0)
#pragma unroll
    for (int u = 0; u < U; u++)
      if (u < there) *(f32x2*)(stats + 2 * (row0 + u)) = f32x2{mean[u], rstd[u]};
  if (codes) {
    static_assert(LPR >= 32 || NC == 1, "a group is one piece");
    constexpr int GLANES = LPR < 32 ? 16 : 32, K = U * NC;
    const int groups = (cols + kGroup - 1) / kGroup;
    float lo[K], hi[K], s[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int u = k / NC, c = k % NC, left = cols - (c * Shape::kSpan + lane * kVec);
      lo[k] = __builtin_inff();
      hi[k] = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < kVec; e++)
        if ((WHOLE ? 0 : e) < left) lo[k] = __builtin_fminf(lo[k], v[u][c][e]), hi[k] = __builtin_fmaxf(hi[k], v[u][c][e]);
      lo[k] = over_lanes<Least, GLANES>(lo[k]);
      hi[k] = over_lanes<Most, GLANES>(hi[k]);
    }
    scales_of<K>(lo, hi, s);
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int u = k / NC, c = k % NC, col = c * Shape::kSpan + lane * kVec;
      if (u >= there || col >= cols) continue;
      const float (&w)[kVec] = v[u][c];
      *(u32x2*)(codes + (row0 + u) * ldc + col) =
          u32x2{four_codes(w[0], w[1], w[2], w[3], lo[k], s[k]), four_codes(w[4], w[5], w[6], w[7], lo[k], s[k])};
      if (lane % GLANES == 0) {
        scale[(row0 + u) * groups + col / kGroup] = s[k];
        mn[(row0 + u) * groups + col / kGroup] = lo[k];
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const int col = c * Shape::kSpan + lane * kVec;
    float w[kVec], b[kVec];
    if (weight)
      load_cols<T, WHOLE>(weight + col, cols - col, w);
    else
      for (int e = 0; e < kVec; e++) w[e] = 1.0f;
    if (bias)
      load_cols<T, WHOLE>(bias + col, cols - col, b);
    else
      for (int e = 0; e < kVec; e++) b[e] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      float o[kVec];
#pragma unroll
      for (int e = 0; e < kVec; e++) o[e] = __builtin_fmaf((v[u][c][e] - mean[u]) * rstd[u], w[e], b[e]);
      if (u < there) store_cols<T, WHOLE>(y + (row0 + u) * cols + col, cols - col, o);
    }
  }
}

// xh = (value - mean) rstd, g = dy w: dx = rstd (g - mean(g) - xh mean(g xh)); a thread adds up dy xh and dy of its columns over the
// rows it sees, a workgroup writes one row of partial sums.  While a row is worked on, the next one's loads are on the way.
// Reads dy and the codes, writes dx: 401408x96 floats 74 us (4.8 TB/s), 65536x1024 halves 80 (4.2), 16384x4096 halves 86 (3.9), 16384x1024
// halves 26 (3.3), the column sums included (they take 4 us, 14 of 86 at 4096 columns).
constexpr int kNormThreads = 512;   // waves that share a row of partial sums (with 4 of them and twice the workgroups there is twice as much to add up)
template <int LPR>
using SharedRows = RowShape<LPR, kNormThreads>;
template <typename T, int LPR, int NC, bool WHOLE>
__global__ __launch_bounds__(SharedRows<LPR>::kThreads) void norm_backward_kernel(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ weight, const uint8_t* __restrict__ codes, int64_t ldc,
    const float* __restrict__ scale, const float* __restrict__ mn, const float* __restrict__ stats, int64_t rows, int cols, float per_col,
    T* __restrict__ dx, float* __restrict__ partial) {
  using Shape = SharedRows<LPR>;
  __shared__ float shared[4 * Shape::kWaves];
  constexpr int kFold = LPR < 64 ? 64 / LPR : 1;        // rows of a wave
  constexpr int kAcross = LPR <= 64 ? kNormThreads / 64 : 1;             // waves whose partial sums a workgroup adds up
  __shared__ float folded[kAcross > 1 ? 64 * kVec * kAcross : 1];
  typedef T T8 __attribute__((ext_vector_type(8), aligned(WHOLE ? 16 : sizeof(T))));
  struct Asked {     // a row on its way
    T8 dy[NC];
    u32x2 codes[NC];
    float scale[NC], lo[NC];
    f32x2 stats;
  };
  const int lane = threadIdx.x % LPR;
  const int groups = (cols + kGroup - 1) / kGroup;
  const int64_t apart = (int64_t)gridDim.x * Shape::kRows;
  auto ask = [&](int64_t row, Asked& a) __attribute__((always_inline)) {
    row = row < rows ? row : rows - 1;
    a.stats = *(const f32x2*)(stats + 2 * row);
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int col = c * Shape::kSpan + lane * kVec, left = cols - col;
      a.dy[c] = T8{};
      a.codes[c] = u32x2{0, 0};
      a.scale[c] = 1.0f;
      a.lo[c] = 0.0f;
      if (left > 0) {
        const T* p = dy + row * lddy + col;
        if (WHOLE || left >= kVec) {
          a.dy[c] = *(const T8*)p;
        } else {
#pragma unroll
          for (int e = 0; e < kVec; e++)
            if (e < left) a.dy[c][e] = p[e];
        }
        a.codes[c] = *(const u32x2*)(codes + row * ldc + col);
        a.scale[c] = scale[row * groups + col / kGroup];
        a.lo[c] = mn[row * groups + col / kGroup];
      }
    }
  };
  float w[NC][kVec], dw[NC][kVec], db[NC][kVec];
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const int col = c * Shape::kSpan + lane * kVec;
    if (weight)
      load_cols<T, WHOLE>(weight + col, cols - col, w[c]);
    else
      for (int e = 0; e < kVec; e++) w[c][e] = 1.0f;
#pragma unroll
    for (int e = 0; e < kVec; e++) dw[c][e] = db[c][e] = 0.0f;
  }
  int turn = 0;
  constexpr bool kAhead = NC <= 2;      // with four pieces the registers do not hold a second row
  Asked next;
  int64_t first = (int64_t)blockIdx.x * Shape::kRows;
  if (kAhead) ask(first + threadIdx.x / LPR, next);
  for (; first < rows; first += apart) {
    const int64_t row = first + threadIdx.x / LPR;
    const bool there = Shape::kRows == 1 || row < rows;
    if (!kAhead) ask(row, next);
    const Asked now = next;
    if (kAhead && first + apart < rows) ask(row + apart, next);
    const float mean = now.stats[0], rstd = now.stats[1];
    float g[NC][kVec], xh[NC][kVec];
    float sum_g = 0.0f, sum_gx = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int left = there ? cols - (c * Shape::kSpan + lane * kVec) : 0;
      eight_values(now.codes[c], inverse_of(now.scale[c]), now.lo[c], xh[c]);
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        const bool in = (WHOLE ? 0 : e) < left;      // columns behind the last one and a row that is not there add nothing
        const float d = in ? (float)now.dy[c][e] : 0.0f;
        xh[c][e] = in ? (xh[c][e] - mean) * rstd : 0.0f;
        dw[c][e] = __builtin_fmaf(d, xh[c][e], dw[c][e]);
        db[c][e] += d;
        g[c][e] = d * w[c][e];
        sum_g += g[c][e];
        sum_gx = __builtin_fmaf(g[c][e], xh[c][e], sum_gx);
      }
    }
    const float mg = row_sum<LPR>(sum_g, shared, turn) * per_col;
    const float mgx = row_sum<LPR>(sum_gx, shared + 2 * Shape::kWaves, turn) * per_col;
    turn ^= 1;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int col = c * Shape::kSpan + lane * kVec;
#pragma unroll
      for (int e = 0; e < kVec; e++) g[c][e] = rstd * (g[c][e] - __builtin_fmaf(xh[c][e], mgx, mg));
      store_cols<T, WHOLE>(dx + row * cols + col, there ? cols - col : 0, g[c]);
    }
  }
  if (!partial) return;
  // rows of the wave first (lanes LPR apart own the same columns), then the workgroup's waves
#pragma unroll
  for (int c = 0; c < NC; c++) {
#pragma unroll
    for (int which = 0; which < 2; which++) {
      float (&s)[kVec] = which ? db[c] : dw[c];
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        if (kFold >= 4) s[e] += __shfl_xor(s[e], 16);
        if (kFold >= 2) s[e] += __shfl_xor(s[e], 32);
      }
      float* out = partial + ((int64_t)blockIdx.x * 2 + which) * cols;
      const int col = c * Shape::kSpan + lane * kVec;
      if constexpr (kAcross > 1) {
        const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
        __syncthreads();
        if (l < LPR)
#pragma unroll
          for (int e = 0; e < kVec; e++) folded[(wave * kVec + e) * 64 + l] = s[e];
        __syncthreads();
        // a wave per column of the pieces
        if (l < LPR && c * Shape::kSpan + l * kVec + wave < cols) {
          static_assert(kAcross == kVec, "eight waves, eight columns");
          float total = 0.0f;
#pragma unroll
          for (int from = 0; from < kAcross; from++) total += folded[(from * kVec + wave) * 64 + l];
          out[c * Shape::kSpan + l * kVec + wave] = total;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; e++)
          if (col + e < cols) out[col + e] = s[e];
      }
    }
  }
}

// out[c] = sum of partial[p][c], in the same order whatever runs beside it; `stride` values from one partial row to the next.  16 waves per 64
// columns: 512 rows of 4096 columns 4.6 us, bound by the latency of a few loads in turn.
template <typename T>
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* __restrict__ partial, int count, int64_t stride, int cols,
                                                        T* __restrict__ out0, T* __restrict__ out1) {
  __shared__ float shared[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  const float* in = partial + (int64_t)blockIdx.y * cols;
  float s = 0.0f;
  if (col < cols) {
    // eight rows' loads at a time: one after the other they would be all latency (1024 partial rows of 1024 columns: 20 us)
    int p = wave;
    for (; p + 7 * 16 < count; p += 8 * 16) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) v[u] = in[(int64_t)(p + u * 16) * stride + col];
#pragma unroll
      for (int u = 0; u < 8; u++) s += v[u];
    }
    for (; p < count; p += 16) s += in[(int64_t)p * stride + col];
  }
  shared[wave][threadIdx.x & 63] = s;
  __syncthreads();
  if (wave == 0 && col < cols) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) s += shared[w][threadIdx.x];
    T* out = blockIdx.y ? out1 : out0;
    if (out) out[col] = rounded<T>(s);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// dz = dy act'(z) from the checkpoint of z, and the column sums of dz before they are rounded.  A thread owns 8 columns and walks
// down `per` rows; without codes (no activation) dz is dy, copied to the products' stride where `dz` is given.  dz is rounded to T, as dy and
// a checkpoint's values are where they enter a product: the matrix instructions of 16-bit types take nothing wider, and those of floats run
// at a tenth of their rate.  (bfloat16, 16384 rows: an error of 0.0024 of the outputs' norm where products of unrounded dz have 0.0017.)
// Bound by memory, 32768x4096 halves GELU 132 us (5.1 TB/s), SiLU 130, sums alone 47 (5.7); 16384x1024 24, 22 and 11.  32 lanes and 256
// columns to a row, as the codes' groups are, 16 lanes where 128 columns are enough: 401408x96 halves 56 (3.4).  In floats GELU's exact error
// function counts where a quarter of the lanes has no columns: 401408x96 112 us (3.1 TB/s), SiLU 87 (4.0); 32768x4096 272 (4.5) and 253 (4.8).
// ---------------------------------------------------------------------------------------------------------------------------------
template <typename T, int LANES, bool WHOLE>
__global__ __launch_bounds__(256) void activation_backward_kernel(const T* __restrict__ dy, int64_t lddy, const uint8_t* __restrict__ codes,
                                                                  int64_t ldc, const float* __restrict__ scale,
                                                                  const float* __restrict__ mn, int act, int64_t rows, int cols, int per,
                                                                  T* __restrict__ dz, int64_t lddz, float* __restrict__ partial) {
  constexpr int kRows = 256 / LANES;      // at a time
  __shared__ float shared[4][LANES][kVec + 1];
  const int lane = threadIdx.x % LANES, strip = threadIdx.x / LANES;
  const int col = (int)blockIdx.x * kGroup + lane * kVec;
  const int groups = (cols + kGroup - 1) / kGroup;
  const int64_t first = (int64_t)blockIdx.y * per, last = first + per < rows ? first + per : rows;
  const int64_t left = cols - col;
  float sum[kVec];
#pragma unroll
  for (int e = 0; e < kVec; e++) sum[e] = 0.0f;
  if (left > 0) {
    for (int64_t row = first + strip; row < last; row += kRows) {
      float g[kVec], z[kVec];
      load_cols<T, WHOLE>(dy + row * lddy + col, left, g);
      if (codes) {
        const int64_t group = row * groups + blockIdx.x;
        eight_values(*(const u32x2*)(codes + row * ldc + col), inverse_of(scale[group]), mn[group], z);
#pragma unroll
        for (int e = 0; e < kVec; e++) g[e] = WHOLE || e < left ? g[e] * slope<std::is_same<T, float>::value>(z[e], act) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < kVec; e++) sum[e] += g[e];
      if (dz) store8(dz + row * lddz + col, g);
    }
  }
  if (!partial) return;
  // over the rows of a wave, then over the waves
#pragma unroll
  for (int o = LANES; o < 64; o *= 2)
#pragma unroll
    for (int e = 0; e < kVec; e++) sum[e] += __shfl_xor(sum[e], o);
  if ((threadIdx.x & 63) < LANES)
#pragma unroll
    for (int e = 0; e < kVec; e++) shared[threadIdx.x >> 6][lane][e] = sum[e];
  __syncthreads();
  const int c = (int)threadIdx.x;
  if (c < LANES * kVec && (int)blockIdx.x * kGroup + c < cols) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) s += shared[w][c / kVec][c % kVec];
    partial[(int64_t)blockIdx.y * cols + (int)blockIdx.x * kGroup + c] = s;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Products.  out[i][j] = sum over r of A(i, r) B(j, r), each operand in one of two layouts: rows of it contiguous along r (x and W of
// the forward pass, dz of dx), or contiguous along i or j, one memory row per r (W of dx; dz and the checkpoint of dW).
//
// A workgroup owns a tile of BM x BN and walks along r in steps of 128 bytes of T, two of which are in LDS: while one is multiplied the next
// one arrives, straight from memory (16 bytes a lane, no registers).  A checkpoint's codes pass through registers, where they
// become values of T.  A lane's fragment is 8 values along r of 16-bit types (one 16x16x32 product) or 4 floats (four 16x16x4
// products).  Operands contiguous along r are read 16 bytes at a time, the others through the transposing LDS read (16-bit) or value by value
// (float).  LDS is addressed so that neither kind of read meets a bank twice: contiguous rows of 128 bytes permute their eight
// 16-byte pieces by the row's number, the others their blocks of 16 columns.
//
// B supplies the matrix instruction's rows and A its columns, so that a lane holds four consecutive j of one i.
//
// 8192x8192x8192 halves: forward 785 to 890 us (1233 to 1400 TFLOP/s), dx 786, dW from codes 1045 (1055), forward with GELU and its codes 837;
// 16384x1024x4096: 109, 103, 140 to 150, 165; floats 4096x4096x4096 976 (141 of the 152 that the library's product reaches).  Zeros in place of
// numbers take 695: the clock drops under the matrix units' load, and the numbers' share of the time is power's.  Without its loads the forward
// product takes 582, so what else there is to gain lies in the loads' path to LDS.
// Measured and not taken, forward 8192x8192x8192: four steps of 64 bytes in LDS with a barrier to each 877 to 912 us; two groups of waves that take
// turns between loading and multiplying 897; four waves of 128x128 873, with a slower epilogue.  16384x1024x4096: stores that bypass the caches
// 174 to 182 us where plain ones take 170.
// ---------------------------------------------------------------------------------------------------------------------------------
[[maybe_unused]] constexpr uint32_t kNowhere = 0x80000000u;   // beyond every window: such a load gives zero

struct ProductArgs {
  const void* a;
  const void* b;
  int64_t lda, ldb;
  int rows, cols;          // of the output
  int64_t depth;           // values along r
  void* out;
  int64_t ldo;
  // a checkpoint as B
  const float* b_scale;
  const float* b_min;
  int b_groups;
  // the forward pass
  const void* bias;
  const void* residual;
  int64_t ldr;
  int act;
  uint8_t* codes;
  int64_t ldc;
  float* scale;
  float* mn;
  // tiles
  int tiles_i, tiles_j, splits;
  int64_t per_split;       // depth of a split, a multiple of the step
  bool wide;               // output rows, and the residual's, are whole 16-byte pieces
};

template <typename T>
struct Mma {
  static constexpr int kStep = 128 / (int)sizeof(T);       // values along r of a step
  static constexpr int kBlock = 16 * (int)sizeof(T);        // bytes of 16 columns
  using Frag = std::conditional_t<std::is_same<T, bf16>::value, bf16x8, std::conditional_t<std::is_same<T, f16>::value, f16x8, f32x4>>;
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    if constexpr (std::is_same<T, bf16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    if constexpr (std::is_same<T, f16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int t = 0; t < 4; t++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
    }
    return c;
  }
  // by which the blocks of 16 columns of a tile row of `COUNT` columns are permuted: the rows that one read touches (16-bit: four
  // neighbours, and those 8 further on; float: every fourth) lie in different banks
  template <int COUNT>
  static __device__ __forceinline__ uint32_t block_turn(uint32_t r) {
    if (sizeof(T) == 4) return (r >> 2) & 3;
    if (COUNT == 64) return ((r >> 1) & 1) | (((r >> 3) & 1) << 1);      // two rows fill the banks: four blocks each
    return (r & 3) | (((r >> 3) & 1) << 2);
  }
};

// what is left of an operand from a tile's corner on, as a buffer that loads beyond it give zero from
struct Window {
  const char* base = nullptr;
  int64_t left = 0;
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    const int64_t n = left <= 0 ? 0 : left > 0x7fffffff ? 0x7fffffff : left;
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)n, 0x00020000);
  }
  __device__ __forceinline__ void advance(int64_t bytes) {
    base += bytes;
    left -= bytes;
  }
};
// buffer_load with its destination in LDS: lane l's BYTES go to `to` + l BYTES (two bytes: 4 l; M0 holds `to`, the same for the wave).  It writes no
// register.  As asm, because the compiler waits for every such load that it knows of before it reads LDS through the transposing
// read, whichever memory that reads; the product counts them itself, and waits before the barrier that gives a step's memory free.
template <int BYTES>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, uint32_t offset, lds_u8* to) {
#ifdef __HIP_DEVICE_COMPILE__
  static_assert(BYTES == 16 || BYTES == 4 || BYTES == 2, "a quad, a word or half a word, which takes a word of LDS");
  if constexpr (BYTES == 2)
    asm volatile("s_nop 0\n\tbuffer_load_ushort %0, %1, 0 offen lds" : : "v"(offset), "s"(rsrc), "{m0}"((uint32_t)(uintptr_t)to) : "memory");
  else if constexpr (BYTES == 16)
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(offset), "s"(rsrc), "{m0}"((uint32_t)(uintptr_t)to) : "memory");
  else
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" : : "v"(offset), "s"(rsrc), "{m0}"((uint32_t)(uintptr_t)to) : "memory");
#endif
}

// Loads a step of COUNT rows (contiguous along r) or COUNT columns (strided) into LDS: an instruction of a wave fills 1 KB.
template <typename T, int COUNT, bool STRIDED, int WAVES>
struct TileLoad {
  static constexpr int kLoads = COUNT * 128 / 1024 / WAVES, kEsz = (int)sizeof(T);
  static_assert(kLoads >= 1, "a wave takes at least one load");
  Window window;
  int64_t step = 0;
  uint32_t at[kLoads];
  int piece = 0, left = 0;     // contiguous: the lane's first value along r, and the values that are left from the step on
  int wave = 0;
  // up to the end of the piece: a window drops a value of 16 bits whose neighbour in the word lies beyond it
  static __device__ __forceinline__ int64_t whole(int64_t n) { return (n + 16 / kEsz - 1) / (16 / kEsz) * (16 / kEsz); }
  __device__ __forceinline__ void set_up(int64_t ld, int w, int lane) {
    wave = w;
    if (STRIDED) {
      constexpr int W = COUNT * kEsz, RPL = 1024 / W, BLK = Mma<T>::kBlock;
      step = (int64_t)Mma<T>::kStep * ld * kEsz;
#pragma unroll
      for (int q = 0; q < kLoads; q++) {
        const uint32_t r = (wave * kLoads + q) * RPL + lane * 16 / W, within = lane * 16 % W;
        at[q] = r * (uint32_t)(ld * kEsz) + ((within / BLK) ^ Mma<T>::template block_turn<COUNT>(r)) * BLK + within % BLK;
      }
    } else {
      step = 128;
      piece = ((lane & 7) ^ (lane >> 3)) * (16 / kEsz);
#pragma unroll
      for (int q = 0; q < kLoads; q++) at[q] = ((wave * kLoads + q) * 8 + (lane >> 3)) * (uint32_t)(ld * kEsz) + piece * kEsz;
    }
  }
  // from row or column i0 of `count` and value r0 of `depth` on
  __device__ __forceinline__ void start(const void* p, int64_t ld, int i0, int count, int64_t depth, int64_t r0) {
    if (STRIDED) {
      window.base = (const char*)p + (r0 * ld + i0) * kEsz;
      window.left = ((depth - 1 - r0) * ld + whole(count) - i0) * kEsz;
    } else {
      window.base = (const char*)p + (i0 * ld + r0) * kEsz;
      window.left = ((count - 1 - i0) * ld + whole(depth) - r0) * kEsz;
      left = (int)(depth - r0 < 0x7fffffff ? depth - r0 : 0x7fffffff);
    }
  }
  __device__ __forceinline__ void stop() { window.left = 0; }
  // load q of the wave's; after the last one the step is done
  __device__ __forceinline__ void issue(int q, lds_u8* to) const {
    load_to_lds<16>(window.rsrc(), !STRIDED && piece >= left ? kNowhere : at[q], to + (wave * kLoads + q) * 1024);
  }
  __device__ __forceinline__ void advance() {
    window.advance(step);
    left -= Mma<T>::kStep;
  }
};

// Codes of a checkpoint, one memory row per r, as a strided step of values: 16 codes of a row are one piece, a block of the step.
template <typename T, int COUNT, int WAVES>
struct CodeLoad {
  static constexpr int kTotal = Mma<T>::kStep * COUNT / 16, kPieces = kTotal > WAVES * 64 ? kTotal / (WAVES * 64) : 1;
  static constexpr int kAcross = COUNT / 16, kApart = WAVES * 64 / kAcross;     // pieces of a row; rows between a thread's pieces
  static constexpr int kLoads = 0;            // straight to LDS
  Window codes, scale, mn;
  int64_t step = 0, stat_step = 0;
  uint32_t at = 0, stat_at = 0, apart = 0, stat_apart = 0;    // of the thread's first piece, and to the next one
  int left = 0, held_left = 0;                                // rows from the next step on, and from the one that is held on
  u32x4 held[kPieces];
  float s[kPieces], lo[kPieces];
  __device__ __forceinline__ void set_up(const ProductArgs& p) {
    const int t = threadIdx.x, row = t / kAcross, col = t % kAcross * 16, groups = p.b_groups;
    step = Mma<T>::kStep * p.ldb;
    stat_step = (int64_t)Mma<T>::kStep * groups * 4;
    at = row * (uint32_t)p.ldb + col;
    stat_at = row * groups * 4;
    apart = kApart * (uint32_t)p.ldb;
    stat_apart = kApart * groups * 4;
  }
  __device__ __forceinline__ void start(const ProductArgs& p, int j0, int64_t depth, int64_t r0) {
    left = (int)(depth - r0 < 0x7fffffff ? depth - r0 : 0x7fffffff);
    const int groups = p.b_groups;
    codes.base = (const char*)p.b + r0 * p.ldb + j0;
    codes.left = (depth - r0) * p.ldb - j0;
    scale.base = (const char*)(p.b_scale + r0 * groups + j0 / kGroup);      // one group of columns: no tile is wider than one or meets two
    mn.base = (const char*)(p.b_min + r0 * groups + j0 / kGroup);
    scale.left = mn.left = ((depth - r0) * groups - j0 / kGroup) * 4;
  }
  __device__ __forceinline__ void stop() { codes.left = scale.left = mn.left = 0; }
  __device__ __forceinline__ void fetch() {
    held_left = left;
    const __amdgpu_buffer_rsrc_t c = codes.rsrc(), f = scale.rsrc(), m = mn.rsrc();
#pragma unroll
    for (int q = 0; q < kPieces; q++) {
      held[q] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(c, (int)(at + q * apart), 0, 0));
      s[q] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(f, (int)(stat_at + q * stat_apart), 0, 0));
      lo[q] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(m, (int)(stat_at + q * stat_apart), 0, 0));
    }
    codes.advance(step);
    scale.advance(stat_step);
    mn.advance(stat_step);
    left -= Mma<T>::kStep;
  }
  // Part k of the thread's values: 16 bytes of them.  One part behind each few products: all at once, after the barrier, they keep the matrix
  // units waiting.
  static constexpr int kParts = kPieces * (int)sizeof(T);
  __device__ __forceinline__ void put(int k, lds_u8* tile) const {
    const int t = threadIdx.x, q = k / (int)sizeof(T), h = k % (int)sizeof(T);
    if (kTotal < WAVES * 64 && t >= kTotal) return;      // floats of a small tile: fewer pieces than threads
    const uint32_t row = t / kAcross + q * kApart, block = t % kAcross;
    const float inv = (int)row < held_left ? inverse_of(s[q]) : 0.0f;      // rows behind the last one: zeros
    lds_u8* to = tile + row * (COUNT * (int)sizeof(T)) + (block ^ Mma<T>::template block_turn<COUNT>(row)) * Mma<T>::kBlock + 16 * h;
    if constexpr (sizeof(T) == 2) {
      typedef T T8 __attribute__((ext_vector_type(8)));
      T8 v;
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = (T)value_of(held[q][2 * h + (e >> 2)], e & 3, inv, lo[q]);
      *(__attribute__((address_space(3))) T8*)to = v;
    } else {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = value_of(held[q][h], e, inv, lo[q]);
      *(__attribute__((address_space(3))) f32x4*)to = v;
    }
  }
};

// A lane's fragment of 16 rows (contiguous) or columns (strided) of half kk of a step, from row or column `first` on
template <typename T, int COUNT, bool STRIDED>
struct TileRead {
  using Frag = typename Mma<T>::Frag;
  static constexpr int W = COUNT * (int)sizeof(T), BLK = Mma<T>::kBlock;
  static __device__ __forceinline__ Frag get(const lds_u8* tile, int first, int kk, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!STRIDED) {
      return *(const __attribute__((address_space(3))) Frag*)(tile + first * 128 + i * 128 + (((kk * 4 + g) ^ (i & 7)) * 16));
    } else if constexpr (sizeof(T) == 2) {
      const uint32_t turn = Mma<T>::template block_turn<COUNT>(g * 8 + (i >> 2));     // the same in every row that the lane reads
      const lds_u8* p = tile + (g * 8 + (i >> 2)) * W + (((first / 16) ^ turn) * BLK) + (i & 3) * 8 + kk * 32 * W;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * W));
      return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const lds_u8* p = tile + (kk * 16 + 4 * g) * W + (((first / 16) ^ g) * BLK) + i * 4;
      f32x4 v;
#pragma unroll
      for (int t = 0; t < 4; t++) v[t] = *(const __attribute__((address_space(3))) float*)(p + t * W);
      return v;
    }
  }
};

// Workgroups go to the 8 XCDs in turn: each XCD has a run of consecutive tiles, which its workgroups take side by side, and a run walks
// down `kTall` tile rows before it moves to the next tile column, so that the tiles that an XCD works on at a time share rows of A and
// B in its L2.
constexpr int kTall = 8;
struct Tile {
  int i, j, split;
};
__device__ __forceinline__ bool tile_of(const ProductArgs& p, int turn, Tile& t) {
  const uint32_t total = (uint32_t)p.tiles_i * p.tiles_j * p.splits, xcd = blockIdx.x % 8;
  const uint32_t mine = total / 8 + (xcd < total % 8), beside = gridDim.x / 8 + (xcd < gridDim.x % 8);
  const uint32_t k = blockIdx.x / 8 + turn * beside;
  if (k >= mine) return false;
  uint32_t at = xcd * (total / 8) + (xcd < total % 8 ? xcd : total % 8) + k;
  const uint32_t tiles = p.tiles_i * p.tiles_j;
  t.split = at / tiles;
  at -= t.split * tiles;
  const uint32_t band = kTall * p.tiles_j, which = at / band, in = at - which * band;
  const uint32_t tall = (uint32_t)p.tiles_i - which * kTall < kTall ? p.tiles_i - which * kTall : kTall;
  t.i = which * kTall + in % tall;
  t.j = in / tall;
  return true;
}

// A lane holds four consecutive columns of blocks n and n + 1 of a row; lanes 16 apart the columns beside them.  Afterwards it holds eight
// consecutive columns of block n + (g & 1), from column 8 (g >> 1) on, g = lane / 16.  The same again undoes it.
__device__ __forceinline__ void swap_rows16(uint32_t& a, uint32_t& b) {
#ifdef __HIP_DEVICE_COMPILE__
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
#endif
}
__device__ __forceinline__ void swap_rows32(uint32_t& a, uint32_t& b) {
#ifdef __HIP_DEVICE_COMPILE__
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
#endif
}
template <typename T>
__device__ __forceinline__ u32x2 rounded4(f32x4 v) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 o;
#pragma unroll
  for (int e = 0; e < 4; e++) o[e] = rounded<T>(v[e]);
  return __builtin_bit_cast(u32x2, o);
}
template <typename T>
__device__ __forceinline__ float low_value(uint32_t word) {
  if constexpr (std::is_same<T, float>::value) return __builtin_bit_cast(float, word);
  if constexpr (std::is_same<T, bf16>::value) return __builtin_bit_cast(float, word << 16);
  if constexpr (std::is_same<T, f16>::value) return (float)__builtin_bit_cast(f16, (uint16_t)word);
  return 0.0f;
}
template <typename T>
__device__ __forceinline__ f32x4 widened4(uint32_t a, uint32_t b) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const T4 o = __builtin_bit_cast(T4, u32x2{a, b});
  return f32x4{(float)o[0], (float)o[1], (float)o[2], (float)o[3]};
}

enum { B_ROWS = 0, B_STRIDED = 1, B_CODES = 2 };

template <typename T, int BM, int BN, int WI, int WJ, bool A_STRIDED, int B_KIND, int ACT, bool CODES>
__global__ __launch_bounds__(WI* WJ * 64) void product_kernel(ProductArgs p) {
  constexpr int WAVES = WI * WJ, MI = BM / WI / 16, MH = MI / 2, NJ = BN / WJ / 16;
  constexpr bool FORWARD = B_KIND == B_ROWS && ACT != ACT_UNFINISHED, CODED = B_KIND == B_CODES;
  using Frag = typename Mma<T>::Frag;
  using LoadA = TileLoad<T, BM, A_STRIDED, WAVES>;
  using LoadB = std::conditional_t<CODED, CodeLoad<T, BN, WAVES>, TileLoad<T, BN, B_KIND == B_STRIDED, WAVES>>;
  constexpr int kA = BM * 128, kB = BN * 128;
  __shared__ __attribute__((aligned(1024))) uint8_t memory[2 * (kA + kB)];
  lds_u8* const a_ring = (lds_u8*)memory;
  lds_u8* const b_ring = a_ring + 2 * kA;
  // the tiles' biases, a word each, by turns: loads run up to three tiles ahead where tiles have but one step
  __shared__ uint32_t biases[4][FORWARD ? BN : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ;

  // s_waitcnt's operands: for all loads and stores, and for all but the newest stores, as many as every wave makes of a whole tile
  constexpr int kStores = MI * NJ / (sizeof(T) == 2 ? 2 : 1);
  static_assert(kStores < 64, "s_waitcnt counts to 63");
  constexpr int kWaitAll = 7 << 4 | 15 << 8, kWaitStored = (kStores & 15) | (kStores >> 4) << 14 | kWaitAll;
  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // What is loaded runs two steps ahead of what is multiplied (a checkpoint's codes, through their registers, three), from tile to tile;
  // behind the last tile there is nothing left to load, and the loads give zeros.
  LoadA a;
  LoadB b;
  a.set_up(p.lda, wave, lane);
  if constexpr (CODED)
    b.set_up(p);
  else
    b.set_up(p.ldb, wave, lane);
  auto steps_of = [&](const Tile& tile, int64_t& r0, int64_t& end) __attribute__((always_inline)) {
    r0 = tile.split * p.per_split;
    end = r0 + p.per_split < p.depth ? r0 + p.per_split : p.depth;
    return (int)((end - r0 + Mma<T>::kStep - 1) / Mma<T>::kStep);
  };
  struct Feed {
    int turn = 0, left = 0;
  } feed, code_feed;
  auto feed_tile = [&]() __attribute__((always_inline)) {
    if (feed.left == 0) {
      Tile next;
      feed.left = 0x7fffffff;
      if (tile_of(p, feed.turn, next)) {
        int64_t r0, end;
        feed.left = steps_of(next, r0, end);
        a.start(p.a, p.lda, next.i * BM, p.rows, end, r0);
        if constexpr (!CODED) b.start(p.b, p.ldb, next.j * BN, p.cols, end, r0);
        if constexpr (FORWARD) {
          Window bias;
          if (p.bias) {
            bias.base = (const char*)p.bias + next.j * BN * (int)sizeof(T);
            bias.left = (p.cols - next.j * BN) * (int64_t)sizeof(T);
          }
          const int part = wave % (BN / 64) * 64;
          load_to_lds<sizeof(T)>(bias.rsrc(), (part + lane) * (uint32_t)sizeof(T), (lds_u8*)&biases[feed.turn & 3][part]);
        }
        feed.turn++;
      } else {
        a.stop();
        if constexpr (!CODED) b.stop();
      }
    }
    feed.left--;
  };
  auto fetch_codes = [&]() __attribute__((always_inline)) {
    if constexpr (CODED) {
      if (code_feed.left == 0) {
        Tile next;
        code_feed.left = 0x7fffffff;
        if (tile_of(p, code_feed.turn, next)) {
          int64_t r0, end;
          code_feed.left = steps_of(next, r0, end);
          b.start(p, next.j * BN, end, r0);
          code_feed.turn++;
        } else {
          b.stop();
        }
      }
      code_feed.left--;
      b.fetch();
    }
  };
  // The loads of a step, spread over the products: the card's address units take 64 bytes a clock, and a wave that waits for them to take
  // one more issues no product.
  auto issue_a = [&](int n, int of, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int q = n * LoadA::kLoads / of; q < (n + 1) * LoadA::kLoads / of; q++) a.issue(q, a_ring + slot * kA);
    if (n + 1 == of) a.advance();
  };
  auto issue_b = [&](int n, int of, int slot) __attribute__((always_inline)) {
    if constexpr (!CODED) {
#pragma unroll
      for (int q = n * LoadB::kLoads / of; q < (n + 1) * LoadB::kLoads / of; q++) b.issue(q, b_ring + slot * kB);
      if (n + 1 == of) b.advance();
    }
  };
  auto put_codes = [&](int n, int of, int slot) __attribute__((always_inline)) {
    if constexpr (CODED) {
#pragma unroll
      for (int k = n * LoadB::kParts / of; k < (n + 1) * LoadB::kParts / of; k++) b.put(k, b_ring + slot * kB);
    }
  };

  f32x4 acc[MI][NJ];
  // A step is four phases: (first, second half of the fragments along r) x (upper, lower half of the wave's rows).  Each phase
  // multiplies what was read from LDS in the phase before and reads for the next; B's fragments are replaced one by one as soon as their
  // last product is under way, which leaves the registers to the sums.  After the third phase nothing is left to read of
  // the step: once every wave is there and the next step has arrived, its memory takes the step after the next.
  Frag fa[2][MH], fb[NJ];
  auto read_a = [&](int slot, int kk, int half, Frag (&f)[MH]) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < MH; m++) f[m] = TileRead<T, BM, A_STRIDED>::get(a_ring + slot * kA, wi * (BM / WI) + (half * MH + m) * 16, kk, lane);
  };
  auto read_b = [&](int slot, int kk, int n) __attribute__((always_inline)) {
    fb[n] = TileRead<T, BN, B_KIND != B_ROWS>::get(b_ring + slot * kB, wj * (BN / WJ) + n * 16, kk, lane);
  };
  auto multiply = [&](const Frag (&x)[MH], int half, int n) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < MH; m++) acc[half * MH + m][n] = Mma<T>::run(fb[n], x[m], acc[half * MH + m][n]);
  };

  // A workgroup takes tile after tile, and the stores of a whole tile go on while the next one is multiplied: they are newer than the
  // loads of its first two steps.
  Tile tile;
  if (!tile_of(p, 0, tile)) return;
  fetch_codes();
#pragma unroll
  for (int slot = 0; slot < 2; slot++) {
    feed_tile();
    issue_a(0, 1, slot);
    issue_b(0, 1, slot);
    put_codes(0, 1, slot);
    fetch_codes();
  }
  __builtin_amdgcn_s_waitcnt(kWaitAll);
  meet();
  bool stored = false;
  int now = 0;      // the step's place
  for (int turn = 1;; turn++) {
#pragma unroll
    for (int m = 0; m < MI; m++)
#pragma unroll
      for (int n = 0; n < NJ; n++) acc[m][n] = f32x4{0, 0, 0, 0};
    int64_t r0, end;
    const int steps = steps_of(tile, r0, end);
    read_a(now, 0, 0, fa[0]);
#pragma unroll
    for (int n = 0; n < NJ; n++) read_b(now, 0, n);
    for (int t = 0; t < steps; t++) {
      const int next = now ^ 1;
      read_a(now, 0, 1, fa[1]);
#pragma unroll
      for (int n = 0; n < NJ; n++) {
        multiply(fa[0], 0, n);
        if (t > 0) issue_b(n, NJ, next);
        __builtin_amdgcn_sched_barrier(0);
      }
      read_a(now, 1, 0, fa[0]);
#pragma unroll
      for (int n = 0; n < NJ; n++) {
        multiply(fa[1], 1, n);
        read_b(now, 1, n);
        __builtin_amdgcn_sched_barrier(0);
      }
      read_a(now, 1, 1, fa[1]);
#pragma unroll
      for (int n = 0; n < NJ; n++) multiply(fa[0], 0, n);
      __builtin_amdgcn_sched_barrier(0);
      if (stored && t == 0)
        __builtin_amdgcn_s_waitcnt(kWaitStored);
      else
        __builtin_amdgcn_s_waitcnt(kWaitAll);
      meet();
      // behind a tile's last step these read the next tile's first one, which is read again when that begins
      read_a(next, 0, 0, fa[0]);
      feed_tile();
#pragma unroll
      for (int n = 0; n < NJ; n++) {
        multiply(fa[1], 1, n);
        read_b(next, 0, n);
        put_codes(n, NJ, now);
        issue_a(n, NJ, now);
        if constexpr (CODED) {
          // one product, then as much of the conversion as it leaves time for
#pragma unroll
          for (int m = 0; m < MH; m++) {
            __builtin_amdgcn_sched_group_barrier(8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(2, 8, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      fetch_codes();
      now = next;
    }
    issue_b(0, 1, now ^ 1);      // of the step that the last one made room for: ahead of the stores
    const Tile done = tile;
    const bool more = tile_of(p, turn, tile);
    if (!more) __builtin_amdgcn_s_waitcnt(kWaitAll);      // no load is on its way to LDS when the workgroup ends
    __builtin_amdgcn_sched_barrier(0);

    const int i0 = done.i * BM, j0 = done.j * BN;
    // the lane's number, counted again: it and the addresses below are made here, not before the loop, where they would take registers from it
    // (with the codes of 256 x 256 there is not one left)
    uint32_t all = ~0u;
    asm volatile("" : "+s"(all));
    const int l = (int)__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0));
    const int i_lane = i0 + wi * (BM / WI) + (l & 15);
    const int j_wave = j0 + wj * (BN / WJ);
    const int j_lane = j_wave + (l >> 4) * 4;
    const bool whole = i0 + BM <= p.rows && j0 + BN <= p.cols;
    if constexpr (FORWARD) {
#pragma unroll
      for (int n = 0; n < NJ; n++) {
        const u32x4 held = *(const u32x4*)&biases[(turn - 1) & 3][wj * (BN / WJ) + n * 16 + (l >> 4) * 4];
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = low_value<T>(held[e]);
#pragma unroll
        for (int m = 0; m < MI; m++) acc[m][n] += v;
      }
      if constexpr (CODES) {
        static_assert(BN == kGroup, "a tile's row is one group");
        {
          // a tile's row is one group: least and most of the wave's columns, then over the waves side by side; one thread per row
          // makes the scale
          __shared__ float ends[2][WJ][BM];
          __shared__ f32x2 ready[BM];
#pragma unroll
          for (int m = 0; m < MI; m++) {
            float lo = __builtin_inff(), hi = -__builtin_inff();
#pragma unroll
            for (int n = 0; n < NJ; n++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (whole || j_lane + n * 16 + e < p.cols) lo = __builtin_fminf(lo, acc[m][n][e]), hi = __builtin_fmaxf(hi, acc[m][n][e]);
            lo = __builtin_fminf(lo, __shfl_xor(lo, 16));
            hi = __builtin_fmaxf(hi, __shfl_xor(hi, 16));
            lo = __builtin_fminf(lo, __shfl_xor(lo, 32));
            hi = __builtin_fmaxf(hi, __shfl_xor(hi, 32));
            if (l < 16) {
              const int at = wi * (BM / WI) + m * 16 + l;
              ends[0][wj][at] = lo;
              ends[1][wj][at] = hi;
            }
          }
          meet();
          if (threadIdx.x < BM) {
            const int at = threadIdx.x;
            float lo = ends[0][0][at], hi = ends[1][0][at];
#pragma unroll
            for (int w = 1; w < WJ; w++) lo = __builtin_fminf(lo, ends[0][w][at]), hi = __builtin_fmaxf(hi, ends[1][w][at]);
            const float s = scale_of(lo, hi);
            ready[at] = f32x2{s, lo};
            if (i0 + at < p.rows) {
              const int64_t g = (int64_t)(i0 + at) * p.tiles_j + done.j;
              p.scale[g] = s;
              p.mn[g] = lo;
            }
          }
          meet();
#pragma unroll
          for (int m = 0; m < MI; m++) {
            const int at = wi * (BM / WI) + m * 16 + (l & 15);
            const f32x2 r = ready[at];
            uint32_t c[NJ];
#pragma unroll
            for (int n = 0; n < NJ; n++) c[n] = four_codes(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3], r[1], r[0]);
            uint8_t* out = p.codes + (int64_t)(i0 + at) * p.ldc;
            if (whole) {
              static_assert(NJ == 4, "16 bytes of a lane are four blocks' codes");
              swap_rows16(c[0], c[1]);
              swap_rows16(c[2], c[3]);
              swap_rows32(c[0], c[2]);
              swap_rows32(c[1], c[3]);
              *(u32x4*)(out + j_wave + (l >> 4) * 16) = u32x4{c[0], c[1], c[2], c[3]};
            } else if (i0 + at < p.rows) {
#pragma unroll
              for (int n = 0; n < NJ; n++)
                if (j_lane + n * 16 < p.cols) *(uint32_t*)(out + j_lane + n * 16) = c[n];
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    const bool partial = ACT == ACT_UNFINISHED || (!FORWARD && p.splits > 1);
    {
      if (partial || (p.wide && sizeof(T) == 4)) {      // 16 bytes are the four columns that a lane holds
#pragma unroll
        for (int m = 0; m < MI; m++) {
          const int64_t i = i_lane + m * 16;
          float* out = (float*)p.out + (partial ? (int64_t)done.split * p.rows + i : i) * p.ldo + j_lane;
          const float* residual = FORWARD && p.residual ? (const float*)p.residual + i * p.ldr + j_lane : nullptr;
#pragma unroll
          for (int n = 0; n < NJ; n++)
            if (whole || (i < p.rows && j_lane + n * 16 < p.cols)) {
              f32x4 v = activated4<T, ACT>(acc[m][n]);
              if (FORWARD && residual) v += *(const f32x4*)(residual + n * 16);
              *(f32x4*)(out + n * 16) = v;
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else if (p.wide) {
        if constexpr (sizeof(T) == 2) {
          const int j_eight = j_wave + ((l >> 4) & 1) * 16 + (l >> 5) * 8;
#pragma unroll
          for (int m = 0; m < MI; m++) {
            const int64_t i = i_lane + m * 16;
            T* out = (T*)p.out + i * p.ldo + j_eight;
            const T* residual = FORWARD && p.residual ? (const T*)p.residual + i * p.ldr + j_eight : nullptr;
#pragma unroll
            for (int n = 0; n < NJ; n += 2) {
              const bool there = whole || (i < p.rows && j_eight + n * 16 < p.cols);
              f32x4 v0 = activated4<T, ACT>(acc[m][n]), v1 = activated4<T, ACT>(acc[m][n + 1]);
              if (FORWARD && residual) {
                u32x4 r = {0, 0, 0, 0};
                if (there) r = *(const u32x4*)(residual + n * 16);
                uint32_t r0 = r[0], r1 = r[1], r2 = r[2], r3 = r[3];
                swap_rows16(r0, r2);
                swap_rows16(r1, r3);
                v0 += widened4<T>(r0, r1);
                v1 += widened4<T>(r2, r3);
              }
              const u32x2 a0 = rounded4<T>(v0), a1 = rounded4<T>(v1);
              uint32_t r0 = a0[0], r1 = a0[1], r2 = a1[0], r3 = a1[1];
              swap_rows16(r0, r2);
              swap_rows16(r1, r3);
              if (there) *(u32x4*)(out + n * 16) = u32x4{r0, r1, r2, r3};
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else {
#pragma unroll
        for (int m = 0; m < MI; m++) {
          const int64_t i = i_lane + m * 16;
          if (i >= p.rows) continue;
#pragma unroll
          for (int n = 0; n < NJ; n++) {
            const f32x4 v = activated4<T, ACT>(acc[m][n]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int j = j_lane + n * 16 + e;
              if (j >= p.cols) continue;
              ((T*)p.out)[i * p.ldo + j] = rounded<T>(FORWARD && p.residual ? v[e] + (float)((const T*)p.residual)[i * p.ldr + j] : v[e]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (!more) return;
    stored = whole && (partial || p.wide);
  }
}

// the parts' sums [splits][rows][ldp] added up, in order: 4 parts of 4096x1024 floats 12.6 us (5.8 TB/s, from the caches in part)
template <typename T>
__global__ __launch_bounds__(256) void join_splits_kernel(const float* __restrict__ partial, int splits, int64_t rows, int cols, int ldp,
                                                          T* __restrict__ out) {
  const int per = ldp / 4;
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = unit / per;
  const int col = (int)(unit - row * per) * 4;
  if (row >= rows) return;
  f32x4 v = *(const f32x4*)(partial + row * ldp + col);
  for (int s = 1; s < splits; s++) v += *(const f32x4*)(partial + (s * rows + row) * ldp + col);
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (col + e < cols) out[row * cols + col + e] = rounded<T>(v[e]);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// The forward product of a few rows (up to 64): the weights are read once, straight into the matrix instruction's fragments, by
// workgroups of 16 output columns whose waves share the depth; their sums meet in LDS.  Bound by the weights' bytes: 1x4096x4096 halves 10 us
// (3.4 TB/s), 16x4096x16384 36.5 (3.7), 16x8192x8192 floats 79 (3.4); 1x1024x4096 4.6, launch and latency.  16 waves to a workgroup are no
// faster (9.7 and 9.1 for 1x4096x4096, 11.6 and 9.6 the other way for 24x1024x4096 floats).
// ---------------------------------------------------------------------------------------------------------------------------------
template <typename T, bool WHOLE>
__device__ __forceinline__ typename Mma<T>::Frag fragment_of(const T* row, int64_t k, int64_t depth) {
  using Frag = typename Mma<T>::Frag;
  constexpr int N = 16 / (int)sizeof(T);
  typedef T Unaligned __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  Frag f;
  if (WHOLE) {
    if (k < depth) return *(const Frag*)(row + k);
#pragma unroll
    for (int e = 0; e < N; e++) f[e] = (T)0.0f;
  } else {
    if (k + N <= depth) return *(const Unaligned*)(row + k);
#pragma unroll
    for (int e = 0; e < N; e++) f[e] = k + e < depth ? row[k + e] : (T)0.0f;
  }
  return f;
}
template <typename T, int MT, bool WHOLE>
__global__ __launch_bounds__(512) void few_rows_kernel(ProductArgs p) {
  constexpr int WAVES = 8;
  constexpr int SPAN = 4 * 16 / (int)sizeof(T);      // values along r of a fragment step of the wave
  __shared__ f32x4 shared[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int j0 = blockIdx.x * 16;
  const int j = j0 + i < p.cols ? j0 + i : p.cols - 1;
  const T* w = (const T*)p.b + j * p.ldb;
  const T* x[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int row = m * 16 + i < p.rows ? m * 16 + i : p.rows - 1;
    x[m] = (const T*)p.a + row * p.lda;
    acc[m] = f32x4{0, 0, 0, 0};
  }
  // the waves take steps of 64 bytes in turn, UNROLL of them with all their loads on the way
  constexpr int UNROLL = !WHOLE || MT == 4 ? 4 : 8;
  const int split = blockIdx.y;
  const int64_t first = split * p.per_split, end = first + p.per_split < p.depth ? first + p.per_split : p.depth;
  for (int64_t k0 = first + wave * SPAN; k0 < end; k0 += (int64_t)WAVES * SPAN * UNROLL) {
    typename Mma<T>::Frag fw[UNROLL], fx[UNROLL][MT];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const int64_t k = k0 + u * WAVES * SPAN + g * (16 / (int)sizeof(T));
      fw[u] = fragment_of<T, WHOLE>(w, k, end);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
#pragma unroll
      for (int m = 0; m < MT; m++) fx[u][m] = fragment_of<T, WHOLE>(x[m], k0 + u * WAVES * SPAN + g * (16 / (int)sizeof(T)), end);
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
#pragma unroll
      for (int m = 0; m < MT; m++) acc[m] = Mma<T>::run(fw[u], fx[u][m], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < MT; m++) shared[wave][m][lane] = acc[m];
  __syncthreads();
  for (int m = wave; m < MT; m += WAVES) {
    f32x4 v = shared[0][m][lane];
#pragma unroll
    for (int s = 1; s < WAVES; s++) v += shared[s][m][lane];
    const int row = m * 16 + i;
    if (row >= p.rows) continue;
    if (p.splits) {      // to be finished
      if (j0 + g * 4 < p.cols) *(f32x4*)((float*)p.out + ((int64_t)split * p.rows + row) * p.ldo + j0 + g * 4) = v;
      continue;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int c = j0 + g * 4 + e;
      if (c >= p.cols) continue;
      float o = v[e] + (p.bias ? (float)((const T*)p.bias)[c] : 0.0f);
      o = activated<std::is_same<T, float>::value>(o, p.act);
      if (p.residual) o += (float)((const T*)p.residual)[row * p.ldr + c];
      ((T*)p.out)[row * p.ldo + c] = rounded<T>(o);
    }
  }
}

// A forward product that was cut along its depth, or whose tiles are no whole groups of columns: the parts [splits][rows][ldp] added up, in order, then what
// the products' epilogues do.  32 lanes own a group of 256 columns.  1024x4096 halves with GELU and codes, one part: 28 us with its product.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ partial, int splits, int64_t ldp, const T* __restrict__ bias,
                                                     const T* __restrict__ residual, int64_t ldr, int act, int64_t rows, int cols, int groups,
                                                     T* __restrict__ y, uint8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale,
                                                     float* __restrict__ mn) {
  const int64_t unit = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t row = unit / groups;
  const int g = (int)(unit - row * groups), lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int col = g * kGroup + lane * kVec, n = cols - col;
  f32x4 part[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
  for (int h = 0; h < 2; h++)
    if (n > 4 * h) {
      part[h] = *(const f32x4*)(partial + row * ldp + col + 4 * h);
      for (int s = 1; s < splits; s++) part[h] += *(const f32x4*)(partial + (s * rows + row) * ldp + col + 4 * h);
    }
  float v[kVec], b[kVec];
  if (bias)
    load_cols<T, false>(bias + col, n, b);
  else
    for (int e = 0; e < kVec; e++) b[e] = 0.0f;
#pragma unroll
  for (int e = 0; e < kVec; e++) v[e] = part[e >> 2][e & 3] + b[e];
  if (codes) {
    float lo = __builtin_inff(), hi = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < kVec; e++)
      if (e < n) lo = __builtin_fminf(lo, v[e]), hi = __builtin_fmaxf(hi, v[e]);
    lo = over_lanes<Least, 32>(lo);
    hi = over_lanes<Most, 32>(hi);
    const float s = scale_of(lo, hi);
    if (n > 0)
      *(u32x2*)(codes + row * ldc + col) = u32x2{four_codes(v[0], v[1], v[2], v[3], lo, s), four_codes(v[4], v[5], v[6], v[7], lo, s)};
    if (lane == 0) {
      scale[unit] = s;
      mn[unit] = lo;
    }
  }
#pragma unroll
  for (int e = 0; e < kVec; e++) v[e] = activated<std::is_same<T, float>::value>(v[e], act);
  if (residual) {
    load_cols<T, WHOLE>(residual + row * ldr + col, n, b);
#pragma unroll
    for (int e = 0; e < kVec; e++) v[e] += b[e];
  }
  store_cols<T, WHOLE>(y + row * cols + col, n, v);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Host side of the ABI
// ---------------------------------------------------------------------------------------------------------------------------------
inline void fresh_launch() { (void)hipGetLastError(); }
inline int launch_status() { return hipGetLastError() == hipSuccess ? GACT_OK : GACT_ELAUNCH; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
inline bool known(int dtype) { return dtype == GACT_F32 || dtype == GACT_F16 || dtype == GACT_BF16; }
inline bool blocks_fit(int64_t blocks) { return blocks > 0 && blocks <= 0x7fffffff; }
// A launch takes fewer than 2^32 threads along x: `blocks` workgroups along x where they fit, else in as many equal rows along y as it takes
// (block_of() counts them; up to a row's worth behind the last one find nothing to do)
inline dim3 grid_of(int64_t blocks, int threads) {
  const int64_t most = 0xffffffff / threads, down = (blocks + most - 1) / most;
  return dim3((unsigned)((blocks + down - 1) / down), (unsigned)down);
}
constexpr int64_t kMostCols = GACT_LAYER_MAX_COLS;

// rows that every lane's piece lies whole and aligned in
inline bool whole_rows(const void* p, int dtype, int64_t cols, int64_t ld) {
  return aligned16(p) && cols % kVec == 0 && ld * size_of(dtype) % 16 == 0;
}
inline bool codes_fit(const void* codes, int64_t cols, int64_t ldc) { return aligned16(codes) && ldc % 16 == 0 && ldc >= cols; }

template <typename F>
int with_type(int dtype, F&& f) {
  switch (dtype) {
    case GACT_F32: return f(float{});
    case GACT_F16: return f(f16{});
    default: return f(bf16{});
  }
}

// Threads of a row, its pieces per thread, and the rows that a thread of the forward pass takes at a time: few threads, whose sums need no
// exchange through LDS, as far as the registers hold the row.  us forward / backward, and with other numbers of threads:
//   401408x96 floats 71 / 73, 32 threads 91 / 124           100352x192 halves 32 / 32, 64 threads 50 / 51
//   65536x512 halves 40 / 43, 32 threads 41 / 46            65536x1024 halves 72 / 81, 256 threads 110 / 194
//   16384x2048 halves 37 / 40, 64 and 256 threads the other way round 46 / 66: the forward pass has no sums to keep between rows
//   16384x4096 halves 67 / 88, 512 threads 72 / 93          8192x8192 halves 71 / 93, 256 threads 84 / 96
template <bool BACKWARD, typename F>
int with_row_shape(int64_t cols, F&& f) {
  using std::integral_constant;
  if (cols <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
  if (cols <= 256) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
  if (cols <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
  if (cols <= 1024) return f(integral_constant<int, 64>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
  if constexpr (BACKWARD) {
    if (cols <= 2048) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
  } else {
    if (cols <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{}, integral_constant<int, 1>{});
  }
  if (cols <= 4096) return f(integral_constant<int, 256>{}, integral_constant<int, 2>{}, integral_constant<int, 1>{});
  if (cols <= 8192) return f(integral_constant<int, 512>{}, integral_constant<int, 2>{}, integral_constant<int, 1>{});
  return f(integral_constant<int, 512>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
}
// workgroups of a layer norm's backward pass: each leaves one row of partial sums.  At most 512, 256 of them / 1024 of them instead: 401408x96
// floats 71 us, 101 / 75; 65536x1024 halves 78, 75 / 84; 16384x4096 83, 125 / 99.  Rows beyond 4096 columns fill a compute unit by
// themselves, at most 256: 8192x8192 87, with 512 99
inline int64_t norm_blocks(int64_t rows, int64_t cols) {
  const int64_t at_a_time = cols <= 128 ? kNormThreads / 16 : cols <= 256 ? kNormThreads / 32 : cols <= 2048 ? kNormThreads / 64 : 1;
  const int64_t needed = (rows + at_a_time - 1) / at_a_time, most = cols <= 4096 ? 512 : 256;
  if (needed <= kComputeUnits) return needed;
  const int64_t shared = needed / 8 > kComputeUnits ? needed / 8 : kComputeUnits;     // enough turns to pay for a row of partial sums
  return shared < most ? shared : most;
}
// lanes of a group where groups are walked one by one: a row of at most 128 columns needs 16 of them (401408x96 floats,
// checkpoint 36 us, with 32 lanes 65, GELU's backward pass 120 and 198; halves 35 and 65, 56 and 91)
inline int lanes_of(int64_t cols) { return cols <= 128 ? 16 : 32; }
// rows of a workgroup of the activation's backward pass: about 2048 workgroups; 65536x1024 halves 73 us, with 1024 of them 82, with 4096 73;
// 16384x4096 72, 83 and 74; 16384x1024 23, 25 and 25
inline int64_t strip_rows(int64_t rows, int64_t cols) {
  const int64_t across = (cols + kGroup - 1) / kGroup;
  int64_t per = (rows * across + 2047) / 2048;
  const int64_t at_a_time = 256 / lanes_of(cols);
  per = (per + at_a_time - 1) / at_a_time * at_a_time;
  if (per < at_a_time) per = at_a_time;
  while ((rows + per - 1) / per > 65535) per *= 2;
  return per;
}

template <typename T>
int sum_rows(const float* partial, int64_t count, int64_t stride, int64_t cols, int parts, void* out0, void* out1, hipStream_t s) {
  hipLaunchKernelGGL((sum_rows_kernel<T>), dim3((unsigned)((cols + 63) / 64), (unsigned)parts), dim3(1024), 0, s, partial, (int)count,
                     stride, (int)cols, (T*)out0, (T*)out1);
  return launch_status();
}

inline int64_t padded4(int64_t cols) { return (cols + 3) / 4 * 4; }

template <typename T, int BM, int BN, int WI, int WJ, bool AS, int BK, int ACT = ACT_NONE, bool CODES = false>
int launch_product(ProductArgs& p, int splits, int64_t per_split, hipStream_t s) {
  p.tiles_i = (p.rows + BM - 1) / BM;
  p.tiles_j = (p.cols + BN - 1) / BN;
  p.splits = splits;
  p.per_split = per_split;
  const int64_t tiles = (int64_t)p.tiles_i * p.tiles_j * splits;
  if (!blocks_fit(tiles)) return GACT_ELIMIT;
  constexpr int kSlots = kComputeUnits * slots_per_cu(BM, BN);      // workgroups that the card holds at a time
  const int64_t blocks = tiles < kSlots ? tiles : kSlots;
  auto kernel = product_kernel<T, BM, BN, WI, WJ, AS, BK, ACT, CODES>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(WI * WJ * 64), 0, s, p);
  return launch_status();
}

template <typename T, int ACT>
int forward_product(ProductArgs& p, int side, hipStream_t s) {
  const int64_t step = Mma<T>::kStep, depth = (p.depth + step - 1) / step * step;
  // the pre-activation's codes need a whole group of columns in a tile; without an activation nobody asks for them
  if constexpr (ACT != ACT_NONE) {
    if (p.codes) {
      if constexpr (sizeof(T) == 2)
        if (coded_rows_of(sizeof(T) == 4, p.rows, p.cols) == 256)
          return launch_product<T, 256, 256, 2, 4, false, B_ROWS, ACT, true>(p, 1, depth, s);
      return launch_product<T, 128, 256, 2, 4, false, B_ROWS, ACT, true>(p, 1, depth, s);
    }
  }
  if constexpr (sizeof(T) == 2)
    if (side == 256) return launch_product<T, 256, 256, 2, 4, false, B_ROWS, ACT>(p, 1, depth, s);
  if (side == 128) return launch_product<T, 128, 128, 2, 2, false, B_ROWS, ACT>(p, 1, depth, s);
  return launch_product<T, 64, 64, 2, 2, false, B_ROWS, ACT>(p, 1, depth, s);
}

template <typename T, bool AS, int BK>
int backward_product(ProductArgs& p, int dtype, void* workspace, hipStream_t s) {
  const Cut t = cut_of(dtype, BK == B_CODES, p.rows, p.cols, p.depth, 256, 256);
  void* out = p.out;
  if (t.parts > 1) {
    if (!workspace || !aligned16(workspace)) return GACT_EALIGN;
    p.out = workspace;
    p.ldo = padded4(p.cols);
  }
  int rc = GACT_ESHAPE;
  if constexpr (sizeof(T) == 2)
    if (t.side == 256) rc = launch_product<T, 256, 256, 2, 4, AS, BK>(p, t.parts, t.per_part, s);
  if (t.side == 128) rc = launch_product<T, 128, 128, 2, 2, AS, BK>(p, t.parts, t.per_part, s);
  if (t.side == 64) rc = launch_product<T, 64, 64, 2, 2, AS, BK>(p, t.parts, t.per_part, s);
  if (rc != GACT_OK || t.parts == 1) return rc;
  const int64_t blocks = ((int64_t)p.rows * (p.ldo / 4) + 255) / 256;
  if (!blocks_fit(blocks)) return GACT_ELIMIT;
  hipLaunchKernelGGL((join_splits_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, (const float*)workspace, t.parts, (int64_t)p.rows,
                     p.cols, (int)p.ldo, (T*)out);
  return launch_status();
}

inline bool layer_sizes(int64_t rows, int64_t a, int64_t b) {
  return rows >= 0 && rows <= GACT_LAYER_MAX_ROWS && a > 0 && a <= kMostCols && b > 0 && b <= kMostCols;
}
// operands that the products load 16 bytes at a time
inline bool operand_fits(const void* p, int64_t ld, int dtype, int64_t cols) {
  return aligned16(p) && ld * size_of(dtype) % 16 == 0 && ld >= cols && ld <= 4 * kMostCols && cols * size_of(dtype) % 16 == 0;
}
}  // namespace

extern "C" {

int gact_checkpoint(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* codes, int64_t ldc, float* scale, float* mn,
                    void* stream) {
  if (!known(dtype) || !layer_sizes(rows, cols, 1) || (ldx < cols && rows > 1)) return GACT_EINVAL;
  if (rows == 0) return GACT_OK;
  if (!x || !codes || !scale || !mn) return GACT_EINVAL;
  if (!codes_fit(codes, cols, ldc)) return GACT_EALIGN;
  const int64_t groups = (cols + kGroup - 1) / kGroup, units = 256 / lanes_of(cols), blocks = (rows * groups + units - 1) / units;
  if (!blocks_fit(blocks)) return GACT_ELIMIT;
  fresh_launch();
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const bool whole = whole_rows(x, dtype, cols, ldx);
    auto kernel = lanes_of(cols) == 16 ? (whole ? checkpoint_kernel<T, 16, true> : checkpoint_kernel<T, 16, false>)
                                       : (whole ? checkpoint_kernel<T, 32, true> : checkpoint_kernel<T, 32, false>);
    hipLaunchKernelGGL(kernel, grid_of(blocks, 256), dim3(256), 0, (hipStream_t)stream, (const T*)x, rows, (int)cols, ldx, (int)groups,
                       (uint8_t*)codes, ldc, scale, mn);
    return launch_status();
  });
}

int gact_restore(const void* codes, int64_t ldc, const float* scale, const float* mn, int dtype, int64_t rows, int64_t cols, void* out,
                 void* stream) {
  if (!known(dtype) || !layer_sizes(rows, cols, 1)) return GACT_EINVAL;
  if (rows == 0) return GACT_OK;
  if (!codes || !scale || !mn || !out) return GACT_EINVAL;
  if (!codes_fit(codes, cols, ldc) || !aligned16(out)) return GACT_EALIGN;
  const int64_t groups = (cols + kGroup - 1) / kGroup, units = 256 / lanes_of(cols), blocks = (rows * groups + units - 1) / units;
  if (!blocks_fit(blocks)) return GACT_ELIMIT;
  fresh_launch();
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const bool whole = whole_rows(out, dtype, cols, cols);
    auto kernel = lanes_of(cols) == 16 ? (whole ? restore_kernel<T, 16, true> : restore_kernel<T, 16, false>)
                                       : (whole ? restore_kernel<T, 32, true> : restore_kernel<T, 32, false>);
    hipLaunchKernelGGL(kernel, grid_of(blocks, 256), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)codes, ldc, scale, mn, rows,
                       (int)cols, (int)groups, (T*)out);
    return launch_status();
  });
}

int gact_pad_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* out, int64_t ldo, void* stream) {
  if (!known(dtype) || !layer_sizes(rows, cols, 1) || (ldx < cols && rows > 1)) return GACT_EINVAL;
  if (rows == 0) return GACT_OK;
  if (!x || !out) return GACT_EINVAL;
  if (!aligned16(out) || ldo % kVec || ldo < cols || ldo > kMostCols + kVec) return GACT_EALIGN;
  const int64_t blocks = (rows * (ldo / kVec) + 255) / 256;
  if (!blocks_fit(blocks)) return GACT_ELIMIT;
  fresh_launch();
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    hipLaunchKernelGGL((pad_rows_kernel<T>), grid_of(blocks, 256), dim3(256), 0, (hipStream_t)stream, (const T*)x, rows, (int)cols, ldx,
                       (T*)out, (int)ldo);
    return launch_status();
  });
}

int gact_norm_forward(const void* x, int64_t ldx, const void* weight, const void* bias, int dtype, int64_t rows, int64_t cols, float eps,
                      void* y, void* codes, int64_t ldc, float* scale, float* mn, float* stats, void* stream) {
  if (!known(dtype) || !layer_sizes(rows, cols, 1) || cols > GACT_NORM_MAX_COLS || (ldx < cols && rows > 1)) return GACT_EINVAL;
  if (rows == 0) return GACT_OK;
  if (!x || !y || (codes && (!scale || !mn || !stats))) return GACT_EINVAL;
  if (codes && !codes_fit(codes, cols, ldc)) return GACT_EALIGN;
  fresh_launch();
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const bool whole = whole_rows(x, dtype, cols, ldx) && whole_rows(y, dtype, cols, cols) && aligned16(weight) && aligned16(bias);
    return with_row_shape<false>(cols, [&](auto lpr, auto nc, auto at_a_time) {
      constexpr int LPR = decltype(lpr)::value, NC = decltype(nc)::value, U = decltype(at_a_time)::value;
      auto run = [&](auto kernel, int u) {
        const int64_t blocks = (rows + RowShape<LPR>::kRows * u - 1) / (RowShape<LPR>::kRows * u);
        if (!blocks_fit(blocks)) return GACT_ELIMIT;
        hipLaunchKernelGGL(kernel, grid_of(blocks, RowShape<LPR>::kThreads), dim3(RowShape<LPR>::kThreads), 0, (hipStream_t)stream, (const T*)x, ldx,
                           (const T*)weight, (const T*)bias, rows, (int)cols, 1.0f / (float)cols, eps, (T*)y, (uint8_t*)codes, ldc, scale, mn,
                           stats);
        return launch_status();
      };
      // few rows: one at a time, on as many compute units as there are (2000x1024 halves 5.7 us, two at a time 6.6; 8000x512 7.0, four 8.5;
      // 25088x384, above the bound, four 19.8)
      if (U > 1 && rows < (int64_t)kComputeUnits * 4 * RowShape<LPR>::kRows * U)
        return whole ? run(norm_forward_kernel<T, LPR, NC, 1, true>, 1) : run(norm_forward_kernel<T, LPR, NC, 1, false>, 1);
      return whole ? run(norm_forward_kernel<T, LPR, NC, U, true>, U) : run(norm_forward_kernel<T, LPR, NC, U, false>, U);
    });
  });
}

int64_t gact_norm_workspace_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : norm_blocks(rows, cols) * 2 * cols * (int64_t)sizeof(float);
}

int gact_norm_backward(const void* dy, int64_t lddy, const void* weight, const void* codes, int64_t ldc, const float* scale,
                       const float* mn, const float* stats, int dtype, int64_t rows, int64_t cols, void* dx, void* dweight, void* dbias,
                       float* workspace, void* stream) {
  if (!known(dtype) || !layer_sizes(rows, cols, 1) || rows == 0 || cols > GACT_NORM_MAX_COLS || (lddy < cols && rows > 1)) return GACT_EINVAL;
  if (!dy || !codes || !scale || !mn || !stats || !dx) return GACT_EINVAL;
  const bool sums = dweight || dbias;
  if (sums && !workspace) return GACT_EINVAL;
  if (!codes_fit(codes, cols, ldc)) return GACT_EALIGN;
  fresh_launch();
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const bool whole = whole_rows(dy, dtype, cols, lddy) && whole_rows(dx, dtype, cols, cols) && aligned16(weight);
    const int64_t blocks = norm_blocks(rows, cols);
    const int rc = with_row_shape<true>(cols, [&](auto lpr, auto nc, auto) {
      constexpr int LPR = decltype(lpr)::value, NC = decltype(nc)::value;
      auto kernel = whole ? norm_backward_kernel<T, LPR, NC, true> : norm_backward_kernel<T, LPR, NC, false>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(SharedRows<LPR>::kThreads), 0, (hipStream_t)stream, (const T*)dy, lddy,
                         (const T*)weight, (const uint8_t*)codes, ldc, scale, mn, stats, rows, (int)cols, 1.0f / (float)cols, (T*)dx,
                         sums ? workspace : nullptr);
      return launch_status();
    });
    if (rc != GACT_OK || !sums) return rc;
    return sum_rows<T>(workspace, blocks, 2 * cols, cols, 2, dweight, dbias, (hipStream_t)stream);
  });
}

int64_t gact_linear_workspace_bytes(int dtype, int64_t rows, int64_t inner, int64_t outer, int codes) {
  if (!known(dtype) || rows <= 0 || inner <= 0 || outer <= 0) return 0;
  int64_t parts = 0;
  for (bool whole : {false, true}) {
    const Forward f = forward_of(dtype, rows, inner, outer, codes != 0, whole);
    if (f.finished && f.cut.parts > parts) parts = f.cut.parts;
  }
  return parts * rows * padded4(outer) * (int64_t)sizeof(float);
}

int gact_linear(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr,
                int activation, int dtype, int64_t rows, int64_t inner, int64_t outer, void* y, void* codes, int64_t ldc, float* scale,
                float* mn, void* workspace, void* stream) {
  if (!known(dtype) || !layer_sizes(rows, inner, outer) || activation < GACT_ACT_NONE || activation > GACT_ACT_SILU) return GACT_EINVAL;
  if (rows == 0) return GACT_OK;
  if (!x || !weight || !y || (codes && (!scale || !mn || activation == GACT_ACT_NONE)) || (residual && ldr < outer && rows > 1)) return GACT_EINVAL;
  if ((rows > 1 && ldx < inner) || (outer > 1 && ldw < inner)) return GACT_EINVAL;
  if (codes && !codes_fit(codes, outer, ldc)) return GACT_EALIGN;
  const bool whole = operand_fits(x, ldx, dtype, inner) && operand_fits(weight, ldw, dtype, inner);
  const Forward f = forward_of(dtype, rows, inner, outer, codes != nullptr, whole);
  if (!whole && !f.few) return GACT_EALIGN;
  if (f.finished && (!workspace || !aligned16(workspace))) return GACT_EALIGN;
  const int64_t groups = (outer + kGroup - 1) / kGroup, units = (rows * groups + 7) / 8;
  if (!blocks_fit(units)) return GACT_ELIMIT;
  ProductArgs p = {};
  p.a = x;
  p.b = weight;
  p.lda = ldx;
  p.ldb = ldw;
  p.rows = (int)rows;
  p.cols = (int)outer;
  p.depth = inner;
  p.out = f.finished ? workspace : y;
  p.ldo = f.finished ? padded4(outer) : outer;
  p.bias = bias;
  p.residual = residual;
  p.ldr = ldr;
  p.act = activation;
  p.codes = (uint8_t*)codes;
  p.ldc = ldc;
  p.scale = scale;
  p.mn = mn;
  p.per_split = f.cut.per_part;
  p.splits = f.finished ? f.cut.parts : 0;
  const bool wide = whole_rows(y, dtype, outer, outer) && (!residual || whole_rows(residual, dtype, outer, ldr));
  p.wide = wide;
  fresh_launch();
  hipStream_t s = (hipStream_t)stream;
  return with_type(dtype, [&](auto zero) -> int {
    using T = decltype(zero);
    int rc;
    if (f.few) {
      auto run = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        auto kernel = whole ? few_rows_kernel<T, MT, true> : few_rows_kernel<T, MT, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((outer + 15) / 16), (unsigned)f.cut.parts), dim3(512), 0, s, p);
        return launch_status();
      };
      rc = rows <= 16 ? run(std::integral_constant<int, 1>{}) : rows <= 32 ? run(std::integral_constant<int, 2>{}) : run(std::integral_constant<int, 4>{});
    } else if (f.finished) {
      rc = launch_product<T, 64, 64, 2, 2, false, B_ROWS, ACT_UNFINISHED>(p, f.cut.parts, f.cut.per_part, s);
    } else {
      switch (activation) {
        case GACT_ACT_GELU: return forward_product<T, ACT_GELU>(p, f.cut.side, s);
        case GACT_ACT_GELU_TANH: return forward_product<T, ACT_GELU_TANH>(p, f.cut.side, s);
        case GACT_ACT_SILU: return forward_product<T, ACT_SILU>(p, f.cut.side, s);
        default: return forward_product<T, ACT_NONE>(p, f.cut.side, s);
      }
    }
    if (rc != GACT_OK || !f.finished) return rc;
    auto kernel = wide ? finish_kernel<T, true> : finish_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)units), dim3(256), 0, s, (const float*)workspace, f.cut.parts, padded4(outer), (const T*)bias,
                       (const T*)residual, ldr, activation, rows, (int)outer, (int)groups, (T*)y, (uint8_t*)codes, ldc, scale, mn);
    return launch_status();
  });
}

int64_t gact_activation_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t per = strip_rows(rows, cols);
  return (rows + per - 1) / per * cols * (int64_t)sizeof(float);
}

int gact_activation_backward(const void* dy, int64_t lddy, const void* codes, int64_t ldc, const float* scale, const float* mn,
                             int activation, int dtype, int64_t rows, int64_t cols, void* dz, int64_t lddz, void* dbias, float* workspace,
                             void* stream) {
  if (!known(dtype) || !layer_sizes(rows, cols, 1) || rows == 0 || (lddy < cols && rows > 1)) return GACT_EINVAL;
  if (activation < GACT_ACT_NONE || activation > GACT_ACT_SILU || (activation != GACT_ACT_NONE && !codes)) return GACT_EINVAL;
  if (!dy || (codes && (!scale || !mn)) || (dbias && !workspace) || (!dz && !dbias)) return GACT_EINVAL;
  if ((codes && !codes_fit(codes, cols, ldc)) || (dz && (!aligned16(dz) || lddz % kVec || lddz < cols || lddz >= cols + kVec))) return GACT_EALIGN;
  const int64_t per = strip_rows(rows, cols), strips = (rows + per - 1) / per;
  fresh_launch();
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const bool whole = whole_rows(dy, dtype, cols, lddy);
    auto kernel = lanes_of(cols) == 16 ? (whole ? activation_backward_kernel<T, 16, true> : activation_backward_kernel<T, 16, false>)
                                       : (whole ? activation_backward_kernel<T, 32, true> : activation_backward_kernel<T, 32, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((cols + kGroup - 1) / kGroup), (unsigned)strips), dim3(256), 0, (hipStream_t)stream,
                       (const T*)dy, lddy, (const uint8_t*)codes, ldc, scale, mn, activation, rows, (int)cols, (int)per, (T*)dz, lddz,
                       dbias ? workspace : nullptr);
    const int rc = launch_status();
    if (rc != GACT_OK || !dbias) return rc;
    return sum_rows<T>(workspace, strips, cols, cols, 1, dbias, nullptr, (hipStream_t)stream);
  });
}

int64_t gact_product_workspace_bytes(int dtype, int64_t rows, int64_t cols, int64_t depth) {
  if (!known(dtype) || rows <= 0 || cols <= 0 || depth <= 0) return 0;
  const int parts = cut_of(dtype, false, rows, cols, depth, 256, 256).parts, of_codes = cut_of(dtype, true, rows, cols, depth, 256, 256).parts;
  const int64_t most = parts > of_codes ? parts : of_codes;
  return most == 1 ? 0 : most * rows * padded4(cols) * (int64_t)sizeof(float);
}

int gact_product(const void* a, int64_t lda, const void* b, int64_t ldb, int dtype, int64_t rows, int64_t depth, int64_t cols, void* out,
                 void* workspace, void* stream) {
  if (!known(dtype) || !layer_sizes(rows, depth, cols)) return GACT_EINVAL;
  if (rows == 0) return GACT_OK;
  if (!a || !b || !out) return GACT_EINVAL;
  const int64_t padded = (cols * size_of(dtype) + 15) / 16 * 16 / size_of(dtype);
  if (!operand_fits(a, lda, dtype, (depth * size_of(dtype) + 15) / 16 * 16 / size_of(dtype)) || !operand_fits(b, ldb, dtype, padded)) return GACT_EALIGN;
  ProductArgs p = {};
  p.a = a;
  p.b = b;
  p.lda = lda;
  p.ldb = ldb;
  p.rows = (int)rows;
  p.cols = (int)cols;
  p.depth = depth;
  p.out = out;
  p.ldo = cols;
  p.wide = whole_rows(out, dtype, cols, cols);
  fresh_launch();
  return with_type(dtype, [&](auto zero) { return backward_product<decltype(zero), false, B_STRIDED>(p, dtype, workspace, (hipStream_t)stream); });
}

int gact_checkpoint_product(const void* grad, int64_t ldg, const void* codes, int64_t ldc, const float* scale, const float* mn, int dtype,
                            int64_t rows, int64_t outer, int64_t inner, void* out, void* workspace, void* stream) {
  if (!known(dtype) || !layer_sizes(rows, outer, inner) || rows == 0) return GACT_EINVAL;
  if (!grad || !codes || !scale || !mn || !out) return GACT_EINVAL;
  const int64_t padded = (outer * size_of(dtype) + 15) / 16 * 16 / size_of(dtype);
  // offsets within a step's rows are 32 bits wide, of the codes as of the other operand
  if (!operand_fits(grad, ldg, dtype, padded) || !codes_fit(codes, inner, ldc) || ldc > 4 * kMostCols) return GACT_EALIGN;
  ProductArgs p = {};
  p.a = grad;
  p.b = codes;
  p.lda = ldg;
  p.ldb = ldc;
  p.rows = (int)outer;
  p.cols = (int)inner;
  p.depth = rows;
  p.out = out;
  p.ldo = inner;
  p.b_scale = scale;
  p.b_min = mn;
  p.b_groups = (int)((inner + kGroup - 1) / kGroup);
  p.wide = whole_rows(out, dtype, inner, inner);
  fresh_launch();
  return with_type(dtype, [&](auto zero) { return backward_product<decltype(zero), true, B_CODES>(p, dtype, workspace, (hipStream_t)stream); });
}

}  // extern "C"
