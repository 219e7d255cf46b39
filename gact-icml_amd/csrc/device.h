// What the kernels' sources share: types, rounding, loads from memory straight to LDS, and the host side's small checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gact_hip.h"

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

// The workgroup's number in a launch of grid_of(): beyond 2^32 threads a launch goes on along y
__device__ __forceinline__ int64_t block_of() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// A result is a float before it is rounded to T, in every kernel and whichever way it is stored: the empty statement keeps the compiler from making
// one instruction of the last operation and its rounding to a half, which rounds once and differs in one of 2^13 values - of rows at one address and
// not of the same rows at another.
template <typename T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (std::is_same<T, f16>::value) asm("" : "+v"(v));
  return (T)v;
}

[[maybe_unused]] constexpr int kVec = 8;   // columns of a lane's piece
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

[[maybe_unused]] constexpr uint32_t kNowhere = 0x80000000u;   // beyond every window: such a load gives zero

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

__device__ __forceinline__ void swap_rows32(uint32_t& a, uint32_t& b) {
#ifdef __HIP_DEVICE_COMPILE__
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
#endif
}

// ---- host side ----
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
template <typename F>
int with_type(int dtype, F&& f) {
  switch (dtype) {
    case GACT_F32: return f(float{});
    case GACT_F16: return f(f16{});
    default: return f(bf16{});
  }
}

}  // namespace
