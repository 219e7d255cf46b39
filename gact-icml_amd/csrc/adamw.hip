// AdamW's step over many tensors in one launch for each 72 of them, with states in floats or in 8 bits.
//
// 8 bits: groups of 256 elements share the largest magnitude of either state.  The first moment's codes are spaced by the square, the second's by the
// fourth power, so that sqrt(v), by which the step is divided, has the same spacing as m: a step of 0.8 % next to the largest, and values down to
// (1/255)^4 of the largest of v.  A v above zero never becomes zero, which would blow its step up.
#include <math.h>

#include "device.h"

namespace {

constexpr int kGroup = 256, kLanes = kGroup / kVec;
constexpr int kTensors = 72;      // of a launch: its arguments hold 4 KB
constexpr float kSquare = 16129.0f, kFourth = 4228250624.0f;      // 127^2, and 255^4 as a float
constexpr float kLeastM = 1e-30f, kLeastV = 1e-28f;      // the quotients below do not overflow above these

struct Tensors {
  gact_adamw_tensor t[kTensors];
  uint32_t first[kTensors + 1];      // block of each, eight groups to a block
  int count;
};
struct Rates {
  float beta1, rest1, beta2, rest2, eps, keep, step, root;      // keep = 1 - lr decay, step = lr / (1 - beta1^step), root = 1 / sqrt(1 - beta2^step)
};
struct Step {
  gact_adamw_options o;
  Rates r;
};

__host__ __device__ inline Rates rates_of(const gact_adamw_options& o, double lr, double step) {
  Rates r;
  r.beta1 = (float)o.beta1;
  r.rest1 = (float)(1.0 - o.beta1);
  r.beta2 = (float)o.beta2;
  r.rest2 = (float)(1.0 - o.beta2);
  r.eps = (float)o.eps;
  r.keep = (float)(1.0 - lr * o.decay);
  r.step = (float)(lr / (1.0 - pow(o.beta1, step)));
  r.root = (float)(1.0 / sqrt(1.0 - pow(o.beta2, step)));
  return r;
}

__device__ __forceinline__ int tensor_of(const Tensors& a, uint32_t block) {
  int low = 0, high = a.count;      // first[low] <= block < first[high]
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (a.first[middle] <= block)
      low = middle;
    else
      high = middle;
  }
  return low;
}

// The larger of two magnitudes as their bits order them: a NaN above everything, which fmaxf would pass over
struct MostBits {
  static __device__ __forceinline__ float of(float a, float b) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    return __builtin_bit_cast(float, x > y ? x : y);
  }
};
// how many of the borders (k - 1/2)^2, k = 1, 2 .., are at most w: the hardware's root is off by a unit in the last place, the squares are exact
__device__ __forceinline__ float nearest_root(float w) {
  float c = __builtin_floorf(__builtin_amdgcn_sqrtf(w) + 0.5f);
  const float below = c - 0.5f, above = c + 0.5f;
  if (w < below * below) c -= 1.0f;
  if (w >= above * above) c += 1.0f;
  return c;
}
// the same of (k - 1/2)^4, whose roundings to float are taken into account: w - p is exact next to the border
__device__ __forceinline__ bool reaches(float w, float half) {
  const float square = half * half, p = square * square, rest = __builtin_fmaf(square, square, -p);
  return w - p >= rest;
}
__device__ __forceinline__ float nearest_fourth_root(float w) {
  float c = __builtin_floorf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(w)) + 0.5f);
  if (c > 0.0f && !reaches(w, c - 0.5f)) c -= 1.0f;
  if (reaches(w, c + 0.5f)) c += 1.0f;
  return c;
}
__device__ __forceinline__ uint32_t byte_of(uint32_t w, int e) { return (w >> (8 * e)) & 0xff; }
// what a code stands for
__device__ __forceinline__ float first_of(uint32_t code, float unit) {
  const float c = (float)(int8_t)code;
  return c * __builtin_fabsf(c) * unit;
}
__device__ __forceinline__ float second_of(uint32_t code, float unit) {
  const float c = (float)code, square = c * c;
  return square * square * unit;
}

// m and v of eight elements, and the step; sums with the product rounded together with them
__device__ __forceinline__ void advance(const Rates& r, float g, float& m, float& v, float& p) {
  m = __builtin_fmaf(m, r.beta1, g * r.rest1);
  v = __builtin_fmaf(v, r.beta2, g * g * r.rest2);
  p = __builtin_fmaf(-r.step, m / __builtin_fmaf(sqrtf(v), r.root, r.eps), p * r.keep);
}

// 32 lanes have a group, eight elements each.  Bound by memory: 16 bytes an element of floats with states in 8 bits, 28 with states in floats.
template <typename T, bool CODES>
__global__ __launch_bounds__(256) void adamw_kernel(Tensors a, Step step) {
  __shared__ Rates made;
  Rates r = step.r;
  if (step.o.lr_at || step.o.step_at) {      // recorded in a graph, say: the same double arithmetic as the host's
    if (threadIdx.x == 0)
      made = rates_of(step.o, step.o.lr_at ? (double)*step.o.lr_at : step.o.lr, (double)(step.o.step_at ? *step.o.step_at : step.o.step));
    __syncthreads();
    r = made;
  }
  const uint32_t block = (uint32_t)block_of();
  if (block >= a.first[a.count]) return;
  const int which = __builtin_amdgcn_readfirstlane(tensor_of(a, block));
  const gact_adamw_tensor& t = a.t[which];
  const int64_t group = (int64_t)(block - a.first[which]) * (256 / kLanes) + threadIdx.x / kLanes, at = group * kGroup + threadIdx.x % kLanes * kVec;
  const int64_t left = t.numel - at;
  T* const p = (T*)t.p + at;
  const T* const g = (const T*)t.g + at;
  const bool whole = (((uintptr_t)t.p | (uintptr_t)t.g) & 15) == 0 && left >= kVec;
  float x[kVec], d[kVec], m[kVec], v[kVec];
  if (whole) {
    load8(p, x);
    load8(g, d);
  } else {
    load_cols<T, false>(p, left, x);
    load_cols<T, false>(g, left, d);
  }
  if constexpr (CODES) {
    uint8_t* const mc = (uint8_t*)t.m + at;
    uint8_t* const vc = (uint8_t*)t.v + at;
    u32x2 cm = {}, cv = {};
    f32x2 unit = {};
    if (left >= kVec) {
      cm = *(const u32x2*)mc;
      cv = *(const u32x2*)vc;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e++)
        if (e < left) {
          cm[e >> 2] |= (uint32_t)mc[e] << (8 * (e & 3));
          cv[e >> 2] |= (uint32_t)vc[e] << (8 * (e & 3));
        }
    }
    if (group * kGroup < t.numel) unit = *(const f32x2*)(t.scale + 2 * group);
    unit = f32x2{unit[0] / kSquare, unit[1] / kFourth};
    float most_m = 0.0f, most_v = 0.0f;
#pragma unroll
    for (int e = 0; e < kVec; e++) {
      m[e] = first_of(byte_of(cm[e >> 2], e & 3), unit[0]);
      v[e] = second_of(byte_of(cv[e >> 2], e & 3), unit[1]);
      advance(r, d[e], m[e], v[e], x[e]);
      if (e < left) {
        most_m = MostBits::of(most_m, __builtin_fabsf(m[e]));
        most_v = MostBits::of(most_v, __builtin_fabsf(v[e]));
      }
    }
    most_m = over_lanes<MostBits, kLanes>(most_m);
    most_v = over_lanes<MostBits, kLanes>(most_v);
    if (most_m < kLeastM) most_m = 0.0f;
    if (most_v < kLeastV) most_v = 0.0f;
    const float inv_m = most_m == 0.0f ? 0.0f : kSquare / most_m, inv_v = most_v == 0.0f ? 0.0f : kFourth / most_v;
    cm = u32x2{};
    cv = u32x2{};
#pragma unroll
    for (int e = 0; e < kVec; e++) {
      const float c = nearest_root(__builtin_fabsf(m[e]) * inv_m);
      float f = nearest_fourth_root(v[e] * inv_v);
      if (v[e] > 0.0f && most_v > 0.0f && f < 1.0f) f = 1.0f;
      const int code = c > 0.0f ? (int)c : 0;      // a NaN becomes 0
      cm[e >> 2] |= ((uint32_t)(m[e] < 0.0f ? -code : code) & 0xff) << (8 * (e & 3));
      cv[e >> 2] |= (f > 0.0f ? (uint32_t)f & 0xff : 0) << (8 * (e & 3));
    }
    if (left >= kVec) {
      *(u32x2*)mc = cm;
      *(u32x2*)vc = cv;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e++)
        if (e < left) {
          mc[e] = (uint8_t)byte_of(cm[e >> 2], e & 3);
          vc[e] = (uint8_t)byte_of(cv[e >> 2], e & 3);
        }
    }
    if (threadIdx.x % kLanes == 0 && left > 0) *(f32x2*)(t.scale + 2 * group) = f32x2{most_m, most_v};
  } else {
    float* const mf = (float*)t.m + at;
    float* const vf = (float*)t.v + at;
    if (left >= kVec) {
      load8(mf, m);
      load8(vf, v);
    } else {
      load_cols<float, false>(mf, left, m);
      load_cols<float, false>(vf, left, v);
    }
#pragma unroll
    for (int e = 0; e < kVec; e++) advance(r, d[e], m[e], v[e], x[e]);
    if (left >= kVec) {
      store8(mf, m);
      store8(vf, v);
    } else {
      store_cols<float, false>(mf, left, m);
      store_cols<float, false>(vf, left, v);
    }
  }
  if (whole)
    store8(p, x);
  else
    store_cols<T, false>(p, left, x);
}

// the same lanes; t.p and t.g: where a tensor's values go
__global__ __launch_bounds__(256) void adamw_values_kernel(Tensors a) {
  const uint32_t block = (uint32_t)block_of();
  if (block >= a.first[a.count]) return;
  const int which = __builtin_amdgcn_readfirstlane(tensor_of(a, block));
  const gact_adamw_tensor& t = a.t[which];
  const int64_t group = (int64_t)(block - a.first[which]) * (256 / kLanes) + threadIdx.x / kLanes, at = group * kGroup + threadIdx.x % kLanes * kVec;
  const int64_t left = t.numel - at;
  if (left <= 0) return;
  const f32x2 scale = *(const f32x2*)(t.scale + 2 * group);
  auto one = [&](const uint8_t* codes, float* to, auto value) __attribute__((always_inline)) {
    if (!to) return;
    float x[kVec];
    u32x2 c = {};
    if (left >= kVec) {
      c = *(const u32x2*)(codes + at);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e++)
        if (e < left) c[e >> 2] |= (uint32_t)codes[at + e] << (8 * (e & 3));
    }
#pragma unroll
    for (int e = 0; e < kVec; e++) x[e] = value(byte_of(c[e >> 2], e & 3));
    if (((uintptr_t)to & 15) == 0 && left >= kVec)
      store8(to + at, x);
    else
      store_cols<float, false>(to + at, left, x);
  };
  one((const uint8_t*)t.m, (float*)t.p, [&](uint32_t c) { return first_of(c, scale[0] / kSquare); });
  one((const uint8_t*)t.v, (float*)const_cast<void*>(t.g), [&](uint32_t c) { return second_of(c, scale[1] / kFourth); });
}

// `run` for each launch's worth of the tensors that have elements
template <typename F>
int in_launches(const gact_adamw_tensor* tensors, int64_t count, F&& run) {
  Tensors a;
  a.count = 0;
  a.first[0] = 0;
  for (int64_t i = 0; i <= count; i++) {
    if (a.count && (i == count || a.count == kTensors)) {
      const int rc = run(a);
      if (rc != GACT_OK) return rc;
      a.count = 0;
    }
    if (i == count || tensors[i].numel == 0) continue;
    const int64_t blocks = (tensors[i].numel + 8 * kGroup - 1) / (8 * kGroup);
    // a launch counts its blocks in 31 bits; a tensor of as many goes on its own
    if (a.count && a.first[a.count] + blocks > 0x7fffffff) {
      const int rc = run(a);
      if (rc != GACT_OK) return rc;
      a.count = 0;
    }
    if (blocks > 0x7fffffff) return GACT_ELIMIT;
    a.t[a.count] = tensors[i];
    a.first[a.count + 1] = a.first[a.count] + (uint32_t)blocks;
    a.count++;
  }
  return GACT_OK;
}

int check_state(const gact_adamw_tensor& t, bool codes) {
  if (t.numel < 0) return GACT_EINVAL;
  if (t.numel == 0) return GACT_OK;
  if (!t.m || !t.v || (codes && !t.scale)) return GACT_EINVAL;
  return aligned16(t.m) && aligned16(t.v) && (!codes || ((uintptr_t)t.scale & 7) == 0) ? GACT_OK : GACT_EALIGN;
}

}  // namespace

extern "C" {

int gact_adamw(const gact_adamw_tensor* tensors, int64_t count, int dtype, int bits, const gact_adamw_options* options, void* stream) {
  if (!known(dtype) || (bits != 8 && bits != 32) || count < 0 || !options || (count && !tensors)) return GACT_EINVAL;
  const gact_adamw_options& o = *options;
  // a number that is none fails every comparison
  if (!(o.lr >= 0.0) || !(o.beta1 >= 0.0 && o.beta1 < 1.0) || !(o.beta2 >= 0.0 && o.beta2 < 1.0) || !(o.eps >= 0.0) || !(o.decay >= 0.0)) return GACT_EINVAL;
  if (!o.step_at && o.step < 1) return GACT_EINVAL;
  const uintptr_t element = dtype == GACT_F32 ? 4 : 2;
  for (int64_t i = 0; i < count; i++) {
    const int rc = check_state(tensors[i], bits == 8);
    if (rc != GACT_OK) return rc;
    if (tensors[i].numel && (!tensors[i].p || !tensors[i].g)) return GACT_EINVAL;
    if (((uintptr_t)tensors[i].p | (uintptr_t)tensors[i].g) % element) return GACT_EALIGN;
  }
  fresh_launch();
  const Step step{o, rates_of(o, o.lr, (double)(o.step_at ? 1 : o.step))};
  return in_launches(tensors, count, [&](const Tensors& a) {
    return with_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      auto kernel = bits == 8 ? adamw_kernel<T, true> : adamw_kernel<T, false>;
      hipLaunchKernelGGL(kernel, grid_of(a.first[a.count], 256), dim3(256), 0, (hipStream_t)stream, a, step);
      return launch_status();
    });
  });
}

int gact_adamw_values(const gact_adamw_tensor* tensors, int64_t count, float* m, float* v, void* stream) {
  if (count < 0 || (count && !tensors)) return GACT_EINVAL;
  for (int64_t i = 0; i < count; i++) {
    const int rc = check_state(tensors[i], true);
    if (rc != GACT_OK) return rc;
  }
  fresh_launch();
  int64_t next = 0;      // the launches' tensors are the list's, in order, without the empty ones
  return in_launches(tensors, count, [&](Tensors& a) {
    for (int i = 0; i < a.count; i++) {
      a.t[i].p = m ? m + next : nullptr;
      a.t[i].g = v ? v + next : nullptr;
      next += a.t[i].numel;
    }
    hipLaunchKernelGGL(adamw_values_kernel, grid_of(a.first[a.count], 256), dim3(256), 0, (hipStream_t)stream, a);
    return launch_status();
  });
}

}  // extern "C"
