// AdamW's step over many tensors in one launch for each 72 of them, with states in floats or in 8 bits.
//
// 8 bits: groups of 256 elements share the largest magnitude of either state.  The first moment's codes are spaced by the square, the second's by the
// fourth power, so that sqrt(v), by which the step is divided, has the same spacing as m: a step of 0.8 % next to the largest, and values down to
// (1/255)^4 of the largest of v.  A v above zero never becomes zero, which would blow its step up: of a group whose largest is too small to divide by, the
// codes are those beside kLeastV, so that a v of 1e-45 still stands for (1/255)^4 of it.
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
// what a code stands for
__device__ __forceinline__ float first_of(uint32_t code, float unit) {
  const float c = (float)(int8_t)code;
  return c * __builtin_fabsf(c) * unit;
}
__device__ __forceinline__ float second_of(uint32_t code, float unit) {
  const float c = (float)code, square = c * c;
  return square * square * unit;
}

// m, v and p of an element after the step; sums with the product rounded together with them
__device__ __forceinline__ void advance(const Rates& r, float g, float& m, float& v, float& p) {
  m = __builtin_fmaf(m, r.beta1, g * r.rest1);
  v = __builtin_fmaf(v, r.beta2, g * g * r.rest2);
  p = __builtin_fmaf(-r.step, m / __builtin_fmaf(sqrtf(v), r.root, r.eps), p * r.keep);
}

// N neighbouring elements, of which `left` are there; WHOLE: all of them, at a multiple of their size
template <typename T, int N>
struct Piece {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef T Loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  template <bool WHOLE>
  static __device__ __forceinline__ V load(const T* p, int64_t left) {
    V v = {};
    if (WHOLE) return *(const V*)p;
    if (left >= N) return *(const Loose*)p;
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e < left) v[e] = p[e];
    return v;
  }
  template <bool WHOLE>
  static __device__ __forceinline__ void store(T* p, int64_t left, V v) {
    if (WHOLE) {
      *(V*)p = v;
    } else if (left >= N) {
      *(Loose*)p = v;
    } else {
#pragma unroll
      for (int e = 0; e < N; e++)
        if (e < left) p[e] = v[e];
    }
  }
};

// 32 lanes have a group, eight elements each.  Bound by memory.  States in 8 bits: the eight lie side by side (302 million floats 890 us, 5.4 TB/s; four of
// either half of the group, so that an instruction loads and stores whole lines of floats but codes by four, 1060).  States in floats: four of either half
// (75 million bfloat16 values 311 us, 5.3 TB/s, eight side by side the same).  Nontemporal loads and stores, and fewer workgroups to a compute unit, change
// nothing or cost 3 %.
template <typename T, bool CODES, bool WHOLE>
__device__ __forceinline__ void step_group(const gact_adamw_tensor& t, const Rates& r, int64_t group, int64_t left_over) {
  constexpr int N = CODES ? 8 : 4, kPieces = kVec / N;
  const int lane = threadIdx.x % kLanes;
  const int64_t begin = group * kGroup;
  typename Piece<T, N>::V p[kPieces], g[kPieces];
  typename Piece<uint8_t, N>::V cm[kPieces], cv[kPieces];
  typename Piece<float, N>::V fm[kPieces], fv[kPieces];
  f32x2 unit = {};
  int64_t at[kPieces], left[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; k++) {
    const int col = k * (kGroup / kPieces) + lane * N;
    at[k] = begin + col;
    left[k] = left_over - col;
    p[k] = Piece<T, N>::template load<WHOLE>((const T*)t.p + at[k], left[k]);
    g[k] = Piece<T, N>::template load<WHOLE>((const T*)t.g + at[k], left[k]);
    if constexpr (CODES) {
      cm[k] = Piece<uint8_t, N>::template load<WHOLE>((const uint8_t*)t.m + at[k], left[k]);
      cv[k] = Piece<uint8_t, N>::template load<WHOLE>((const uint8_t*)t.v + at[k], left[k]);
    } else {
      fm[k] = Piece<float, N>::template load<WHOLE>((const float*)t.m + at[k], left[k]);
      fv[k] = Piece<float, N>::template load<WHOLE>((const float*)t.v + at[k], left[k]);
    }
  }
  if constexpr (CODES) {
    if (WHOLE || left_over > 0) unit = *(const f32x2*)(t.scale + 2 * group);
    unit = f32x2{unit[0] / kSquare, unit[1] / kFourth};
  }
  float most_m = 0.0f, most_v = 0.0f;
#pragma unroll
  for (int k = 0; k < kPieces; k++)
#pragma unroll
    for (int e = 0; e < N; e++) {
      float m, v, x = (float)p[k][e];
      if constexpr (CODES) {
        m = first_of(cm[k][e], unit[0]);
        v = second_of(cv[k][e], unit[1]);
      } else {
        m = fm[k][e];
        v = fv[k][e];
      }
      advance(r, (float)g[k][e], m, v, x);
      p[k][e] = rounded<T>(x);
      fm[k][e] = m;
      fv[k][e] = v;
      if (CODES && (WHOLE || e < left[k])) {
        most_m = MostBits::of(most_m, __builtin_fabsf(m));
        most_v = MostBits::of(most_v, __builtin_fabsf(v));
      }
    }
#pragma unroll
  for (int k = 0; k < kPieces; k++) Piece<T, N>::template store<WHOLE>((T*)t.p + at[k], left[k], p[k]);
  if constexpr (!CODES) {
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
      Piece<float, N>::template store<WHOLE>((float*)t.m + at[k], left[k], fm[k]);
      Piece<float, N>::template store<WHOLE>((float*)t.v + at[k], left[k], fv[k]);
    }
    return;
  }
  most_m = over_lanes<MostBits, kLanes>(most_m);
  most_v = over_lanes<MostBits, kLanes>(most_v);
  if (most_m < kLeastM) most_m = 0.0f;
  if (most_v > 0.0f && most_v < kLeastV) most_v = kLeastV;      // zero, the first moment would be divided by eps alone
  const float inv_m = most_m == 0.0f ? 0.0f : kSquare / most_m, inv_v = most_v == 0.0f ? 0.0f : kFourth / most_v;
#pragma unroll
  for (int k = 0; k < kPieces; k++) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      const float c = nearest_root(__builtin_fabsf(fm[k][e]) * inv_m);
      float f = nearest_fourth_root(fv[k][e] * inv_v);
      if (fv[k][e] > 0.0f && most_v > 0.0f && f < 1.0f) f = 1.0f;
      const int code = c > 0.0f ? (int)c : 0;      // a NaN becomes 0
      cm[k][e] = (uint8_t)(fm[k][e] < 0.0f ? -code : code);
      cv[k][e] = (uint8_t)(f > 0.0f ? (uint32_t)f : 0u);
    }
    Piece<uint8_t, N>::template store<WHOLE>((uint8_t*)t.m + at[k], left[k], cm[k]);
    Piece<uint8_t, N>::template store<WHOLE>((uint8_t*)t.v + at[k], left[k], cv[k]);
  }
  if (lane == 0 && (WHOLE || left_over > 0)) *(f32x2*)(t.scale + 2 * group) = f32x2{most_m, most_v};
}

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
  const int64_t first = (int64_t)(block - a.first[which]) * (256 / kLanes), group = first + threadIdx.x / kLanes;
  // the block's groups are whole and lie at multiples of 16 bytes
  const bool whole = (((uintptr_t)t.p | (uintptr_t)t.g) & 15) == 0 && (first + 256 / kLanes) * kGroup <= t.numel;
  if (whole)
    step_group<T, CODES, true>(t, r, group, t.numel - group * kGroup);
  else
    step_group<T, CODES, false>(t, r, group, t.numel - group * kGroup);
}

// What codes stand for: one of the moments to a block (blockIdx.z), four elements of either half of a group to a lane, so that an instruction stores whole
// lines; t.p and t.g: where a tensor's values go.  302 million elements 496 us (6.1 TB/s); eight side by side and both moments in turn 703.
__global__ __launch_bounds__(256) void adamw_values_kernel(Tensors a) {
  const uint32_t block = (uint32_t)block_of();
  if (block >= a.first[a.count]) return;
  const int which = __builtin_amdgcn_readfirstlane(tensor_of(a, block));
  const gact_adamw_tensor& t = a.t[which];
  const bool second = blockIdx.z == 1;
  float* const to = (float*)(second ? const_cast<void*>(t.g) : t.p);
  const uint8_t* const codes = (const uint8_t*)(second ? t.v : t.m);
  if (!to) return;
  const int64_t group = (int64_t)(block - a.first[which]) * (256 / kLanes) + threadIdx.x / kLanes;
  const int64_t at = group * kGroup + threadIdx.x % kLanes * 4, left = t.numel - at;
  typedef Piece<uint8_t, 4> Codes;
  const Codes::V c[2] = {Codes::load<false>(codes + at, left), Codes::load<false>(codes + at + kGroup / 2, left - kGroup / 2)};
  const float unit = (group * kGroup < t.numel ? t.scale[2 * group + second] : 0.0f) / (second ? kFourth : kSquare);
#pragma unroll
  for (int k = 0; k < 2; k++) {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = second ? second_of(c[k][e], unit) : first_of(c[k][e], unit);
    Piece<float, 4>::store<false>(to + at + k * (kGroup / 2), left - k * (kGroup / 2), x);
  }
}

// `run` for each launch's worth of the tensors that have elements
template <typename F>
int in_launches(const gact_adamw_tensor* tensors, int64_t count, int groups, F&& run) {
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
    const int64_t blocks = (tensors[i].numel + groups * kGroup - 1) / (groups * kGroup);
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
  return in_launches(tensors, count, 256 / kLanes, [&](const Tensors& a) {
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
  return in_launches(tensors, count, 256 / kLanes, [&](Tensors& a) {
    for (int i = 0; i < a.count; i++) {
      a.t[i].p = m ? m + next : nullptr;
      a.t[i].g = v ? v + next : nullptr;
      next += a.t[i].numel;
    }
    dim3 grid = grid_of(a.first[a.count], 256);
    grid.z = 2;
    hipLaunchKernelGGL(adamw_values_kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
    return launch_status();
  });
}

}  // extern "C"
