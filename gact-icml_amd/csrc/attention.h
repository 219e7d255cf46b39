// Attention's kernels, for one element type: the three sources that compile them differ in it alone, and are built side by side.
//
//   s_ij = scale q_i.k_j + bias[j - i + queries - 1]      hidden: absent keys, and with `causal` keys behind i + keys - queries
//   p_ij = exp(s_ij - L_i), L_i = log sum_j exp(s_ij)      o_i = sum_j p_ij v_j
//   ds_ij = p_ij (do_i.v_j - do_i.o_i)                     dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i
//
// Exponentials are of base 2: scores, biases and L are held multiplied by log2(e).  Probabilities and ds enter their products rounded to T, which is
// what the matrix instructions of 16-bit types take; sums, maxima and L are floats.
//
// All kernels are built alike.  A wave owns 32 rows of one side (queries; keys in the kernel of dk and dv) and keeps them in registers as the matrix
// instruction's columns; the other side passes by in tiles of rows that are in LDS, its rows being the instruction's rows.  A lane so has 16 of the 32
// scores of one of its own rows, the lane 32 further on the others: a maximum or sum over the other side stays in the lane but for one exchange, and the
// scores are in place as the second product's operand, whose depth is the tile's rows in whatever order - its other operand is read from the
// tile through the transposing LDS read in the same order.  Neither scores nor probabilities leave the registers.
#pragma once
#include "device.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));

// rows of [batch, head, row, width], strides in bytes
struct Side {
  const char* p;
  int64_t batch, head, row;
  __device__ __forceinline__ const char* at(int64_t b, int64_t h, int64_t r) const { return p + b * batch + h * head + r * row; }
};

struct AttentionArgs {
  Side q, k, v, out, d_out, dq, dk, dv;
  float* lse;                // [batch, heads, queries]; infinite for a query that sees nothing
  float* delta;              // the same: -do_i.o_i, with which the sums of do_i.v_j begin
  int8_t* rest;              // [batch, queries, heads, width]: what rounding o to T has left out, see Rest; may be null
  const float* bias;         // [heads, queries + keys - 1], times log2(e)
  const uint8_t* mask;       // [batch, keys]
  int64_t mask_stride;
  float* along;              // sums of ds along the diagonals, of every 32 queries
  int64_t along_stride;
  int heads, kv_heads, group, queries, keys, width;
  bool causal;
  bool blind;                // there may be queries that see nothing
  float scale, scale2;       // and times log2(e)
  uint32_t tiles, blocks;    // of a head, and in all
  bool by_length;            // see work_of
  int splits, per_split;     // of the other side; keys of a split, whole blocks of 32 (in the backward pass whole tiles)
  // the forward pass: [tile, split][32, width rounded up], and [tile, split][32, 2]; dq: [split][head, row of its tiles][width rounded up]; dk and dv the
  // same, one behind the other
  float* part;
  float* part_stats;
  // keys that query i sees
  __device__ __forceinline__ int seen(int i) const {
    const int n = i + keys - queries + 1;
    return !causal || n > keys ? keys : n;
  }
  __device__ __forceinline__ int8_t* rest_at(int b, int head, int query) const {
    return rest ? rest + (((int64_t)b * queries + query) * heads + head) * width : nullptr;
  }
  __device__ __forceinline__ int distances() const { return queries + keys - 1; }
};

namespace {

template <typename T>
struct Matrix {
  using Frag = std::conditional_t<std::is_same<T, bf16>::value, bf16x8, std::conditional_t<std::is_same<T, f16>::value, f16x8, f32x4>>;
  // 16 bytes a lane and operand: 16 values of depth of 16-bit types, 8 floats
  static __device__ __forceinline__ f32x16 run(Frag a, Frag b, f32x16 c) {
    if constexpr (std::is_same<T, bf16>::value) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    if constexpr (std::is_same<T, f16>::value) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int t = 0; t < 4; t++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
    }
    return c;
  }
};
// the row, within 32, of element e of a result: lanes 32 and up have the rows 4 further down
constexpr int row_of(int e) { return 8 * (e >> 2) + (e & 3); }

// Rows of DP values (the width rounded up to 32) in LDS, W bytes each.  A row's pieces of 16 bytes are permuted by turn() of its number: the 16 rows of
// which the product's first operand takes a piece each, and the four rows of which the transposing read takes 64 bytes (of floats: the rows r and r + 4
// whose 128 bytes go together), lie in different banks.
template <typename T, int DP, int WAVES = 4>
struct Tile {
  using Frag = typename Matrix<T>::Frag;
  static constexpr int kEsz = (int)sizeof(T), kWide = DP * kEsz;
  static constexpr int W = kWide <= 64 ? 64 : kWide <= 128 ? 128 : kWide <= 256 ? 256 : 512;
  // tiles of 64 rows, of which a compute unit's LDS holds two of either side at least twice; of 32 for workgroups of two waves, of which there are more
  static constexpr int kRows = W <= 256 && WAVES == 4 ? 64 : W == 64 ? 64 : 32;
  static constexpr int NC = kWide / 32, ND = DP / 32;
  static constexpr __device__ __forceinline__ uint32_t turn(uint32_t r) {
    const uint32_t a = r & 1, b = (r >> 1) & 1, c = (r >> 2) & 1, d = (r >> 3) & 1;
    if (W == 64) return c | d << 1;
    if (W == 128) return b << 2 | c << 1 | d;
    return sizeof(T) == 2 ? a << 2 | b << 3 | c | d << 1 : a << 2 | b << 1 | c << 3 | d;
  }
  // pieces 2c and 2c + 1 of rows first .. first + 31: lane l has row l % 32
  static __device__ __forceinline__ Frag direct(const lds_u8* tile, int first, int c, int lane) {
    const uint32_t r = lane & 31, g = lane >> 5;
    return *(const __attribute__((address_space(3))) Frag*)(tile + first * W + r * W + (((2 * c) ^ g ^ turn(r)) * 16));
  }
  // 32 rows by 32 columns of results as an operand
  struct Halves {
    Frag f[2];
  };
  using Packed = std::conditional_t<sizeof(T) == 2, Halves, f32x16>;
  static __device__ __forceinline__ Packed pack(const f32x16& p) {
    if constexpr (sizeof(T) == 2) {
      Packed k;
#pragma unroll
      for (int e = 0; e < 16; e++) k.f[e >> 3][e & 7] = rounded<T>(p[e]);
      return k;
    } else {
      return p;
    }
  }
  // `up` times it, and what rounding that has left out; up: a power of two, so that what is left out is exact before it is rounded itself
  static __device__ __forceinline__ Packed pack_up(const f32x16& p, float up) {
    Packed k;
#pragma unroll
    for (int e = 0; e < 16; e++) k.f[e >> 3][e & 7] = (T)(p[e] * up);
    return k;
  }
  static __device__ __forceinline__ Packed rest_up(const f32x16& p, float up, const Packed& k) {
    Packed r;
#pragma unroll
    for (int e = 0; e < 16; e++) r.f[e >> 3][e & 7] = (T)__builtin_fmaf(p[e], up, -(float)k.f[e >> 3][e & 7]);
    return r;
  }
  // whether one of them is 2 or more, an infinity or no number, in float16
  static __device__ __forceinline__ bool some_large(const Packed& k) {
    uint32_t any = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int w = 0; w < 4; w++) any |= __builtin_bit_cast(u32x4, k.f[h])[w];
    return (any & 0x40004000u) != 0;
  }
  // what rounding p has left out
  static __device__ __forceinline__ Packed rest(const f32x16& p, const Packed& k) {
    f32x16 r = {};
    if constexpr (std::is_same<T, bf16>::value) {
#pragma unroll
      for (int e = 0; e < 16; e += 2) {      // out of the pairs as they are: left to itself the compiler rounds every value again, on its own
        uint32_t w = __builtin_bit_cast(u32x4, k.f[e >> 3])[(e & 7) / 2];
        asm("" : "+v"(w));
        r[e] = p[e] - __builtin_bit_cast(float, w << 16);
        r[e + 1] = p[e + 1] - __builtin_bit_cast(float, w & 0xffff0000u);
      }
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 16; e++) r[e] = p[e] - (float)k.f[e >> 3][e & 7];
    }
    return pack(r);
  }
  // the sum of what a lane has of it
  static __device__ __forceinline__ float sum(const Packed& p) {
    float s[2] = {};
    if constexpr (sizeof(T) == 2) {
      typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        [[maybe_unused]] const T2 v = {p.f[e >> 3][e & 7], p.f[e >> 3][(e & 7) + 1]}, one = {(T)1.0f, (T)1.0f};
#ifdef __HIP_DEVICE_COMPILE__
        if constexpr (std::is_same<T, bf16>::value)
          s[(e >> 1) & 1] = __builtin_amdgcn_fdot2_f32_bf16(v, one, s[(e >> 1) & 1], false);
        else
          s[(e >> 1) & 1] = __builtin_amdgcn_fdot2(v, one, s[(e >> 1) & 1], false);
#endif
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) s[e & 1] += p[e];
    }
    return s[0] + s[1];
  }
  // the tile's rows transposed, as the first operand of a product of 32 values of the width by 32 columns, whose depth is the rows
  struct Turned {
    Frag f[2][ND];
  };
  static __device__ __forceinline__ Frag turned(const lds_u8* tile, int first, int s, int d, int lane) {
    const uint32_t i = lane & 15, half = (lane >> 4) & 1, g = lane >> 5;
    const uint32_t r = 4 * g + (i >> 2), piece = 4 * d + 2 * half + ((i & 3) >> 1);
    const lds_u8* lo = tile + (first + 16 * s) * W + r * W + ((piece ^ turn(r)) * 16) + (i & 1) * 8;
    const lds_u8* hi = tile + (first + 16 * s) * W + (r + 8) * W + ((piece ^ turn(r + 8)) * 16) + (i & 1) * 8;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi);
    return __builtin_bit_cast(Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ Turned turned(const lds_u8* tile, int first, int lane) {
    Turned t;
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int d = 0; d < ND; d++) t.f[s][d] = turned(tile, first, s, d, lane);
    return t;
  }
  // acc[32 values of the width, 32 columns] += the tile's rows transposed [., 32 rows] times p [32 rows, 32 columns]; and times `more`
  template <bool TWICE = false>
  static __device__ __forceinline__ void add(f32x16 (&acc)[ND], const lds_u8* tile, int first, const Packed& p, int lane, const Packed* more = nullptr) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int s = 0; s < 2; s++) {
#pragma unroll
        for (int d = 0; d < ND; d++) {
          const Frag a = turned(tile, first, s, d, lane);
          acc[d] = Matrix<T>::run(a, p.f[s], acc[d]);
          if constexpr (TWICE) acc[d] = Matrix<T>::run(a, more->f[s], acc[d]);
        }
      }
    } else {
      // the addresses anew each time, beside products of 64 cycles: kept from one block to the next they would take more registers than there are
      const uint32_t g = lane >> 5;
      uint32_t l = lane & 31;
      asm volatile("" : "+v"(l));
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const uint32_t r = row_of(e) + 4 * g;
#pragma unroll
        for (int d = 0; d < ND; d++) {
          const float a = *(const __attribute__((address_space(3))) float*)(tile + (first + r) * W + (((8 * d + (l >> 2)) ^ turn(r)) * 16) + (l & 3) * 4);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[e], acc[d], 0, 0, 0);
        }
      }
    }
  }
};

// Loads rows into a tile, straight to LDS: an instruction of a wave fills 1 KB.  What lies behind the width or the last row becomes zero.
template <typename T, int DP, int ROWS, int WAVES>
struct RowsLoad {
  using Shape = Tile<T, DP>;
  static constexpr int W = Shape::W, kLoads = ROWS * W / 1024 / WAVES;
  static_assert(kLoads >= 1, "a wave takes at least one load");
  Window window;
  int64_t step;
  uint32_t at[kLoads];
  int wave;
  static __device__ __forceinline__ uint32_t row(int wave, int q, int lane) { return ((wave * kLoads + q) * 1024 + lane * 16) / W; }
  // (rows before `from` become zero as well)
  __device__ __forceinline__ void set_up(int64_t stride, int width, int w, int lane, int from = 0) {
    wave = w;
#pragma unroll
    for (int q = 0; q < kLoads; q++) {
      const uint32_t r = row(w, q, lane), piece = ((lane * 16 % W) / 16) ^ Shape::turn(r);
      at[q] = (int)piece * 16 < width * Shape::kEsz && (int)r >= from ? r * (uint32_t)stride + piece * 16 : kNowhere;
    }
  }
  // from `base` on, of which `left` rows are there; `tiles` of ROWS rows to a step
  __device__ __forceinline__ void start(const char* base, int64_t left, int64_t stride, int width, int tiles = 1) {
    window.base = base;
    window.left = left <= 0 ? 0 : (left - 1) * stride + width * Shape::kEsz;
    step = tiles * ROWS * stride;
  }
  // the next tile, without the rows whose bit of `there` is not set
  __device__ __forceinline__ void next(bool some_absent, uint64_t there, lds_u8* to, int lane) {
    const __amdgpu_buffer_rsrc_t rsrc = window.rsrc();
#pragma unroll
    for (int q = 0; q < kLoads; q++) {
      uint32_t from = at[q];
      if (some_absent && !((there >> row(wave, q, lane)) & 1)) from = kNowhere;
      load_to_lds<16>(rsrc, from, to + (wave * kLoads + q) * 1024);
    }
    window.advance(step);
  }
};

// `count` floats from `at` on of an array of `size`, 64 to a wave's instruction; zeros where the array ends on either side
__device__ __forceinline__ void load_floats(const float* base, int size, int at, int count, int turn, int waves, lds_u8* to, int lane) {
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, size * 4, 0x00020000);
  for (int l = turn; l * 64 < count; l += waves) {
    const uint32_t from = (uint32_t)(at + l * 64 + lane);
    load_to_lds<4>(rsrc, from < (uint32_t)size ? from * 4 : kNowhere, to + l * 256);
  }
}

// all loads and stores are done, and all LDS reads
__device__ __forceinline__ void wait_all() { __builtin_amdgcn_s_waitcnt(7 << 4); }
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// a wave's LDS accesses are executed in its order, and the compiler keeps it
__device__ __forceinline__ void in_turn() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// a and b: a value of the lane's and the one of the lane 32 further on, in whichever order
__device__ __forceinline__ float most_of_both(float v) {
  uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
  swap_rows32(a, b);
  return __builtin_fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float sum_of_both(float v) {
  uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
  swap_rows32(a, b);
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// Workgroups go to the 8 XCDs in turn: each XCD has a run of consecutive heads, so that the tiles of a head, which read the same rows, share its L2.
// Where the tiles are of different lengths and the heads fill the XCDs evenly, an XCD takes all heads' longest tiles first: head by head, the last one's
// long tiles would be left to a few compute units (two prompts of 4096 tokens 405 us, so 330).
struct Work {
  uint32_t tile, head;      // the tile's number in that order
};
__device__ __forceinline__ bool work_of(const AttentionArgs& p, uint32_t per_tile, Work& work) {
  const uint32_t id = (uint32_t)block_of(), xcd = id % 8, i = id / 8;
  if (id >= p.blocks) return false;
  if (p.by_length) {
    const uint32_t heads = p.blocks / per_tile / p.tiles / 8;
    work.tile = i / heads;
    work.head = xcd * heads + i % heads;
  } else {
    const uint32_t most = p.blocks / 8, rest = p.blocks % 8, w = xcd * most + (xcd < rest ? xcd : rest) + i;
    work.tile = w % (p.tiles * per_tile);
    work.head = w / (p.tiles * per_tile);
  }
  return true;
}

// pieces 2c and 2c + 1 of one row, from memory
template <typename T, int NC>
__device__ __forceinline__ void own_row(const char* row, bool there, int width, int lane, typename Matrix<T>::Frag (&f)[NC]) {
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const int piece = 2 * c + (lane >> 5);
    f[c] = typename Matrix<T>::Frag{};
    if (there && piece * 16 < width * (int)sizeof(T)) f[c] = *(const typename Matrix<T>::Frag*)(row + piece * 16);
  }
}
// What a result of 16 bits leaves out of a float, in eight bits: at most half a step, 2^-8 (bfloat16) or 2^-11 of the value's power of two, in 127ths.
// ds_ij = p_ij (do_i.v_j - do_i.o_i) is a difference of nearly equal numbers where one key has most of the probability: with o as it was rounded
// dq and dk were off by 0.0040 of their norm (bfloat16, scores of deviation 2) where the other roundings leave 0.0025; a byte of each o is what that takes.
template <typename T>
struct Rest {
  static constexpr bool kept = sizeof(T) == 2;
  static constexpr float kSteps = 127.0f * (std::is_same<T, bf16>::value ? 256.0f : 2048.0f);
  static constexpr uint32_t kLeast = std::is_same<T, bf16>::value ? 1u << 23 : 113u << 23;      // the power of two below which steps stay the same
  static __device__ __forceinline__ uint32_t power(T v) {
    const uint32_t e = __builtin_bit_cast(uint32_t, (float)v) & 0x7f800000u;
    return e > kLeast ? e : kLeast;
  }
  static __device__ __forceinline__ uint32_t of(float exact, T v) {
    const float x = (exact - (float)v) * __builtin_bit_cast(float, 0x7f000000u - power(v)) * kSteps;
    return (uint32_t)(int)__builtin_rintf(__builtin_fminf(__builtin_fmaxf(x, -127.0f), 127.0f)) & 0xff;
  }
  static __device__ __forceinline__ float add(T v, uint32_t code) {
    return __builtin_fmaf((float)(int8_t)code, __builtin_bit_cast(float, power(v)) * (1.0f / kSteps), (float)v);
  }
};
// four neighbouring values of a row, and what they leave out
template <typename T>
__device__ __forceinline__ void store4(char* row, int8_t* rest, int col, f32x4 v) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 o;
#pragma unroll
  for (int t = 0; t < 4; t++) o[t] = rounded<T>(v[t]);
  *(T4*)(row + col * sizeof(T)) = o;
  if constexpr (Rest<T>::kept) {
    if (!rest) return;
    uint32_t w = 0;
#pragma unroll
    for (int t = 0; t < 4; t++) w |= Rest<T>::of(v[t], o[t]) << (8 * t);
    *(uint32_t*)(rest + col) = w;
  }
}
// acc, whose columns are a wave's rows, to memory: a lane has four neighbouring values of its row at a time
template <typename T, int ND>
__device__ __forceinline__ void store_row(char* row, int8_t* rest, int width, int lane, const f32x16 (&acc)[ND], float factor) {
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int col = 32 * d + row_of(e) + 4 * (lane >> 5);
      if (col < width) store4<T>(row, rest, col, f32x4{acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]} * factor);
    }
}

// The largest of them, as the middle one of each two and `top`, infinity: a maximum of two would have every product's result made a quiet NaN first, if it
// is one, in an instruction of its own
__device__ __forceinline__ float most_of(const f32x16& s, float top) {
  float m[2] = {__builtin_amdgcn_fmed3f(s[0], s[1], top), __builtin_amdgcn_fmed3f(s[2], s[3], top)};
#pragma unroll
  for (int e = 4; e < 16; e++) m[e & 1] = __builtin_amdgcn_fmed3f(m[e & 1], s[e], top);
  return __builtin_amdgcn_fmed3f(m[0], m[1], top);
}

// the same of a split, to be added up and multiplied later; `down`: what takes it to the others' scale
template <int DP, int ND>
__device__ __forceinline__ void store_part(float* row, int width, int lane, const f32x16 (&acc)[ND], float down) {
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int col = 32 * d + row_of(e) + 4 * (lane >> 5);
      if (col < width) *(f32x4*)(row + col) = f32x4{acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]} * down;
    }
}

// do_i . o_i of the lane's row, which two lanes share, with what the rounding of o has left out
template <typename T, int NC>
__device__ __forceinline__ float delta_of(const typename Matrix<T>::Frag (&o)[NC], const typename Matrix<T>::Frag (&dy)[NC], const int8_t* rest, int width, int lane) {
  float delta = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; c++) {
    u32x2 code = {};
    const int piece = 2 * c + (lane >> 5);
    if constexpr (Rest<T>::kept)
      if (rest && piece * 8 < width) code = *(const u32x2*)(rest + piece * 8);
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); e++) {
      float exact = (float)o[c][e];
      if constexpr (Rest<T>::kept)
        if (rest) exact = Rest<T>::add(o[c][e], code[e >> 2] >> (8 * (e & 3)));
      delta = __builtin_fmaf(exact, (float)dy[c][e], delta);
    }
  }
  return sum_of_both(delta);
}
// A block's ds into dq or dk.  A row's ds add up to zero, or nearly, and few of them are large: their roundings do not average out.  What they leave out
// makes a product of its own (bfloat16, a BERT-large layer: dq 0.0029 of its norm off without and 0.0021 with it, dk 0.0025 and 0.0019, of which 0.0017 is
// the result's rounding; 12 us of 80, and 13 of 101)
//
// A float16 has nothing below 2^-25, and ds is about dy / keys: with dy of 1e-3 and 4096 keys dq was 0.0053 of its norm off where the result's rounding
// is 0.0007, with 1e-4 0.053 (0.0066), and behind 65536 keys dv was 0.0007 (0.0002), whose probabilities are below 2^-14.  So in float16 the probabilities of
// dv are multiplied by 2^15, and ds by `up`, a power of two for each row of dq or dk, which the lane and the one 32 further on share: the one that takes
// the largest of its first block to 1/64, 2^15 at most, and, where a product reaches 2, the one that does so with that; what has been added up follows.  A
// ds is so off by 2^-19 of the row's largest or by 2^-40, and what is left is the result's own rounding.  It begins as infinity, with which every product
// is too large, and in a block that changes nothing it is an OR of the pairs, a third of an instruction a score (the sum of their squares, with a limit of
// 2^15 and so hardly a change, takes as long where rows change and 2 % longer where they do not).  32 x 16 heads of 512 tokens, width 64, float16: dq 104 us as without
// it, dk and dv 109 -> 113; 8 x 16 of 1000 with a bias: 113 as without, 107 -> 118, and where some channels are larger, so that the largest grows along a
// row, 117 -> 123 and 111 -> 124; 2 x 16 causal heads on 4 of 2048 tokens, width 128, where one wave has a SIMD and waits at the branch: 98 -> 102 and
// 109 -> 118 (both blocks of a tile behind one branch: no faster).
template <typename T>
struct Up {
  static constexpr bool kept = std::is_same<T, f16>::value;
  static constexpr float kMost = 32768.0f, kBegin = __builtin_inff();
  // 1 / up; of a row without a block: of nothing
  static __device__ __forceinline__ float down(float up) {
    return kept ? __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(uint32_t, __builtin_fminf(up, kMost))) : 1.0f;
  }
  template <typename Shape>
  static __device__ __forceinline__ typename Shape::Packed probabilities(const f32x16& p) {
    if constexpr (kept) return Shape::pack_up(p, kMost);
    else return Shape::pack(p);
  }
  static constexpr float kDown = kept ? 1.0f / kMost : 1.0f;      // of dv
};
template <typename T, int DP, int WAVES>
__device__ __forceinline__ void add_ds(f32x16 (&acc)[DP / 32], float& up, const lds_u8* keys, int first, const f32x16& ds, int lane) {
  using Shape = Tile<T, DP, WAVES>;
  if constexpr (Up<T>::kept) {
    // what the product reads is on its way before the branch
    const typename Shape::Turned rows = Shape::turned(keys, first, lane);
    typename Shape::Packed k = Shape::pack_up(ds, up);
    if (__builtin_expect(__ballot(Shape::some_large(k)) != 0, 0)) {
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; e++) most = __builtin_fmaxf(most, __builtin_fabsf(ds[e]));
      most = most_of_both(most);
      const uint32_t power = __builtin_bit_cast(uint32_t, most) >> 23;
      // what takes the largest to 1/64 and above; an infinity, whose row's result is none either way, has none
      const float fits = __builtin_fminf(power < 247 ? __builtin_bit_cast(float, (248 - power) << 23) : power < 255 ? 0x1p-126f : Up<T>::kMost, Up<T>::kMost);
      // a row's own products alone move it, so that its bits are the same whatever rows it shares the wave with
      const bool moves = up == Up<T>::kBegin || ((float)(T)(most * up) >= 2.0f && power < 255);
      const float factor = moves ? fits * Up<T>::down(up) : 1.0f;
      up = moves ? fits : up;
      // through a product of zeros: read by a vector instruction themselves, wide rows' sums would be moved from the matrix unit's registers to the vector
      // instructions' and back for every block
#pragma unroll
      for (int d = 0; d < DP / 32; d++) acc[d] = Matrix<T>::run({}, {}, acc[d]) * factor;
      k = Shape::pack_up(ds, up);
    }
    const typename Shape::Packed more = Shape::rest_up(ds, up, k);
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int d = 0; d < DP / 32; d++) acc[d] = Matrix<T>::run(rows.f[s][d], more.f[s], Matrix<T>::run(rows.f[s][d], k.f[s], acc[d]));
  } else if constexpr (sizeof(T) == 2) {
    const typename Shape::Packed k = Shape::pack(ds);
    const typename Shape::Packed more = Shape::rest(ds, k);
    Shape::template add<true>(acc, keys, first, k, lane, &more);
  } else {
    Shape::add(acc, keys, first, Shape::pack(ds), lane);
  }
}

// hidden scores of a block of 32 rows of the tile: the lane sees rows below `seen`, and of those the ones whose bit is set
// (the empty statement keeps the branch around it: without one the compiler makes the selections for every block)
__device__ __forceinline__ void hide(f32x16& s, int seen, uint32_t there, int lane) {
  asm volatile("");
  const int g4 = 4 * (lane >> 5);
  // as a mask of the lane's rows
  seen -= g4;
  there = (there >> g4) & (seen >= 32 ? ~0u : seen <= 0 ? 0u : (1u << seen) - 1);
#pragma unroll
  for (int e = 0; e < 16; e++) s[e] = there >> row_of(e) & 1 ? s[e] : -__builtin_inff();
}

// The gradients of queries that see nothing are nobody's, whatever they are: zeros take their place in a tile, where a NaN times a probability of zero
// would be one.  A wave clears every WAVES-th row.  -> whether there are any, which all waves find alike
template <int W, int ROWS, int WAVES>
__device__ __forceinline__ bool clear_blind(lds_u8* tile, const __attribute__((address_space(3))) float* lse, int wave, int lane) {
  const uint64_t all = __ballot(lse[lane & (ROWS - 1)] == __builtin_inff()), none = ROWS < 64 ? all & 0xffffffffu : all;
  if (__builtin_expect(none == 0, 1)) return false;
  for (uint64_t left = none; left; left &= left - 1) {
    const int r = __builtin_ctzll(left);
    if (r % WAVES == wave && lane * 16 < W) *(__attribute__((address_space(3))) u32x4*)(tile + r * W + lane * 16) = u32x4{};
  }
  return true;
}

// what the kernels over keys share: which keys of a tile there are.  The bytes of the next tile but one are on their way while a tile is worked on.
struct Present {
  const uint8_t* mask;
  int keys;
  uint32_t byte = 0;
  __device__ __forceinline__ void ask(int key) {
    if (mask) byte = key < keys ? mask[key] : 0;
  }
  __device__ __forceinline__ uint64_t answer() const { return mask ? __ballot(byte != 0) : ~0ull; }
};

// Waves that a SIMD is to hold: with two the compiler has 256 registers, and the products' results stay where the vector instructions reach them; beyond
// that they pass through the matrix unit's own registers, an instruction each way for every value (a BERT-large layer's forward pass 95 us, 61 without).
// Where the registers are too few for a kernel's rows, one.
enum { FORWARD, FORWARD_APART, DQ, DKV, SHORT };
template <typename T, int DP>
constexpr int waves_held(int kernel) {
  const int wide = DP * (int)sizeof(T);
  if (kernel == FORWARD) return wide <= 256 ? 2 : 1;
  if (kernel == FORWARD_APART) return wide <= 128 ? 2 : 1;
  if (kernel == DQ) return wide <= 256 && DP <= 96 ? 2 : 1;
  return wide <= 128 ? 2 : 1;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// The forward pass.  APART: for few queries the waves of a workgroup have the same 32 rows (the queries of all heads that share a key head), take the
// keys in turn, each in tiles of its own, and add up at the end; splits of the keys go to workgroups of their own, which the joining kernels add up.
// Bound by the vector instructions between its two products, of which a score takes four and an exponential, and which the products of a SIMD's two waves
// hardly overlap: 32 x 16 heads of 512 tokens, width 64, bfloat16, of which a mask leaves 0.69 of the tiles, 59 us (400 TFLOP/s of those; the SIMDs are at the
// vector instructions for 72 of 108 thousand cycles, at the products for 22), 2 x 32 causal heads of 4096, width 128, 305 (900), where the products alone would
// take 10 and 110 at the instructions' peak.  One token
// behind 65537 keys of 8 heads, width 128: 43 us, 6.3 TB/s, which is what memory gives.
// ---------------------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int WAVES, bool APART, bool BIAS>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(waves_held<T, DP>(APART ? FORWARD_APART : FORWARD)))) void attention_forward_kernel(AttentionArgs p) {
  using Shape = Tile<T, DP, WAVES>;
  using Frag = typename Shape::Frag;
  constexpr int R = APART ? 32 : Shape::kRows, NB = R / 32, W = Shape::W, NC = Shape::NC, ND = Shape::ND;
  constexpr int kTile = R * W, kRing = 4 * kTile, BM = APART ? 32 : WAVES * 32;
  constexpr int kBias = BIAS && !APART ? (BM + R + 63) / 64 * 256 : 0;
  using Load = RowsLoad<T, DP, R, APART ? 1 : WAVES>;
  __shared__ __attribute__((aligned(1024))) uint8_t memory[(APART ? WAVES : 1) * kRing + 2 * kBias];
  Work work;
  if (!work_of(p, APART ? p.splits : 1, work)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_u8* const ring = (lds_u8*)memory + (APART ? wave * kRing : 0);
  lds_u8* const biases = (lds_u8*)memory + (APART ? WAVES : 1) * kRing;

  const int split = APART ? (int)(work.tile % p.splits) : 0;
  const int turn = APART ? work.tile / p.splits : work.tile, tile = p.causal ? p.tiles - 1 - turn : turn;      // the longest first
  const uint32_t bh = work.head;
  const int heads = APART ? p.kv_heads : p.heads, b = bh / heads, h = bh % heads;
  const int kv = APART ? h : h / p.group;
  // the lane's query; behind the last one: that one, of which nothing is stored
  int head = h, query = tile * BM + (APART ? 0 : wave * 32) + (lane & 31);
  bool own;
  if constexpr (APART) {
    own = query < p.group * p.queries;
    query = own ? query : p.group * p.queries - 1;
    head = h * p.group + query / p.queries;
    query %= p.queries;
  } else {
    own = query < p.queries;
    query = own ? query : p.queries - 1;
  }
  Frag q[NC];
  own_row<T, NC>(p.q.at(b, head, query), true, p.width, lane, q);
  const int seen = p.seen(query);
  // of the wave's queries: what all of them see, and what any does
  const int first = APART ? 0 : tile * BM + wave * 32, last = APART ? p.queries - 1 : tile * BM + BM - 1;
  const int all_see = p.seen(first < p.queries ? first : p.queries - 1), some_see = p.seen(APART ? last : first + 31 < p.queries ? first + 31 : p.queries - 1);
  const int from = split * (APART ? p.per_split : 0);
  int to = p.seen(last < p.queries ? last : p.queries - 1);
  if (APART && from + p.per_split < to) to = from + p.per_split;
  // tiles of the wave: every WAVES-th block of keys where they are apart
  const int step = APART ? WAVES * R : R, begin = from + (APART ? wave * R : 0);
  const int steps = to > begin ? (to - begin + step - 1) / step : 0;

  Load load_k, load_v;
  load_k.set_up(p.k.row, p.width, APART ? 0 : wave, lane);
  load_v.set_up(p.v.row, p.width, APART ? 0 : wave, lane);
  Present present{p.mask ? p.mask + (int64_t)b * p.mask_stride : nullptr, p.keys};
  load_k.start(p.k.at(b, kv, begin), p.keys - begin, p.k.row, p.width, APART ? WAVES : 1);
  load_v.start(p.v.at(b, kv, begin), p.keys - begin, p.v.row, p.width, APART ? WAVES : 1);
  auto issue = [&](int t, uint64_t there) __attribute__((always_inline)) {
    lds_u8* const at = ring + (t & 1) * 2 * kTile;
    load_k.next(false, there, at, lane);
    load_v.next(p.mask != nullptr, there, at + kTile, lane);      // what is absent may be a NaN
    if constexpr (kBias > 0)
      load_floats(p.bias + (int64_t)h * p.distances(), p.distances(), begin + t * step - (tile * BM + BM - 1) + p.queries - 1, BM + R - 1, wave, WAVES,
                  biases + (t & 1) * kBias, lane);
  };
  // In float16 the probabilities are multiplied by 2^7, which 2^8, the most that one of them is before the maximum follows, leaves room for: unscaled, 100000 keys of
  // 2^-19 beside one of 1 are subnormal numbers, off by 2^-6 each, and the result by 0.004.  Sums and lse follow.
  constexpr float kUp = std::is_same<T, f16>::value ? 7.0f : 0.0f;
  // with a bias the scores are multiplied before it is added.  In vector registers: a scalar operand makes the multiplication take twice as long
  float unit2 = BIAS ? 1.0f : p.scale2, scale2 = p.scale2;
  float top = __builtin_inff();
  asm("" : "+v"(unit2), "+v"(scale2), "+v"(top));
  const float* const far = BIAS && APART ? p.bias + (int64_t)head * p.distances() + p.queries - 1 - query : nullptr;
  float most = -__builtin_inff(), limit = most, off = 0.0f, total = 0.0f;
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = f32x16{};

  uint64_t there = 0, next = 0;
  present.ask(begin + lane);
  next = present.answer();
  if (steps > 0) issue(0, next);
  present.ask(begin + step + lane);
  for (int t = 0; t < steps; t++) {
    wait_all();
    if (!APART) meet();
    __builtin_amdgcn_sched_barrier(0);
    there = next;
    next = present.answer();
    if (t + 1 < steps) issue(t + 1, next);
    present.ask(begin + (t + 2) * step + lane);
    const int key = begin + t * step;
    if (key >= some_see || !there) continue;
    const lds_u8* const keys = ring + (t & 1) * 2 * kTile;
    const bool edge = key + R > all_see || (p.mask && (R == 64 ? ~there : ~there & 0xffffffffu) != 0);
    auto scores = [&](int n) __attribute__((always_inline)) {
      f32x16 s = {};
#pragma unroll
      for (int c = 0; c < NC; c++) s = Matrix<T>::run(Shape::direct(keys, 32 * n, c, lane), q[c], s);
      return s;
    };
    auto add_bias = [&](int n, f32x16& s) __attribute__((always_inline)) {
      if constexpr (BIAS) {
        const int g4 = 4 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int r = 32 * n + row_of(e) + g4;
          float add;
          if constexpr (APART)
            add = far[key + r < p.keys ? key + r : p.keys - 1];
          else
            add = ((const __attribute__((address_space(3))) float*)(biases + (t & 1) * kBias))[r - (wave * 32 + (lane & 31)) + BM - 1];
          s[e] = __builtin_fmaf(s[e], scale2, add);
        }
      }
    };
    f32x16 s[NB];
#pragma unroll
    for (int n = 0; n < NB; n++) s[n] = scores(n);
#pragma unroll
    for (int n = 0; n < NB; n++) {
      add_bias(n, s[n]);
      if (edge) hide(s[n], seen - key - 32 * n, (uint32_t)(there >> (32 * n)), lane);
    }
    float m = most_of(s[0], top);
#pragma unroll
    for (int n = 1; n < NB; n++) m = __builtin_amdgcn_fmed3f(m, most_of(s[n], top), top);
    // the maximum follows when it is left behind by 2^8, which probabilities of every type hold: mostly in the first tile alone
    if (__ballot(m > limit)) {
      m = __builtin_fmaxf(most_of_both(m), most);
      const float factor = m > most ? __builtin_amdgcn_exp2f((most - m) * unit2) : 1.0f;
      most = m;
      off = m == -__builtin_inff() ? 0.0f : m * unit2 - kUp;
      limit = m + 8.0f / unit2;
      total *= factor;
#pragma unroll
      for (int d = 0; d < ND; d++) acc[d] *= factor;
    }
#pragma unroll
    for (int n = 0; n < NB; n++) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[n][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][e], unit2, -off));
      // the sum is of the probabilities as they enter the product: where one key has nearly all of a query's, its rounding cancels in the quotient
      const typename Shape::Packed k = Shape::pack(s[n]);
      total += Shape::sum(k);
      if constexpr (BIAS && sizeof(T) == 2) {
        // A bias's gradient adds up many ds, and those of a query are all off by what do_i . o_i is: with the probabilities' roundings in o a table's
        // gradient was up to 0.00035 of its norm off (float16, 8 x 1000 tokens) where its own rounding leaves 0.0002, which is all that is left of it now;
        // 71 us become 94
        const typename Shape::Packed more = Shape::rest(s[n], k);
        total += Shape::sum(more);
        Shape::template add<true>(acc, keys + kTile, 32 * n, k, lane, &more);
      } else {
        Shape::add(acc, keys + kTile, 32 * n, k, lane);
      }
    }
  }
  wait_all();

  total = sum_of_both(total);
  most = most == -__builtin_inff() ? most : most * unit2 - kUp;
  if constexpr (!APART) {
    if (!own) return;
    store_row<T, ND>((char*)p.out.at(b, head, query), p.rest_at(b, head, query), p.width, lane, acc, total > 0.0f ? 1.0f / total : total);
    if (p.lse && lane < 32)
      p.lse[((int64_t)b * p.heads + head) * p.queries + query] = total == 0.0f ? __builtin_inff() : most + __builtin_amdgcn_logf(total);
  } else {
    // the waves' maxima and sums, then each wave adds up its share of the values
    constexpr int kAll = ND * 16, kShare = kAll / WAVES;
    static_assert((WAVES * kAll + 2 * WAVES) * 256 <= (int)sizeof(memory) || WAVES == 1, "the rings hold the waves' results");
    __attribute__((address_space(3))) float* const all = (__attribute__((address_space(3))) float*)(lds_u8*)memory;
    __attribute__((address_space(3))) float* const stats = all + WAVES * kAll * 64;
    meet();
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int e = 0; e < 16; e++) all[(wave * kAll + 16 * d + e) * 64 + lane] = acc[d][e];
    stats[(2 * wave) * 64 + lane] = most;
    stats[(2 * wave + 1) * 64 + lane] = total;
    __syncthreads();
    float factor[WAVES];
    most = -__builtin_inff();
#pragma unroll
    for (int o = 0; o < WAVES; o++) most = __builtin_fmaxf(most, stats[(2 * o) * 64 + lane]);
    total = 0.0f;
#pragma unroll
    for (int o = 0; o < WAVES; o++) {
      const float m = stats[(2 * o) * 64 + lane];
      factor[o] = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - most);
      total = __builtin_fmaf(stats[(2 * o + 1) * 64 + lane], factor[o], total);
    }
    const bool whole = p.splits == 1;
    const float scale = !whole ? 1.0f : total > 0.0f ? 1.0f / total : total;
    const int64_t place = (((int64_t)bh * p.tiles + tile) * p.splits + split) * 32 + (lane & 31);
    char* const row = (char*)p.out.at(b, head, query);
#pragma unroll
    for (int n = 0; n < kShare; n += 4) {
      const int k = wave * kShare + n, col = 32 * (k / 16) + row_of(k % 16) + 4 * (lane >> 5);
      f32x4 v;
#pragma unroll
      for (int t = 0; t < 4; t++) {
        v[t] = 0.0f;
#pragma unroll
        for (int o = 0; o < WAVES; o++) v[t] = __builtin_fmaf(all[(o * kAll + k + t) * 64 + lane], factor[o], v[t]);
        v[t] *= scale;
      }
      if (!own || col >= p.width) continue;
      if (whole) {
        store4<T>(row, p.rest_at(b, head, query), col, v);
      } else {
        *(f32x4*)(p.part + place * DP + col) = v;
      }
    }
    if (own && wave == 0 && lane < 32) {
      if (!whole)
        *(f32x2*)(p.part_stats + place * 2) = f32x2{most, total};
      else if (p.lse)
        p.lse[((int64_t)b * p.heads + head) * p.queries + query] = total == 0.0f ? __builtin_inff() : most + __builtin_amdgcn_logf(total);
    }
  }
}

// The splits' results as one.
struct Joined {
  int64_t first;      // its place in split 0 of its tile
  int b, head, query;
};
__device__ __forceinline__ bool row_to_join(const AttentionArgs& p, int64_t at, Joined& j) {
  const int rows = p.group * p.queries, row = (int)(at % rows);
  const int64_t bh = at / rows;
  if (bh >= (int64_t)(p.blocks / p.splits / p.tiles)) return false;
  j = Joined{(bh * p.tiles + row / 32) * p.splits * 32 + row % 32, (int)(bh / p.kv_heads), (int)(bh % p.kv_heads) * p.group + row / p.queries, row % p.queries};
  return true;
}
template <typename T>
__device__ __forceinline__ void store_joined(const AttentionArgs& p, const Joined& j, int lane, f32x4 sum, float total, float most) {
  sum *= total > 0.0f ? 1.0f / total : total;
  if (lane * 4 < p.width) store4<T>((char*)p.out.at(j.b, j.head, j.query), p.rest_at(j.b, j.head, j.query), lane * 4, sum);
  if (p.lse && lane == 0) p.lse[((int64_t)j.b * p.heads + j.head) * p.queries + j.query] = total == 0.0f ? __builtin_inff() : most + __builtin_amdgcn_logf(total);
}
// Few of them: DP / 4 lanes have a row (8 heads of 512 tokens, two splits: 4 us, 7.5 with the kernel below; with up to eight splits this way 5.9 where the
// other takes 4.2)
constexpr int kFewSplits = 4;
template <typename T, int DP>
__global__ __launch_bounds__(256) void attention_join_few_kernel(AttentionArgs p) {
  constexpr int kLanes = DP / 4, kDown = 256 / kLanes;
  const int lane = threadIdx.x % kLanes, down = threadIdx.x / kLanes;
  Joined j;
  if (down >= kDown || !row_to_join(p, block_of() * kDown + down, j)) return;
  f32x2 stat[kFewSplits];
  f32x4 part[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; s++) {      // all on their way at once
    const int64_t place = j.first + 32 * (int64_t)(s < p.splits ? s : 0);
    stat[s] = *(const f32x2*)(p.part_stats + place * 2);
    if (lane * 4 < p.width) part[s] = *(const f32x4*)(p.part + place * DP + lane * 4);
  }
  float most = stat[0][0];
#pragma unroll
  for (int s = 1; s < kFewSplits; s++) most = __builtin_fmaxf(most, stat[s][0]);
  f32x4 sum = {};
  float total = 0.0f;
#pragma unroll
  for (int s = 0; s < kFewSplits; s++) {
    if (s >= p.splits) break;
    const float factor = stat[s][0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(stat[s][0] - most);
    total = __builtin_fmaf(stat[s][1], factor, total);
    sum += part[s] * factor;
  }
  store_joined<T>(p, j, lane, sum, total, most);
}
// Many: a workgroup has a row, its lanes the width, its waves the splits.  Latency: a launch, and three loads one after the other (32 rows, 32 splits of
// width 128: 5 us)
template <typename T, int DP>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs p) {
  constexpr int kLanes = DP / 4, kDown = 256 / kLanes;
  __shared__ f32x4 sums[kDown][kLanes];
  __shared__ float totals[kDown];
  const int lane = threadIdx.x % kLanes, down = threadIdx.x / kLanes;
  Joined j;
  if (!row_to_join(p, block_of(), j)) return;
  const int64_t first = j.first;
  __shared__ float mosts[4];
  float most = -__builtin_inff();
  for (int s = threadIdx.x; s < p.splits; s += 256) most = __builtin_fmaxf(most, p.part_stats[(first + 32 * (int64_t)s) * 2]);
  most = over_lanes<Most, 64>(most);
  if ((threadIdx.x & 63) == 0) mosts[threadIdx.x >> 6] = most;
  __syncthreads();
  most = __builtin_fmaxf(__builtin_fmaxf(mosts[0], mosts[1]), __builtin_fmaxf(mosts[2], mosts[3]));
  f32x4 sum = {};
  float total = 0.0f;
  if (down < kDown) {
    for (int s = down; s < p.splits; s += kDown) {
      const int64_t place = first + 32 * (int64_t)s;
      const f32x2 stat = *(const f32x2*)(p.part_stats + place * 2);
      const float factor = stat[0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(stat[0] - most);
      total = __builtin_fmaf(stat[1], factor, total);
      if (lane * 4 < p.width) sum += *(const f32x4*)(p.part + place * DP + lane * 4) * factor;
    }
    sums[down][lane] = sum;
    if (lane == 0) totals[down] = total;
  }
  __syncthreads();
  if (down != 0) return;
  sum = f32x4{};
  total = 0.0f;
  for (int d = 0; d < kDown; d++) {
    sum += sums[d][lane];
    total += totals[d];
  }
  store_joined<T>(p, j, lane, sum, total, most);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// dq, and do_i.o_i for the other kernel.  With a bias: the sums of ds along the diagonals, for the wave's 32 queries.  Element e of a block of 32 keys is
// key row_of(e) + 4 g of query l = 16 half + m of the lane (its row of 16 lanes: g and half); its diagonal, key - query, moves by one with either.  Shifted
// down its row of lanes by row_of(e) mod 16, lane m has the diagonals 16 c - m + 4 g - 16 half of all elements, where c is 0 for what stays in the row,
// 1 for what leaves it, and one more for the keys from 16 on: three running sums a lane, two additions an element that shift as they add.  After a block
// the sums of c = 0 and 1 are complete and the one of 2 is the next block's 0.  The four rows' sums, each a sequence along c and -m, meet in LDS.
// Three products, and two of 16-bit types for what rounding leaves out; bound as the forward pass is: 32 x 16 heads of 512 tokens, width 64, bfloat16 80 us;
// 8 x 16 of 1000, halves, with a bias 116, of which the diagonals take 30.
// (Additions into LDS by the hardware's atomics, 16 a block: 750 us for 8 x 16 heads of 1000 x 1000 halves where the kernel without them takes 100.)
// ---------------------------------------------------------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ float shifted(float v) {      // lane m of a row of 16: the value of lane m + N, zero behind the row's end (N < 0: before its beginning)
  constexpr int kControl = N > 0 ? 0x100 + N : 0x110 - N;
  const int b = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, b, kControl, 0xf, 0xf, true));
}
template <int E = 0>
__device__ __forceinline__ void add_diagonals(const f32x16& s, float (&sums)[3]) {
  if constexpr (E < 16) {
    constexpr int kShift = row_of(E) % 16, kUp = row_of(E) / 16;
    if constexpr (kShift == 0) {
      sums[kUp] += s[E];
    } else {
      sums[kUp] += shifted<kShift>(s[E]);
      sums[kUp + 1] += shifted<kShift - 16>(s[E]);
    }
    add_diagonals<E + 1>(s, sums);
  }
}
template <typename T, int DP, int WAVES, bool BIAS>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(waves_held<T, DP>(DQ)))) void attention_dq_kernel(AttentionArgs p) {
  using Shape = Tile<T, DP, WAVES>;
  using Frag = typename Shape::Frag;
  constexpr int R = Shape::kRows, NB = R / 32, W = Shape::W, NC = Shape::NC, ND = Shape::ND, BM = WAVES * 32;
  constexpr int kTile = R * W, kBias = BIAS ? (BM + R + 63) / 64 * 256 : 0;
  using Load = RowsLoad<T, DP, R, WAVES>;
  __shared__ __attribute__((aligned(1024))) uint8_t memory[4 * kTile + 2 * kBias];
  __shared__ float diagonals[BIAS ? WAVES : 1][4][64];      // the last 64 of each row's sequence
  Work work;
  if (!work_of(p, p.splits, work)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_u8* const ring = (lds_u8*)memory;
  lds_u8* const biases = ring + 4 * kTile;
  const int split = work.tile % p.splits, turn = work.tile / p.splits, tile = p.causal ? p.tiles - 1 - turn : turn;
  const uint32_t bh = work.head;
  const int b = bh / p.heads, h = bh % p.heads, kv = h / p.group;
  const int first = tile * BM + wave * 32, mine = first + (lane & 31), last = tile * BM + BM - 1;
  const bool own = mine < p.queries;
  const int query = own ? mine : p.queries - 1;
  Frag q[NC], dy[NC];
  own_row<T, NC>(p.q.at(b, h, query), own, p.width, lane, q);
  own_row<T, NC>(p.d_out.at(b, h, query), own, p.width, lane, dy);
  const int64_t at = ((int64_t)b * p.heads + h) * p.queries + query;
  const float lse = own ? p.lse[at] : __builtin_inff();
  if (p.blind && __ballot(lse == __builtin_inff())) {
#pragma unroll
    for (int c = 0; c < NC; c++)
      if (lse == __builtin_inff()) dy[c] = Frag{};
  }
  float delta;
  {
    Frag o[NC];
    own_row<T, NC>(p.out.at(b, h, query), own, p.width, lane, o);
    delta = delta_of<T, NC>(o, dy, p.rest_at(b, h, query), p.width, lane);
    if (own && lane < 32 && split == 0) p.delta[at] = -delta;
  }
  const int seen = p.seen(query);
  const int all_see = p.seen(first < p.queries ? first : p.queries - 1), some_see = p.seen(first + 31 < p.queries ? first + 31 : p.queries - 1);
  const int from = split * p.per_split;
  int to = p.seen(last < p.queries ? last : p.queries - 1);
  if (p.splits > 1 && from + p.per_split < to) to = from + p.per_split;
  const int steps = to > from ? (to - from + R - 1) / R : 0;

  Load load_k, load_v;
  load_k.set_up(p.k.row, p.width, wave, lane);
  load_v.set_up(p.v.row, p.width, wave, lane);
  Present present{p.mask ? p.mask + (int64_t)b * p.mask_stride : nullptr, p.keys};
  load_k.start(p.k.at(b, kv, from), p.keys - from, p.k.row, p.width);
  load_v.start(p.v.at(b, kv, from), p.keys - from, p.v.row, p.width);
  auto issue = [&](int t, uint64_t there) __attribute__((always_inline)) {
    lds_u8* const to = ring + (t & 1) * 2 * kTile;
    load_k.next(p.mask != nullptr, there, to, lane);
    load_v.next(p.mask != nullptr, there, to + kTile, lane);
    if constexpr (BIAS)
      load_floats(p.bias + (int64_t)h * p.distances(), p.distances(), from + t * R - last + p.queries - 1, BM + R - 1, wave, WAVES, biases + (t & 1) * kBias, lane);
  };
  f32x16 acc[ND];
  float up = Up<T>::kBegin;
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = f32x16{};
  typedef __attribute__((address_space(3))) float lds_float;
  lds_float* const sequence = (lds_float*)diagonals[BIAS ? wave : 0][0];
  float sums[3] = {};
  if constexpr (BIAS) {
#pragma unroll
    for (int n = 0; n < 4; n++) sequence[64 * n + lane] = 0.0f;
  }
  // block k is done: numbers 32 k to 32 k + 31 of the wave's diagonals, which begin at the first key and the last query, are complete.  Number y of a row's
  // sequence, 16 c - m + 15, belongs to number y + 4 g + 16 (1 - half)
  auto leave = [&](int k, float* to) __attribute__((always_inline)) {
    const int at = (32 * k + 15 - (lane & 15)) & 63;
    in_turn();
    sequence[64 * (lane >> 4) + at] = sums[0];
    sequence[64 * (lane >> 4) + ((at + 16) & 63)] = sums[1];
    in_turn();
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 4; n++) sum += sequence[64 * n + ((32 * k + (lane & 31) - 4 * (n >> 1) - 16 * (1 - (n & 1))) & 63)];
    if (lane < 32) to[32 * k + lane] = sum;
    sums[0] = sums[2];
    sums[1] = sums[2] = 0.0f;
  };
  // of the diagonals of the wave's queries, which begin at the split's first key and query first + 31
  float* const along = BIAS && p.along ? p.along + (((bh * (int64_t)p.tiles + tile) * WAVES + wave) * p.splits + split) * p.along_stride : nullptr;

  float scale2 = p.scale2;
  asm("" : "+v"(scale2));
  // what the sums of do_i.v_j begin with, in registers of its own; floats have none to spare, and their instructions take far longer than a subtraction
  constexpr bool kBegin = sizeof(T) == 2;
  f32x16 minus = {};
  if constexpr (kBegin) {
#pragma unroll
    for (int e = 0; e < 16; e++) minus[e] = -delta;
    asm("" : "+v"(minus));
  }
  uint64_t there = 0, next = 0;
  present.ask(from + lane);
  next = present.answer();
  if (steps > 0) issue(0, next);
  present.ask(from + R + lane);
  for (int t = 0; t < steps; t++) {
    wait_all();
    meet();
    __builtin_amdgcn_sched_barrier(0);
    there = next;
    next = present.answer();
    if (t + 1 < steps) issue(t + 1, next);
    present.ask(from + (t + 2) * R + lane);
    const int key = from + t * R;
    const lds_u8* const keys = ring + (t & 1) * 2 * kTile;
    const bool edge = key + R > all_see || (p.mask && (R == 64 ? ~there : ~there & 0xffffffffu) != 0);
    auto product = [&](const lds_u8* rows, int n, const Frag (&own)[NC], f32x16 s) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < NC; c++) s = Matrix<T>::run(Shape::direct(rows, 32 * n, c, lane), own[c], s);
      return s;
    };
    // ds of a block from its scores and do.v - do.o; `hidden`: with some of them hidden
    auto gradient = [&](int n, f32x16 s, const f32x16& dp, bool hidden) __attribute__((always_inline)) {
      const int g4 = 4 * (lane >> 5);
#pragma unroll
      for (int e = 0; e < 16; e++) {
        float off = -lse;
        if constexpr (BIAS)
          off += ((const lds_float*)(biases + (t & 1) * kBias))[32 * n + row_of(e) + g4 - (wave * 32 + (lane & 31)) + BM - 1];
        s[e] = __builtin_fmaf(s[e], scale2, off);
      }
      if (hidden) hide(s, seen - key - 32 * n, (uint32_t)(there >> (32 * n)), lane);
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = __builtin_amdgcn_exp2f(s[e]) * (kBegin ? dp[e] : dp[e] - delta);
      if constexpr (BIAS)
        if (along) add_diagonals(s, sums);
      return s;
    };
#pragma unroll
    for (int n = 0; n < NB; n++) {
      if (key + 32 * n < some_see && there) {
        const f32x16 ds = gradient(n, product(keys, n, q, f32x16{}), product(keys + kTile, n, dy, minus), edge);
        add_ds<T, DP, WAVES>(acc, up, keys, 32 * n, ds, lane);
      }
      if constexpr (BIAS)
        if (along) leave(t * NB + n, along);
    }
  }
  wait_all();
  if constexpr (BIAS)
    if (along) leave(steps * NB, along);
  if (!own || !p.dq.p) return;
  if (p.splits > 1)
    store_part<DP, ND>(p.part + (((int64_t)split * (p.blocks / p.splits / p.tiles) + bh) * p.tiles * BM + mine) * DP, p.width, lane, acc, Up<T>::down(up));
  else
    store_row<T, ND>((char*)p.dq.at(b, h, query), nullptr, p.width, lane, acc, p.scale * Up<T>::down(up));
}

// ---------------------------------------------------------------------------------------------------------------------------------
// dk and dv: a wave has 32 keys, and the queries of all heads that share the key head pass by.  No sums through atomics: a result has the same bits every
// time, for seven products in two kernels where one with atomics for dq would make five.  32 x 16 heads of 512 tokens, width 64, bfloat16: 101 us, bound as
// the forward pass is; nothing that is loaded at the beginning waits for the mask (2 us).
// ---------------------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int WAVES, bool BIAS>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(waves_held<T, DP>(DKV)))) void attention_dkv_kernel(AttentionArgs p) {
  using Shape = Tile<T, DP, WAVES>;
  using Frag = typename Shape::Frag;
  constexpr int R = Shape::kRows, NB = R / 32, W = Shape::W, NC = Shape::NC, ND = Shape::ND, BM = WAVES * 32;
  constexpr int kTile = R * W, kBias = BIAS ? (BM + R + 63) / 64 * 256 : 0, kStats = 256;
  using Load = RowsLoad<T, DP, R, WAVES>;
  typedef __attribute__((address_space(3))) float lds_float;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  __shared__ __attribute__((aligned(1024))) uint8_t memory[4 * kTile + 4 * kStats + 2 * kBias];
  Work work;
  if (!work_of(p, p.splits, work)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_u8* const ring = (lds_u8*)memory;
  lds_u8* const stats = ring + 4 * kTile;
  lds_u8* const biases = stats + 4 * kStats;
  const int split = work.tile % p.splits, tile = work.tile / p.splits;
  const uint32_t bh = work.head;
  const int b = bh / p.kv_heads, kv = bh % p.kv_heads;
  const int first = tile * BM + wave * 32, key = first + (lane & 31);
  // which of the workgroup's keys there are, two bytes to a lane.  Nothing that is loaded waits for it
  uint32_t present[BM / 64];
#pragma unroll
  for (int n = 0; n < BM / 64; n++) {
    const int at = tile * BM + 64 * n + lane;
    present[n] = at < p.keys;
    if (p.mask && at < p.keys) present[n] = p.mask[(int64_t)b * p.mask_stride + at];
  }
  Frag k[NC], v[NC];
  own_row<T, NC>(p.k.at(b, kv, key), key < p.keys, p.width, lane, k);
  own_row<T, NC>(p.v.at(b, kv, key), key < p.keys, p.width, lane, v);
  // queries from `seen_from` on see the lane's key
  const int behind = p.keys - p.queries;
  const int seen_from = p.causal && key > behind ? key - behind : 0;
  const int all_from = p.causal && first + 31 > behind ? first + 31 - behind : 0, some_from = p.causal && first > behind ? first - behind : 0;
  const int begin = (p.causal && tile * BM > behind ? tile * BM - behind : 0) / R * R;
  const int per_head = begin < p.queries ? (p.queries - begin + R - 1) / R : 0;
  // the split's share of the tiles of queries of all heads, one after the other
  const int all_steps = per_head * p.group;
  const int first_step = (int)((int64_t)all_steps * split / p.splits), planned = (int)((int64_t)all_steps * (split + 1) / p.splits) - first_step;

  Load load_q, load_dy;
  load_q.set_up(p.q.row, p.width, wave, lane);
  load_dy.set_up(p.d_out.row, p.width, wave, lane);
  // the next tile to load: of head `head`, from query `ahead` on
  int head = kv * p.group, ahead = begin;
  if (planned > 0) {
    head += first_step / per_head;
    ahead += first_step % per_head * R;
  }
  int now = ahead;
  const float* stat = nullptr;
  auto issue = [&](int t) __attribute__((always_inline)) {
    if (ahead >= p.queries || t == 0) {
      if (t) {
        head++;
        ahead = begin;
      }
      load_q.start(p.q.at(b, head, ahead), p.queries - ahead, p.q.row, p.width);
      load_dy.start(p.d_out.at(b, head, ahead), p.queries - ahead, p.d_out.row, p.width);
      stat = (wave ? p.delta : p.lse) + ((int64_t)b * p.heads + head) * p.queries;
    }
    lds_u8* const to = ring + (t & 1) * 2 * kTile;
    load_q.next(false, 0, to, lane);
    load_dy.next(false, 0, to + kTile, lane);
    if (wave < 2) load_floats(stat, p.queries, ahead, R, 0, 1, stats + (2 * (t & 1) + wave) * kStats, lane);
    if constexpr (BIAS)
      load_floats(p.bias + (int64_t)head * p.distances(), p.distances(), tile * BM - (ahead + R - 1) + p.queries - 1, BM + R - 1, wave, WAVES,
                  biases + (t & 1) * kBias, lane);
    ahead += R;
  };
  f32x16 dk[ND], dv[ND];
  float up = Up<T>::kBegin;
#pragma unroll
  for (int d = 0; d < ND; d++) dk[d] = dv[d] = f32x16{};

  float scale2 = p.scale2;
  asm("" : "+v"(scale2));
  if (planned > 0) issue(0);
  bool own = false, some = false;
#pragma unroll
  for (int n = 0; n < BM / 64; n++) {
    const uint64_t keys = __ballot(present[n] != 0);
    some |= keys != 0;
    if (wave / 2 == n) own = keys >> (wave % 2 * 32 + (lane & 31)) & 1;
  }
  if (!own) {
#pragma unroll
    for (int c = 0; c < NC; c++) k[c] = v[c] = Frag{};
  }
  const int steps = some ? planned : 0;      // no key of the workgroup's is there: only zeros to store
  for (int t = 0; t < steps; t++) {
    wait_all();
    meet();
    __builtin_amdgcn_sched_barrier(0);
    if (t + 1 < steps) issue(t + 1);
    const int query = now;
    now += R;
    if (now >= p.queries) now = begin;
    const lds_u8* const rows = ring + (t & 1) * 2 * kTile;
    const lds_float* const lse = (const lds_float*)(stats + 2 * (t & 1) * kStats);
    const lds_float* const delta = (const lds_float*)(stats + (2 * (t & 1) + 1) * kStats);
    // (with a mask alone a query that sees nothing is one of a batch entry without keys, which has no steps)
    if (BIAS || (p.causal && p.blind))
      if (clear_blind<W, R, WAVES>(ring + (t & 1) * 2 * kTile + kTile, lse, wave, lane)) meet();
    const bool edge = query < all_from || query + R > p.queries;
    auto product = [&](const lds_u8* from, int n, const Frag (&own)[NC], f32x16 s) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < NC; c++) s = Matrix<T>::run(Shape::direct(from, 32 * n, c, lane), own[c], s);
      return s;
    };
    // what the sums of do_i.v_j of a block begin with
    auto minus = [&](int n) __attribute__((always_inline)) {
      f32x16 x;
#pragma unroll
      for (int e4 = 0; e4 < 16; e4 += 4) {
        const f32x4 part = *(const lds_f32x4*)(delta + 32 * n + row_of(e4) + 4 * (lane >> 5));
#pragma unroll
        for (int e = 0; e < 4; e++) x[e4 + e] = part[e];
      }
      return x;
    };
    // a block's scores to probabilities, and do.v - do.o to ds
    auto gradient = [&](int n, f32x16& s, f32x16& dp, bool hidden) __attribute__((always_inline)) {
      const int g4 = 4 * (lane >> 5);
#pragma unroll
      for (int e4 = 0; e4 < 16; e4 += 4) {
        const f32x4 l = *(const lds_f32x4*)(lse + 32 * n + row_of(e4) + g4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float off = -l[e];
          if constexpr (BIAS)
            off += ((const lds_float*)(biases + (t & 1) * kBias))[wave * 32 + (lane & 31) - (32 * n + row_of(e4) + e + g4) + R - 1];
          s[e4 + e] = __builtin_fmaf(s[e4 + e], scale2, off);
        }
      }
      if (hidden) {
        asm volatile("");
        const int from = seen_from - query - 32 * n - g4, to = p.queries - query - 32 * n - g4;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = row_of(e) >= from && row_of(e) < to ? s[e] : -__builtin_inff();
      }
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[e] = __builtin_amdgcn_exp2f(s[e]);
        dp[e] *= s[e];
      }
    };
#pragma unroll
    for (int n = 0; n < NB; n++) {
      if (query + 32 * n + 31 < some_from || query + 32 * n >= p.queries) continue;
      f32x16 s = product(rows, n, k, f32x16{}), dp = product(rows + kTile, n, v, minus(n));
      gradient(n, s, dp, edge);
      Shape::add(dv, rows + kTile, 32 * n, Up<T>::template probabilities<Shape>(s), lane);
      add_ds<T, DP, WAVES>(dk, up, rows, 32 * n, dp, lane);
    }
  }
  wait_all();
  if (key >= p.keys) return;
  // an absent key's lane has seen zeros for it
  const float there = own ? 1.0f : 0.0f;
  if (!own) {
#pragma unroll
    for (int d = 0; d < ND; d++) dk[d] = dv[d] = f32x16{};
  }
  if (p.splits > 1) {
    const int64_t heads = p.blocks / p.splits / p.tiles, row = ((split * heads + bh) * p.tiles * BM + key) * DP;
    if (p.dk.p) store_part<DP, ND>(p.part + row, p.width, lane, dk, Up<T>::down(up));
    if (p.dv.p) store_part<DP, ND>(p.part + p.splits * heads * p.tiles * BM * DP + row, p.width, lane, dv, Up<T>::kDown);
    return;
  }
  if (p.dk.p) store_row<T, ND>((char*)p.dk.at(b, kv, key), nullptr, p.width, lane, dk, p.scale * Up<T>::down(up) * there);
  if (p.dv.p) store_row<T, ND>((char*)p.dv.at(b, kv, key), nullptr, p.width, lane, dv, Up<T>::kDown * there);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// dq, dk and dv of sequences of up to 64 queries and keys in one pass: a workgroup has a key head and takes the heads that share it one after the other.
// Five products instead of the seven of two kernels, and every operand read once: dk's and dv's leave ds with a key to a lane, which passes through LDS, in
// the place of the queries and of dy, to become a query to a lane for dq.  24576 heads of 49 tokens of width 32: 420 us in floats, 575 in two kernels, and
// 218 and 282 in bfloat16; 6144 of 64 tokens, width 64: 133 and 182.  The matrix unit is busy for half the time (the products of 64 x 64 take 205 us of the
// 420); the rest goes to the loads and the four meetings of two waves that three workgroups beside each other do not cover.
// ---------------------------------------------------------------------------------------------------------------------------------
template <typename T, int DP>
constexpr bool kShortFits = DP * sizeof(T) <= 256;
template <typename T, int DP>
__global__ __launch_bounds__(128) __attribute__((amdgpu_waves_per_eu(waves_held<T, DP>(SHORT)))) void attention_short_kernel(AttentionArgs p) {
  using Shape = Tile<T, DP, 2>;
  using Frag = typename Shape::Frag;
  constexpr int R = 64, W = Shape::W, NC = Shape::NC, ND = Shape::ND;
  constexpr int kTile = R * W, kRow = (R + 4) * 4, kDs = R * kRow, kShared = 2 * kTile > kDs ? 2 * kTile : kDs;
  using Load = RowsLoad<T, DP, R, 2>;
  typedef __attribute__((address_space(3))) float lds_float;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  __shared__ __attribute__((aligned(1024))) uint8_t memory[kTile + kShared + 2 * R * 4];
  Work work;
  if (!work_of(p, 1, work)) return;
  const int thread = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_u8* const keys = (lds_u8*)memory;
  lds_u8* const queries = keys + kTile;
  lds_float* const lse = (lds_float*)(queries + kShared);
  lds_float* const deltas = lse + R;
  const int b = work.head / p.kv_heads, kv = work.head % p.kv_heads;
  const int first = wave * 32;
  int lane = thread, mine = first + (lane & 31);      // the lane's key, and its query
  Load load;
  load.set_up(p.k.row, p.width, wave, lane);
  Present present{p.mask ? p.mask + (int64_t)b * p.mask_stride : nullptr, p.keys};
  present.ask(lane);
  const uint64_t there = present.answer();
  load.start(p.k.at(b, kv, 0), p.keys, p.k.row, p.width);
  load.next(p.mask != nullptr, there, keys, lane);
  const bool own = mine < p.keys && (there >> mine & 1);
  Frag k[NC], v[NC];
  own_row<T, NC>(p.v.at(b, kv, mine), own, p.width, lane, v);
  const int behind = p.keys - p.queries;
  const int seen_from = p.causal && mine > behind ? mine - behind : 0;
  const int all_from = p.causal && first + 31 > behind ? first + 31 - behind : 0, some_from = p.causal && first > behind ? first - behind : 0;
  // keys that the wave's queries see
  const int some_see = first < p.queries ? p.seen(first + 31 < p.queries ? first + 31 : p.queries - 1) : 0;
  const bool all_own = __ballot(own) == ~0ull;
  // queries before it see nothing, and zeros take the place of their gradients, which are nobody's
  const uint64_t keys_there = p.keys < 64 ? there & ((1ull << p.keys) - 1) : there;
  const int first_key = keys_there ? __builtin_ctzll(keys_there) : 0;
  const int sees_from = !keys_there ? 64 : p.causal && first_key > behind ? first_key - behind : 0;
  f32x16 dk[ND], dv[ND];
  float up = Up<T>::kBegin;
#pragma unroll
  for (int d = 0; d < ND; d++) dk[d] = dv[d] = f32x16{};
  float scale2 = p.scale2;
  asm("" : "+v"(scale2));
  for (int g = 0; g < p.group; g++) {
    const int head = kv * p.group + g;
    if (g) meet();
    // addresses anew for each head: kept, they would take more registers than there are for three waves
    lane = thread;
    asm volatile("" : "+v"(lane));
    mine = first + (lane & 31);
    const int g4 = 4 * (lane >> 5);
    // ds: rows of 64 keys, 16 bytes apart, so that neighbouring rows' pieces lie in different banks
    lds_u8* const ds_of_key = queries + g4 * kRow + mine * 4;
    const lds_u8* const ds_of_query = queries + mine * kRow + g4 * 4;
    load.set_up(p.q.row, p.width, wave, lane);
    load.start(p.q.at(b, head, 0), p.queries, p.q.row, p.width);
    load.next(false, 0, queries, lane);
    load.set_up(p.d_out.row, p.width, wave, lane, sees_from);
    load.start(p.d_out.at(b, head, 0), p.queries, p.d_out.row, p.width);
    load.next(false, 0, queries + kTile, lane);
    const int64_t at = ((int64_t)b * p.heads + head) * p.queries;
    if (wave == 0) load_floats(p.lse + at, p.queries, 0, R, 0, 1, (lds_u8*)lse, lane);
    {
      Frag o[NC], dy[NC];
      own_row<T, NC>(p.out.at(b, head, mine), mine < p.queries, p.width, lane, o);
      wait_all();
      meet();
#pragma unroll
      for (int c = 0; c < NC; c++) dy[c] = Shape::direct(queries + kTile, first, c, lane);
      const float delta = delta_of<T, NC>(o, dy, mine < p.queries ? p.rest_at(b, head, mine) : nullptr, p.width, lane);
      if (lane < 32) deltas[mine] = delta;
    }
    if (g == 0) {
#pragma unroll
      for (int c = 0; c < NC; c++) k[c] = Shape::direct(keys, first, c, lane);
    }
    meet();
    f32x16 ds[2] = {};
#pragma unroll
    for (int n = 0; n < 2; n++) {
      if (32 * n + 31 < some_from || 32 * n >= p.queries || first >= p.keys) continue;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < NC; c++) s = Matrix<T>::run(Shape::direct(queries, 32 * n, c, lane), k[c], s);
#pragma unroll
      for (int c = 0; c < NC; c++) dp = Matrix<T>::run(Shape::direct(queries + kTile, 32 * n, c, lane), v[c], dp);
#pragma unroll
      for (int e4 = 0; e4 < 16; e4 += 4) {
        const f32x4 l = *(const lds_f32x4*)(lse + 32 * n + row_of(e4) + g4);
#pragma unroll
        for (int e = 0; e < 4; e++) s[e4 + e] = __builtin_fmaf(s[e4 + e], scale2, -l[e]);
      }
      if (32 * n < all_from || 32 * n + 32 > p.queries || !all_own) {
        int from = seen_from - 32 * n - g4, to = own ? p.queries - 32 * n - g4 : -64;
        asm volatile("" : "+v"(from), "+v"(to));      // compared anew for each head: what the comparisons leave would fill the scalar registers
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = row_of(e) >= from && row_of(e) < to ? s[e] : -__builtin_inff();
      }
#pragma unroll
      for (int e4 = 0; e4 < 16; e4 += 4) {
        const f32x4 x = *(const lds_f32x4*)(deltas + 32 * n + row_of(e4) + g4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s[e4 + e] = __builtin_amdgcn_exp2f(s[e4 + e]);
          ds[n][e4 + e] = s[e4 + e] * (dp[e4 + e] - x[e]);
        }
      }
      Shape::add(dv, queries + kTile, 32 * n, Up<T>::template probabilities<Shape>(s), lane);
      add_ds<T, DP, 2>(dk, up, queries, 32 * n, ds[n], lane);
      __builtin_amdgcn_sched_barrier(0);
    }
    meet();
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 16; e++) *(lds_float*)(ds_of_key + (32 * n + row_of(e)) * kRow) = ds[n][e];
    meet();
    f32x16 dq[ND];
    float dq_up = Up<T>::kBegin;
#pragma unroll
    for (int d = 0; d < ND; d++) dq[d] = f32x16{};
#pragma unroll
    for (int n = 0; n < 2; n++) {
      if (32 * n >= some_see) continue;
      f32x16 x;
#pragma unroll
      for (int e4 = 0; e4 < 16; e4 += 4) {
        const f32x4 part = *(const lds_f32x4*)(ds_of_query + (32 * n + row_of(e4)) * 4);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e4 + e] = part[e];
      }
      add_ds<T, DP, 2>(dq, dq_up, keys, 32 * n, x, lane);
    }
    if (mine < p.queries && p.dq.p) store_row<T, ND>((char*)p.dq.at(b, head, mine), nullptr, p.width, lane, dq, p.scale * Up<T>::down(dq_up));
  }
  if (mine >= p.keys) return;
  if (!own) {
#pragma unroll
    for (int d = 0; d < ND; d++) dk[d] = dv[d] = f32x16{};
  }
  if (p.dk.p) store_row<T, ND>((char*)p.dk.at(b, kv, mine), nullptr, p.width, lane, dk, p.scale * Up<T>::down(up));
  if (p.dv.p) store_row<T, ND>((char*)p.dv.at(b, kv, mine), nullptr, p.width, lane, dv, Up<T>::kDown);
}

// out = factor times the sum of the splits' rows, in their order; which of two outputs: blockIdx.z.  Four columns to a lane, four loads on their way.  Latency:
// 3 x 6 heads of 197 queries of width 72, 6 splits, 4 us; dq, dk and dv of 4096 rows of width 128, 8 splits (50 MB), 10.7 in two launches.
struct PartRows {
  const float* part[2];
  Side out[2];
  float factor[2];
  int64_t rows;              // of all heads
  int heads, length, padded, splits, width;
};
template <typename T, int DP>
__global__ __launch_bounds__(256) void attention_add_kernel(PartRows p) {
  constexpr int kLanes = DP / 4, kDown = 256 / kLanes;
  const int lane = threadIdx.x % kLanes, down = threadIdx.x / kLanes;
  const int64_t row = block_of() * kDown + down;
  if (down >= kDown || row >= p.rows || lane * 4 >= p.width) return;
  const int64_t bh = row / p.length, n = row - bh * p.length, apart = p.rows / p.length * p.padded * DP;
  const int z = blockIdx.z;
  const float* from = p.part[z] + (bh * p.padded + n) * DP + lane * 4;
  f32x4 sum = {};
  int k = 0;
  for (; k + 4 <= p.splits; k += 4) {
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = *(const f32x4*)(from + (k + u) * apart);
#pragma unroll
    for (int u = 0; u < 4; u++) sum += v[u];
  }
  for (; k < p.splits; k++) sum += *(const f32x4*)(from + k * apart);
  store4<T>((char*)p.out[z].at(bh / p.heads, bh % p.heads, n), nullptr, lane * 4, sum * p.factor[z]);
}

// ---- launches ----
// the width rounded up to whole blocks of the products
template <typename F>
int with_width(int width, F&& f) {
  using std::integral_constant;
  if (width <= 32) return f(integral_constant<int, 32>{});
  if (width <= 64) return f(integral_constant<int, 64>{});
  if (width <= 96) return f(integral_constant<int, 96>{});
  return f(integral_constant<int, 128>{});
}
template <typename K>
int launch(K kernel, int64_t blocks, int threads, const AttentionArgs& p, hipStream_t s) {
  if (blocks == 0) return GACT_OK;
  if (!blocks_fit(blocks)) return GACT_ELIMIT;
  hipLaunchKernelGGL(kernel, grid_of(blocks, threads), dim3((unsigned)threads), 0, s, p);
  return launch_status();
}

// few queries: waves of a workgroup that take the keys in turn, as many as LDS holds tiles for
template <typename T, int DP>
constexpr int apart_waves() { return Tile<T, DP>::W == 512 ? 2 : 4; }

}  // namespace

// what attention.hip asks of the three sources; `waves` of a workgroup: 2 or 4; `apart` as above
template <typename T>
int attention_forward(AttentionArgs p, int64_t batch, int waves, bool apart, hipStream_t s) {
  return with_width(p.width, [&](auto width) {
    constexpr int DP = decltype(width)::value, A = apart_waves<T, DP>();
    const int64_t heads = batch * (apart ? p.kv_heads : p.heads), rows = apart ? (int64_t)p.group * p.queries : p.queries;
    const int64_t tall = apart ? 32 : waves * 32, tiles = (rows + tall - 1) / tall, blocks = heads * tiles * (apart ? p.splits : 1);
    p.tiles = (uint32_t)tiles;
    p.blocks = (uint32_t)blocks;
    p.by_length = p.causal && !apart && heads % 8 == 0;
    if (apart) {
      const int rc = p.bias ? launch(attention_forward_kernel<T, DP, A, true, true>, blocks, A * 64, p, s)
                            : launch(attention_forward_kernel<T, DP, A, true, false>, blocks, A * 64, p, s);
      if (rc != GACT_OK || p.splits == 1) return rc;
      constexpr int kDown = 256 / (DP / 4);
      if (p.splits <= kFewSplits) return launch(attention_join_few_kernel<T, DP>, (heads * rows + kDown - 1) / kDown, 256, p, s);
      return launch(attention_join_kernel<T, DP>, heads * rows, 256, p, s);
    }
    if (waves == 2)
      return p.bias ? launch(attention_forward_kernel<T, DP, 2, false, true>, blocks, 128, p, s)
                    : launch(attention_forward_kernel<T, DP, 2, false, false>, blocks, 128, p, s);
    return p.bias ? launch(attention_forward_kernel<T, DP, 4, false, true>, blocks, 256, p, s)
                  : launch(attention_forward_kernel<T, DP, 4, false, false>, blocks, 256, p, s);
  });
}
template <typename T, int DP>
int add_parts(const PartRows& p, int outputs, hipStream_t s) {
  constexpr int kDown = 256 / (DP / 4);
  const int64_t blocks = (p.rows + kDown - 1) / kDown;
  if (!blocks_fit(blocks)) return GACT_ELIMIT;
  dim3 grid = grid_of(blocks, 256);
  grid.z = outputs;
  hipLaunchKernelGGL((attention_add_kernel<T, DP>), grid, dim3(256), 0, s, p);
  return launch_status();
}
// how a kernel of the backward pass is cut: waves of a workgroup, splits of the other side, keys of a split
struct BackwardCut {
  int waves, splits, per_split;
};
// Heads that share keys pass one after the other: with few workgroups that takes longer than two kernels that split them (4 workgroups of 16 heads of 50
// tokens 86 us, and 18; 256 of 4 heads of 4 tokens 20 and 17; 4096 of 4 heads of 32 tokens 139 and 145)
inline bool sequences_are_short(const AttentionArgs& p, int64_t batch) {
  return p.queries <= 64 && p.keys <= 64 && !p.bias && (p.group == 1 || batch * p.kv_heads >= 512);
}
template <typename T>
int attention_backward(AttentionArgs p, int64_t batch, BackwardCut for_dq, BackwardCut for_dkv, hipStream_t s) {
  return with_width(p.width, [&](auto width) {
    constexpr int DP = decltype(width)::value;
    auto shape = [&](int64_t heads, int64_t rows, const BackwardCut& cut) {
      const int64_t tiles = (rows + cut.waves * 32 - 1) / (cut.waves * 32);
      p.splits = cut.splits;
      p.per_split = cut.per_split;
      p.tiles = (uint32_t)tiles;
      p.blocks = (uint32_t)(heads * tiles * cut.splits);
      p.by_length = p.causal && heads % 8 == 0;
      return heads * tiles * cut.splits;
    };
    if constexpr (kShortFits<T, DP>)
      if (sequences_are_short(p, batch)) return launch(attention_short_kernel<T, DP>, shape(batch * p.kv_heads, 1, BackwardCut{2, 1, 0}), 128, p, s);
    const int64_t blocks = shape(batch * p.heads, p.queries, for_dq);
    int rc;
    if (for_dq.waves == 2)
      rc = p.bias ? launch(attention_dq_kernel<T, DP, 2, true>, blocks, 128, p, s) : launch(attention_dq_kernel<T, DP, 2, false>, blocks, 128, p, s);
    else
      rc = p.bias ? launch(attention_dq_kernel<T, DP, 4, true>, blocks, 256, p, s) : launch(attention_dq_kernel<T, DP, 4, false>, blocks, 256, p, s);
    if (rc == GACT_OK && for_dq.splits > 1 && p.dq.p && blocks > 0) {
      const int padded = (int)p.tiles * for_dq.waves * 32;
      rc = add_parts<T, DP>(PartRows{{p.part, nullptr}, {p.dq, p.dq}, {p.scale, 0.0f}, batch * p.heads * p.queries, p.heads, p.queries, padded, p.splits, p.width}, 1, s);
    }
    if (rc != GACT_OK || !(p.dk.p || p.dv.p)) return rc;
    const int64_t others = shape(batch * p.kv_heads, p.keys, for_dkv);
    if (for_dkv.waves == 2)
      rc = p.bias ? launch(attention_dkv_kernel<T, DP, 2, true>, others, 128, p, s) : launch(attention_dkv_kernel<T, DP, 2, false>, others, 128, p, s);
    else
      rc = p.bias ? launch(attention_dkv_kernel<T, DP, 4, true>, others, 256, p, s) : launch(attention_dkv_kernel<T, DP, 4, false>, others, 256, p, s);
    if (rc != GACT_OK || for_dkv.splits == 1 || others == 0) return rc;
    const int padded = (int)p.tiles * for_dkv.waves * 32;
    const float* const of_v = p.part + (int64_t)p.splits * batch * p.kv_heads * padded * DP;
    PartRows rows{{p.part, of_v}, {p.dk, p.dv}, {p.scale, 1.0f}, batch * p.kv_heads * p.keys, p.kv_heads, p.keys, padded, p.splits, p.width};
    if (!p.dk.p) {      // dv alone
      rows.part[0] = of_v;
      rows.out[0] = p.dv;
      rows.factor[0] = 1.0f;
    }
    return add_parts<T, DP>(rows, p.dk.p && p.dv.p ? 2 : 1, s);
  });
}
