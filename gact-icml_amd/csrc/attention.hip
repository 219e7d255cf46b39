// Attention's host side, its small kernels, and the relative position bias.
#include "attention.h"

#include <math.h>

extern template int attention_forward<float>(AttentionArgs, int64_t, int, bool, hipStream_t);
extern template int attention_forward<f16>(AttentionArgs, int64_t, int, bool, hipStream_t);
extern template int attention_forward<bf16>(AttentionArgs, int64_t, int, bool, hipStream_t);
extern template int attention_backward<float>(AttentionArgs, int64_t, BackwardCut, BackwardCut, hipStream_t);
extern template int attention_backward<f16>(AttentionArgs, int64_t, BackwardCut, BackwardCut, hipStream_t);
extern template int attention_backward<bf16>(AttentionArgs, int64_t, BackwardCut, BackwardCut, hipStream_t);

namespace {

constexpr float kLog2e = 1.44269504f;
// A bias of this or less hides the key, as -inf does: with the lowest value of a type for a whole row the scores would be lost in it
constexpr float kHidden = -1e30f;

// The bias as the kernels add it.  A launch of its own (2 us): in the kernels the product and the comparison would be made for every score
__global__ __launch_bounds__(256) void attention_bias_kernel(const float* __restrict__ bias, int64_t n, float* __restrict__ out) {
  const int64_t i = block_of() * 256 + threadIdx.x;
  if (i >= n) return;
  const float v = bias[i];
  out[i] = v <= kHidden ? -__builtin_inff() : v * kLog2e;
}

// dbias[h][t]: what the blocks of 32 queries of all batch entries have on diagonal t, in their order.  Bound by what the caches give of its one use of every
// float: 8 x 16 heads of 1000 x 1000 (17 MB) 7 us; with the loads one after the other 24.
struct AlongArgs {
  const float* along;
  int64_t stride;
  int64_t batch;
  int heads, queries, keys, tall, rows, waves, splits, per_split;     // queries of a workgroup, rows of a tile, waves
  bool causal;
  float* out;
};
__global__ __launch_bounds__(1024) void attention_along_kernel(AlongArgs p) {
  __shared__ float shared[16][64];
  const int distances = p.queries + p.keys - 1, t = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6, h = blockIdx.y;
  const int blocks = (p.queries + 31) / 32, tiles = (p.queries + p.tall - 1) / p.tall;
  // a wave has every 16th of the blocks of queries and the splits of their keys, for the batch entries in turn, or, where there are fewer than 16, one of
  // them for every few batch entries (492 heads of 54 tokens 8 us, with one wave at work 22); diagonal t is number t + 32 (k + 1) - queries of block k from its first key on
  float sum = 0.0f;
  const int units = blocks * p.splits, shares = units < 16 ? 16 / (units > 0 ? units : 1) : 1;
  for (int n = wave / shares; n < units; n += 16 / shares) {
    const int k = n / p.splits, from_key = n % p.splits * p.per_split, tile = 32 * k / p.tall;
    const int last = tile * p.tall + p.tall - 1 < p.queries ? tile * p.tall + p.tall - 1 : p.queries - 1;
    int to = last + p.keys - p.queries + 1;
    to = !p.causal || to > p.keys ? p.keys : to;
    if (p.splits > 1 && to > from_key + p.per_split) to = from_key + p.per_split;
    const int at = t + 32 * (k + 1) - p.queries - from_key, there = to > from_key ? (to - from_key + p.rows - 1) / p.rows * p.rows : 0;
    if (t >= distances || at < 0 || at >= there + 32) continue;
    const float* from = p.along + (((int64_t)h * tiles * p.waves + k) * p.splits + n % p.splits) * p.stride + at;
    const int64_t entry = (int64_t)p.heads * tiles * p.waves * p.splits * p.stride, apart = shares * entry;
    const int64_t share = wave % shares, entries = (p.batch + shares - 1 - share) / shares;
    from += share * entry;
    int64_t b = 0;
    for (; b + 8 <= entries; b += 8) {      // eight loads on their way at a time
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) v[u] = from[u * apart];
#pragma unroll
      for (int u = 0; u < 8; u++) sum += v[u];
      from += 8 * apart;
    }
    for (; b < entries; b++, from += apart) sum += *from;
  }
  shared[wave][threadIdx.x & 63] = sum;
  __syncthreads();
  if (wave == 0 && t < distances) {
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) sum += shared[w][threadIdx.x];
    p.out[(int64_t)h * distances + t] = sum;
  }
}

// ---- the relative position bias by buckets ----
constexpr int kMostBuckets = GACT_MAX_BUCKETS;
struct Buckets {
  int near, steps, per;       // buckets of one distance each, buckets behind them, and both together: those of one direction
  bool both;
  int32_t border[kMostBuckets];      // the least distance of bucket near + k
  __device__ __forceinline__ int of(int d) const {       // key - query
    const int away = both ? (d < 0 ? -d : d) : d < 0 ? -d : 0, side = both && d > 0 ? per : 0;
    if (away < near) return side + away;
    int low = 0, high = steps;       // border[low] <= away < border[high]
    while (high - low > 1) {
      const int middle = (low + high) / 2;
      (border[middle] <= away ? low : high) = middle;
    }
    return side + near + low;
  }
};
// A thread has a distance and eight heads, whose values lie side by side in the table.  64 heads of 32767 distances (8.4 MB) 5.9 us, 12 of 393 2.8: start and
// end of a launch and the search for the bucket.
template <typename T>
__global__ __launch_bounds__(256) void position_bias_kernel(const T* __restrict__ table, int heads, int keys, int distances, Buckets buckets,
                                                            float* __restrict__ out) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= distances) return;
  const T* const row = table + (int64_t)buckets.of(t - (keys - 1)) * heads;
  const int first = blockIdx.y * 8;
#pragma unroll
  for (int h = 0; h < 8; h++)
    if (first + h < heads) out[(int64_t)(first + h) * distances + t] = (float)row[first + h];
}
// A bucket's distances are neighbours: a workgroup adds up one bucket of one head, always in the same order.  64 heads of 32767 distances 7.7 us, of which
// the largest bucket's workgroups, 65 KB each, are the last; 12 of 393 2.6.
template <typename T>
__global__ __launch_bounds__(256) void position_bias_backward_kernel(const float* __restrict__ grad, int heads, int queries, int keys, Buckets buckets,
                                                                     T* __restrict__ d_table) {
  __shared__ float shared[4];
  const int bucket = blockIdx.x, h = blockIdx.y, side = buckets.both && bucket >= buckets.per, n = bucket - (side ? buckets.per : 0);
  const int distances = queries + keys - 1;
  // distances from `low` to below `high` on this side of the query
  const int low = n < buckets.near ? n : buckets.border[n - buckets.near];
  const int high = n < buckets.near ? n + 1 < buckets.near ? n + 1 : buckets.border[0] : n + 1 < buckets.per ? buckets.border[n + 1 - buckets.near] : 0x40000000;
  int begin = side ? keys - 1 + (low > 1 ? low : 1) : keys - high, end = side ? (high > queries ? distances : keys - 1 + high) : keys - low;
  if (!buckets.both && n == 0) end = distances;       // keys behind the query
  if (begin < 0) begin = 0;
  if (end > distances) end = distances;
  const float* const row = grad + (int64_t)h * distances;
  float sum[4] = {};
  int t = begin + threadIdx.x;
  for (; t + 3 * 256 < end; t += 4 * 256)
#pragma unroll
    for (int u = 0; u < 4; u++) sum[u] += row[t + u * 256];
  for (; t < end; t += 256) sum[0] += row[t];
  const float all = over_lanes<Sum, 64>((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = all;
  __syncthreads();
  if (threadIdx.x == 0) d_table[(int64_t)bucket * heads + h] = rounded<T>((shared[0] + shared[1]) + (shared[2] + shared[3]));
}

// ---- host side ----
constexpr int kComputeUnits = 256;
inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
inline int64_t esz(int dtype) { return dtype == GACT_F32 ? 4 : 2; }

bool sizes_fit(const gact_attention* a) {
  if (!known(a->dtype) || a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return false;
  if (a->queries > GACT_ATTENTION_MAX_LENGTH || a->keys > GACT_ATTENTION_MAX_LENGTH || a->heads > 65535 || a->batch > 0x7fffffff) return false;
  return a->width >= 1 && a->width <= GACT_ATTENTION_MAX_WIDTH && a->scale > 0.0f && a->scale * kLog2e < __builtin_inff();
}
int64_t distances(const gact_attention* a) { return a->queries + a->keys > 0 ? a->queries + a->keys - 1 : 0; }
// whole 16-byte pieces, and rows that the kernels' offsets reach.  GACT_OK where nothing of it is read
int check_rows(const gact_attention* a, const gact_rows* r, int64_t heads, int64_t rows) {
  if (!r) return GACT_EINVAL;
  if (a->batch == 0 || rows == 0) return GACT_OK;
  const int64_t e = esz(a->dtype);
  if (!r->p || r->batch < 0 || r->head < 0 || (rows > 1 && r->row < a->width)) return GACT_EINVAL;
  if (!aligned16(r->p) || a->width * e % 16 || (rows > 1 && r->row * e % 16) || (a->batch > 1 && r->batch * e % 16) || (heads > 1 && r->head * e % 16))
    return GACT_EALIGN;
  return rows > 1 && r->row * e > GACT_ATTENTION_MAX_STRIDE ? GACT_EINVAL : GACT_OK;
}
// (a single row may have any stride)
Side side_of(const gact_attention* a, const gact_rows* r, int64_t rows) {
  const int64_t e = esz(a->dtype);
  return r ? Side{(const char*)r->p, r->batch * e, r->head * e, (rows > 1 ? r->row : a->width) * e} : Side{nullptr, 0, 0, 0};
}
int check_all(const gact_attention* a) {
  if (!a || !sizes_fit(a)) return GACT_EINVAL;
  if ((a->mask && a->mask_stride < 0) || (a->bias && a->heads * distances(a) > ((int64_t)1 << 40))) return GACT_EINVAL;
  int rc = check_rows(a, &a->q, a->heads, a->queries);
  if (rc == GACT_OK) rc = check_rows(a, &a->k, a->kv_heads, a->keys);
  return rc == GACT_OK ? check_rows(a, &a->v, a->kv_heads, a->keys) : rc;
}

// How the forward pass is cut.  Workgroups of two waves for up to 64 queries (24576 heads of 49 floats' tokens 179 us, with four 334; 1024 heads of 40
// tokens 7.2 and 8.5).  Few queries: workgroups of 32 rows whose waves take the keys in turn, and splits of the keys until there is a workgroup to a compute
// unit (32 heads' token on 8 key heads of 65537 keys 47 us, with twice the splits 52, in tiles 1728), each wave with at least two blocks of 32 keys (8 heads'
// token behind 2048 keys 9.2 us, with four blocks 10.6).  The same for more queries where their tiles are fewer than the compute units (4 heads of 4096
// tokens 36 us, in tiles 74; 12 of 2048 33 and 40), but not above (24 of 2048, width 128: 76 us in 384 tiles, 136 so).
struct ForwardCut {
  int waves;
  bool apart;
  int splits, per_split;
};
int waves_of(int64_t rows) { return rows <= 64 ? 2 : 4; }
int64_t padded_width(const gact_attention* a) { return round_up(a->width, 32); }
ForwardCut forward_cut(const gact_attention* a) {
  ForwardCut c{waves_of(a->queries), false, 1, 0};
  const int64_t group = a->heads / a->kv_heads, rows = group * a->queries;
  const int64_t blocks = a->batch * a->heads * ((a->queries + c.waves * 32 - 1) / (c.waves * 32));
  const int64_t units = a->batch * a->kv_heads * ((rows + 31) / 32);
  c.apart = rows <= 32 || (blocks < kComputeUnits && a->keys >= 256);
  if (!c.apart || units == 0) return c;
  c.waves = esz(a->dtype) * padded_width(a) > 256 ? 2 : 4;
  const int64_t least = c.waves * 64;
  int64_t splits = kComputeUnits / units, most = a->keys / least;
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  const int64_t per = round_up((a->keys + splits - 1) / splits, c.waves * 32);
  c.per_split = (int)(per > 0 ? per : c.waves * 32);
  c.splits = (int)(a->keys > 0 ? (a->keys + c.per_split - 1) / c.per_split : 1);
  return c;
}
int64_t bias_bytes(const gact_attention* a) { return a->bias ? round_up(a->heads * distances(a) * 4, 256) : 0; }
int64_t split_rows(const gact_attention* a, const ForwardCut& c) {
  return c.splits > 1 ? a->batch * a->kv_heads * ((a->heads / a->kv_heads * a->queries + 31) / 32) * c.splits * 32 : 0;
}
// rows of a tile in the backward pass, as Tile has them
int tile_rows(const gact_attention* a, int waves) {
  const int64_t wide = padded_width(a) * esz(a->dtype);
  return (wide <= 256 && waves == 4) || wide <= 64 ? 64 : 32;
}
// How the backward pass is cut: where tiles are few, splits of the other side, whose sums are floats that a kernel of its own adds up.  Two workgroups to a
// compute unit where 16 tiles are left to each split (4 heads of 4096 tokens, width 64: 121 us for dq, dk and dv with one, 105 with two; 12 causal heads:
// 249 unsplit, 196), else one with two tiles at least: shorter splits are all sums to write and to add (one head of 4096, width 128: 78 us with splits of
// 8 tiles, 100 with 4; 48 heads of 512 tokens: 36 unsplit, 49 with splits of 4).
int splits_of(int64_t blocks, int64_t steps) {
  if (blocks == 0 || blocks >= 2 * kComputeUnits) return 1;
  const int64_t twice = (2 * kComputeUnits + blocks - 1) / blocks;
  if (steps / twice >= 16) return (int)twice;
  int64_t splits = kComputeUnits / blocks;
  if (splits > steps / 2) splits = steps / 2;
  return splits < 1 ? 1 : (int)splits;
}
BackwardCut dq_cut(const gact_attention* a) {
  BackwardCut c{waves_of(a->queries), 1, 0};
  const int64_t rows = tile_rows(a, c.waves), steps = (a->keys + rows - 1) / rows;
  const int64_t blocks = a->batch * a->heads * ((a->queries + c.waves * 32 - 1) / (c.waves * 32));
  c.splits = splits_of(blocks, steps);
  c.per_split = (int)(((steps + c.splits - 1) / c.splits) * rows);
  if (c.per_split > 0) c.splits = (int)((a->keys + c.per_split - 1) / c.per_split);
  if (c.splits < 1) c.splits = 1;
  return c;
}
BackwardCut dkv_cut(const gact_attention* a) {
  BackwardCut c{waves_of(a->keys), 1, 0};
  const int64_t rows = tile_rows(a, c.waves), steps = (a->queries + rows - 1) / rows * (a->heads / a->kv_heads);
  c.splits = splits_of(a->batch * a->kv_heads * ((a->keys + c.waves * 32 - 1) / (c.waves * 32)), steps);
  return c;
}
int64_t along_stride(const gact_attention* a, const BackwardCut& c) {
  return (c.splits > 1 ? c.per_split : round_up(a->keys, tile_rows(a, c.waves))) + 32;
}
int64_t along_bytes(const gact_attention* a, const BackwardCut& c) {
  return a->batch * a->heads * ((a->queries + c.waves * 32 - 1) / (c.waves * 32)) * c.waves * c.splits * along_stride(a, c) * 4;
}
int64_t part_bytes(const gact_attention* a, const BackwardCut& c, int64_t heads, int64_t rows, int outputs) {
  return c.splits > 1 ? a->batch * heads * round_up(rows, c.waves * 32) * padded_width(a) * 4 * c.splits * outputs : 0;
}
// both kernels' sums have the same place, one after the other
int64_t parts_bytes(const gact_attention* a) {
  const int64_t q = part_bytes(a, dq_cut(a), a->heads, a->queries, 1), k = part_bytes(a, dkv_cut(a), a->kv_heads, a->keys, 2);
  return q > k ? q : k;
}
int64_t delta_bytes(const gact_attention* a) { return round_up(a->batch * a->heads * a->queries * 4, 256); }

AttentionArgs args_of(const gact_attention* a) {
  AttentionArgs p{};
  p.q = side_of(a, &a->q, a->queries);
  p.k = side_of(a, &a->k, a->keys);
  p.v = side_of(a, &a->v, a->keys);
  p.mask = a->mask;
  p.mask_stride = a->mask_stride;
  p.heads = (int)a->heads;
  p.kv_heads = (int)a->kv_heads;
  p.group = (int)(a->heads / a->kv_heads);
  p.queries = (int)a->queries;
  p.keys = (int)a->keys;
  p.width = (int)a->width;
  p.causal = a->causal != 0;
  p.blind = a->bias || a->mask || (p.causal && a->queries > a->keys);
  p.scale = a->scale;
  p.scale2 = a->scale * kLog2e;
  p.splits = 1;
  return p;
}
int prepare_bias(const gact_attention* a, AttentionArgs& p, float* to, hipStream_t s) {
  const int64_t n = a->heads * distances(a);
  if (!a->bias || n == 0) return GACT_OK;
  p.bias = to;
  hipLaunchKernelGGL(attention_bias_kernel, grid_of((n + 255) / 256, 256), dim3(256), 0, s, a->bias, n, to);
  return launch_status();
}

template <typename T>
int with_buckets(const void* table, int64_t buckets, int64_t heads, int64_t queries, int64_t keys, int both, int64_t most, const void* out, T&& f) {
  const int64_t per = both ? buckets / 2 : buckets, near = per / 2;
  if (buckets < 2 || buckets > GACT_MAX_BUCKETS || (both && buckets % 2) || per < 2 || heads < 1 || heads > 65535) return GACT_EINVAL;
  if (queries < 1 || keys < 1 || queries > GACT_ATTENTION_MAX_LENGTH || keys > GACT_ATTENTION_MAX_LENGTH || most <= near || most > GACT_ATTENTION_MAX_LENGTH)
    return GACT_EINVAL;
  if (!table || !out) return GACT_EINVAL;
  Buckets b{};
  b.near = (int)near;
  b.steps = (int)(per - near);
  b.per = (int)per;
  b.both = both != 0;
  // the least whole distance n with (n / near)^steps >= (most / near)^k; where that is an equation of whole numbers the logarithm's rounding must not
  // push it to the next one
  for (int k = 0; k < b.steps; k++) {
    const long double x = (long double)near * powl((long double)most / (long double)near, (long double)k / (long double)b.steps);
    b.border[k] = (int32_t)ceill(x * (1.0L - 1e-13L));
  }
  return f(b);
}

}  // namespace

extern "C" {

int64_t gact_attention_workspace_bytes(const gact_attention* a) {
  if (!a || !sizes_fit(a)) return 0;
  const ForwardCut c = forward_cut(a);
  return bias_bytes(a) + split_rows(a, c) * (padded_width(a) + 2) * 4;
}

int gact_attention_forward(const gact_attention* a, const gact_rows* out, float* lse, int8_t* rest, void* workspace, void* stream) {
  int rc = check_all(a);
  if (rc == GACT_OK) rc = check_rows(a, out, a->heads, a->queries);
  if (rc != GACT_OK) return rc;
  if (a->batch == 0 || a->queries == 0) return GACT_OK;
  if ((uintptr_t)rest % 8) return GACT_EALIGN;
  if (gact_attention_workspace_bytes(a) > 0) {
    if (!workspace) return GACT_EINVAL;
    if (!aligned16(workspace)) return GACT_EALIGN;
  }
  fresh_launch();
  const hipStream_t s = (hipStream_t)stream;
  AttentionArgs p = args_of(a);
  p.out = side_of(a, out, a->queries);
  p.lse = lse;
  p.rest = rest;
  rc = prepare_bias(a, p, (float*)workspace, s);
  if (rc != GACT_OK) return rc;
  const ForwardCut c = forward_cut(a);
  p.splits = c.splits;
  p.per_split = c.per_split;
  p.part = (float*)((char*)workspace + bias_bytes(a));
  p.part_stats = p.part + split_rows(a, c) * padded_width(a);
  return with_type(a->dtype, [&](auto zero) { return attention_forward<decltype(zero)>(p, a->batch, c.waves, c.apart, s); });
}

int64_t gact_attention_backward_workspace_bytes(const gact_attention* a, int dbias) {
  if (!a || !sizes_fit(a)) return 0;
  return bias_bytes(a) + delta_bytes(a) + parts_bytes(a) + (dbias ? along_bytes(a, dq_cut(a)) : 0);
}

int gact_attention_backward(const gact_attention* a, const gact_rows* out, const float* lse, const int8_t* rest, const gact_rows* d_out,
                            const gact_rows* dq, const gact_rows* dk, const gact_rows* dv, float* dbias, void* workspace, void* stream) {
  int rc = check_all(a);
  if (rc == GACT_OK) rc = check_rows(a, out, a->heads, a->queries);
  if (rc == GACT_OK) rc = check_rows(a, d_out, a->heads, a->queries);
  if (rc == GACT_OK && dq) rc = check_rows(a, dq, a->heads, a->queries);
  if (rc == GACT_OK && dk) rc = check_rows(a, dk, a->kv_heads, a->keys);
  if (rc == GACT_OK && dv) rc = check_rows(a, dv, a->kv_heads, a->keys);
  if (rc != GACT_OK) return rc;
  if (dbias && !a->bias) return GACT_EINVAL;
  const bool some = a->batch > 0 && a->queries > 0;
  if (some && !lse) return GACT_EINVAL;
  if ((uintptr_t)rest % 8) return GACT_EALIGN;
  if (gact_attention_backward_workspace_bytes(a, dbias != nullptr) > 0) {
    if (!workspace) return GACT_EINVAL;
    if (!aligned16(workspace)) return GACT_EALIGN;
  }
  fresh_launch();
  const hipStream_t s = (hipStream_t)stream;
  AttentionArgs p = args_of(a);
  p.out = side_of(a, out, a->queries);
  p.d_out = side_of(a, d_out, a->queries);
  p.dq = side_of(a, dq, a->queries);
  p.dk = side_of(a, a->keys > 0 ? dk : nullptr, a->keys);
  p.dv = side_of(a, a->keys > 0 ? dv : nullptr, a->keys);
  p.lse = const_cast<float*>(lse);
  p.rest = const_cast<int8_t*>(rest);
  rc = prepare_bias(a, p, (float*)workspace, s);
  if (rc != GACT_OK) return rc;
  p.delta = (float*)((char*)workspace + bias_bytes(a));
  p.part = (float*)((char*)p.delta + delta_bytes(a));
  const BackwardCut for_dq = dq_cut(a), for_dkv = dkv_cut(a);
  p.along = dbias ? (float*)((char*)p.part + parts_bytes(a)) : nullptr;
  p.along_stride = along_stride(a, for_dq);
  if (a->batch > 0) {
    rc = with_type(a->dtype, [&](auto zero) { return attention_backward<decltype(zero)>(p, a->batch, for_dq, for_dkv, s); });
    if (rc != GACT_OK) return rc;
  }
  if (dbias && distances(a) > 0) {
    const AlongArgs along{p.along, p.along_stride, some ? a->batch : 0, p.heads, p.queries, p.keys, for_dq.waves * 32, tile_rows(a, for_dq.waves), for_dq.waves,
                          for_dq.splits, for_dq.per_split, p.causal, dbias};
    hipLaunchKernelGGL(attention_along_kernel, dim3((unsigned)((distances(a) + 63) / 64), (unsigned)a->heads), dim3(1024), 0, s, along);
    return launch_status();
  }
  return GACT_OK;
}

int gact_position_bias(const void* table, int dtype, int64_t buckets, int64_t heads, int64_t queries, int64_t keys, int both, int64_t max_distance,
                       float* out, void* stream) {
  if (!known(dtype)) return GACT_EINVAL;
  return with_buckets(table, buckets, heads, queries, keys, both, max_distance, out, [&](const Buckets& b) {
    fresh_launch();
    return with_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      const int distances = (int)(queries + keys - 1);
      hipLaunchKernelGGL((position_bias_kernel<T>), dim3((unsigned)((distances + 255) / 256), (unsigned)((heads + 7) / 8)), dim3(256), 0,
                         (hipStream_t)stream, (const T*)table, (int)heads, (int)keys, distances, b, out);
      return launch_status();
    });
  });
}

int gact_position_bias_backward(const float* grad, int dtype, int64_t buckets, int64_t heads, int64_t queries, int64_t keys, int both,
                                int64_t max_distance, void* d_table, void* stream) {
  if (!known(dtype)) return GACT_EINVAL;
  return with_buckets(grad, buckets, heads, queries, keys, both, max_distance, d_table, [&](const Buckets& b) {
    fresh_launch();
    return with_type(dtype, [&](auto zero) {
      using T = decltype(zero);
      hipLaunchKernelGGL((position_bias_backward_kernel<T>), dim3((unsigned)buckets, (unsigned)heads), dim3(256), 0, (hipStream_t)stream, grad,
                         (int)heads, (int)queries, (int)keys, b, (T*)d_table);
      return launch_status();
    });
  });
}

}  // extern "C"
