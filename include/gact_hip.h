/*
 * C ABI of libgact_hip.so: GACT's saved-activation compression path on MI355X (gfx950).
 *
 * Every entry point takes plain device pointers and sizes, launches on the HIP stream it
 * is given (0 = the null stream), allocates no device memory and returns 0 or a negative
 * GACT_E* code (gact_strerror() names it).  The current HIP device must be the one the
 * pointers live on.  Calls are asynchronous; nothing synchronises the stream.
 *
 * "Reference" below is LiuXiaoxuanPKU/GACT-ICML; paths are relative to its root.
 */
#ifndef GACT_HIP_H
#define GACT_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GACT_ABI_VERSION 7

/* element types of activations, min, max and scale */
#define GACT_F32 0
#define GACT_F16 1
/* bfloat16 activations (no counterpart in the reference, which knows float and half).  Taken by
 * gact_quantize, gact_dequantize and the batched launches only.  min and max are bfloat16, the scale is
 * FLOAT32: the codes, the scale and the minimum are those of the float path on the widened values, and
 * dequantize rounds float(code) / scale + min to bfloat16, to nearest even. */
#define GACT_BF16 2

/* where the stochastic-rounding uniform u of each element comes from */
#define GACT_NOISE_CONST 0  /* u = 0.5: deterministic round-to-nearest                          */
#define GACT_NOISE_INJECT 1 /* u read from a float tensor laid out like the (padded) data        */
#define GACT_NOISE_REF 2    /* the reference's stream: one Philox4x32-10 state per output byte,  */
                            /* (seed, subsequence = byte index, offset 0), cuRAND uniform map    */
#define GACT_NOISE_FAST 3   /* one Philox4x32-7 block per 32 elements, 8-bit centred noise (ours)  */

#define GACT_OK 0
#define GACT_EINVAL (-1) /* bad argument (bits not in {1,2,4,8}, negative size, null pointer ...) */
#define GACT_EALIGN (-2) /* a pointer is not aligned as the kernels need (16 bytes)               */
#define GACT_ESHAPE (-3) /* shape not supported by this entry point                               */
#define GACT_ELAUNCH (-4) /* the HIP runtime reported an error at launch                          */
#define GACT_EBUDGET (-5) /* calc_precision: every tensor is at 1 bit and the budget is not met   */
#define GACT_ELIMIT (-6)  /* beyond the size limit of an entry point that brings its own workspace */

const char* gact_strerror(int code);
int gact_abi_version(void);

/* Bytes the pack kernels write for N groups rows of G*D elements: bits*N_round*G*D/8 with N rounded
 * up to a multiple of 8/bits.  The reference allocates one byte more and never writes it
 * (gact/gact/cpp_extension/quantization_cuda_kernel.cu:88-91). */
int64_t gact_packed_bytes(int bits, int64_t N, int64_t G, int64_t D);

/* Per-row minimum and maximum of a contiguous [N, D] tensor; D % 32 == 0 and D > 32.
 * Replaces minimax_cuda (gact/gact/cpp_extension/minimax_cuda_kernel.cu:70-89, bound at
 * minimax.cc:7-14). */
int gact_minimax(const void* data, int dtype, int64_t N, int64_t D, void* mn, void* mx, void* stream);

/* scale = T(2^bits-1)/(max-min+2e-6) for N*G entries, then the packed codes of data[N,G,D].
 * Writes gact_packed_bytes() bytes to `packed` and N*G values to `scale`.
 * Replaces pack_single_precision_cuda (quantization_cuda_kernel.cu:74-146, bound at
 * quantization.cc:51-61).  `noise` is only read in GACT_NOISE_INJECT mode. */
int gact_pack(const void* data, const void* mn, const void* mx, int dtype, int bits, int64_t N, int64_t G,
              int64_t D, int noise_mode, uint64_t seed, const float* noise, void* packed, void* scale,
              void* stream);

/* out[N,G,D] = T(code)/scale + min.  Replaces unpack_single_precision_cuda
 * (quantization_cuda_kernel.cu:180-221, bound at quantization.cc:36-49). */
int gact_unpack(const void* packed, int bits, const void* scale, const void* mn, int dtype, int64_t N,
                int64_t G, int64_t D, void* out, void* stream);

/* The whole of no_scheme_quantize_pack (gact/gact/ops.py:11-32) for group size 256 in one pass over
 * the data: `x` holds `numel` contiguous elements, treated as zero-padded to N = ceil(numel/256)
 * groups; writes min[N], scale[N] (and max[N] when `mx` is not null) and gact_packed_bytes(bits,N,1,256)
 * bytes.  Same results as gact_minimax + gact_pack on the padded tensor.  (GACT_BF16: scale is float32.) */
int gact_quantize(const void* x, int dtype, int64_t numel, int bits, int noise_mode, uint64_t seed,
                  const float* noise, void* packed, void* scale, void* mn, void* mx, void* stream);

/* gact_quantize with a second part of the seed that is read from device memory when the kernel runs: the
 * streams are seeded with seed + *seed_add (seed_add: one uint64 in device memory, 8-byte aligned; null = 0).
 * For launches recorded in a HIP graph, whose host arguments are frozen at capture: the caller rewrites the
 * device word between replays (gact/gact/quantizer.py:119-124 adds the iteration count to every tensor's seed)
 * and every replay draws fresh noise.  No counterpart in the reference. */
int gact_quantize_seeded(const void* x, int dtype, int64_t numel, int bits, int noise_mode, uint64_t seed,
                         const uint64_t* seed_add, const float* noise, void* packed, void* scale, void* mn,
                         void* mx, void* stream);

/* The whole of dequantize_and_unpack + the slice of op_dequantize (gact/gact/ops.py:34-47,61-69) for
 * group size 256: writes exactly `numel` elements. */
int gact_dequantize(const void* packed, int bits, const void* scale, const void* mn, int dtype,
                    int64_t numel, void* out, void* stream);

/* The same two with the group size as an argument: 256 (the entry points above), or 64, 128 and 512 for float and half
 * (config.group_size, gact/gact/conf.py:50) and every noise stream but GACT_NOISE_REF.  Same results as zero-padding to
 * whole groups, gact_minimax and gact_pack / gact_unpack, in one pass over the data; GACT_ESHAPE for any other group size and for
 * GACT_NOISE_REF at a group size other than 256, which take that sequence. */
int gact_quantize_groups(const void* x, int dtype, int64_t numel, int group, int bits, int noise_mode, uint64_t seed,
                         const uint64_t* seed_add, const float* noise, void* packed, void* scale, void* mn, void* mx,
                         void* stream);
int gact_dequantize_groups(const void* packed, int bits, const void* scale, const void* mn, int dtype, int64_t numel, int group,
                           void* out, void* stream);

/* gact_quantize_seeded for a tensor that is not contiguous: `ndim` sizes and strides (in elements), the groups being
 * consecutive elements in index order, as in a contiguous copy of the tensor - which this entry point saves.  Taken: tensors
 * whose innermost runs are contiguous and whole 16-byte pieces (at most three more dimensions once those that lie one inside
 * the other are joined), and tensors whose last but one dimension is the contiguous one (channels-last activations,
 * transposed matrices; at most one more dimension), both with 16-byte aligned base and strides; streams GACT_NOISE_CONST and
 * GACT_NOISE_FAST.  Anything else, and layouts of the second kind of which a contiguous copy is the faster way (one or a few
 * of the strided dimension's elements per channel; channels far longer than what a workgroup holds): GACT_ESHAPE and no
 * launch - make a contiguous copy.  No counterpart in the reference, whose reshape copies (gact/gact/ops.py:12-19). */
int gact_quantize_strided(const void* x, int dtype, int ndim, const int64_t* sizes, const int64_t* strides, int bits, int noise_mode,
                          uint64_t seed, const uint64_t* seed_add, void* packed, void* scale, void* mn, void* mx, void* stream);

/* What a gact_quantize (kind 0; fast, deterministic or injected noise) or gact_dequantize (kind 1) launch of a tensor of
 * N groups is made of, without launching anything: the threads of a workgroup, the dynamic LDS the launch asks for -
 * on large tensors some kernels ask for LDS they never touch, which is how the library caps their occupancy - and
 * the workgroups of that kernel a compute unit holds under both (hipOccupancyMaxActiveBlocksPerMultiprocessor).
 * Any of the three pointers may be null.  No counterpart in the reference; for tests and tuning. */
int gact_launch_geometry(int kind, int dtype, int bits, int64_t N, int* threads, int* lds_bytes,
                         int* workgroups_per_cu);

/* Dropout-mask bit packing: n bytes (nonzero = 1) <-> ceil(n/32) int32 words.
 * Replace act_quantize_dropout_mask_cuda / act_dequantize_dropout_mask_cuda
 * (quantization_cuda_kernel.cu:254-303, bound at quantization.cc:26-33). */
int gact_mask_pack(const uint8_t* data, int64_t n, int32_t* mask, void* stream);
int gact_mask_unpack(const int32_t* mask, int64_t n, uint8_t* out, void* stream);

/* Greedy bit allocation on host memory; mutates b.  Replaces calc_precision
 * (gact/gact/cpp_extension/calc_precision.cc:66-118, bound at :120-123). */
int gact_calc_precision(int32_t* b, const float* C, const int64_t* w, int64_t L, double target);

/* The same allocation computed on the GPU from device arrays (b is updated in place), so that the
 * sensitivities never leave the device.  `status` (device int32, may be null) receives 0 or GACT_EBUDGET.
 * No counterpart in the reference, which runs calc_precision on the host. */
int gact_calc_precision_device(int32_t* b, const float* C, const int64_t* w, int64_t L, double target,
                               int32_t* status, void* stream);

/* One saved tensor of a batched launch.  The table itself lives in device memory. */
typedef struct gact_batch_entry {
  const void* x;      /* activation (quantize input / dequantize output), numel elements          */
  int64_t numel;
  int32_t dtype;      /* GACT_F32 / GACT_F16 / GACT_BF16                                           */
  int32_t reserved;
  uint64_t seed;      /* per-tensor seed: seeds[tid] + seed_iter (gact/gact/quantizer.py:119-124)  */
  int64_t first_block; /* exclusive prefix sum of ceil(N/128) over the table (128 groups per block) */
  int64_t packed_offset; /* byte offset of this tensor's codes in the packed arena (written by     */
                         /* gact_batch_plan from the device-resident bits)                          */
  int64_t stats_offset;  /* element offset of this tensor's scale/min rows in the stats arenas      */
} gact_batch_entry;

/* Bytes of device workspace gact_batch_plan fills for a table of L tensors whose grid has total_blocks
 * blocks (the sum of ceil(N_i/128): a block is 128 groups whatever the width).  16-byte aligned memory.
 * The batched entry points take L <= 2^30 and total_blocks < 2^29 (GACT_EINVAL beyond). */
int64_t gact_batch_workspace_bytes(int64_t L, int64_t total_blocks);

/* Plan a batched launch from device-resident bits: fills packed_offset of every table entry (256-byte
 * aligned, in table order) and the workspace - a header of 32 int64 ([0] the arena bytes the table needs,
 * [1] 1 when every bits[i] is in {1,2,4,8}, every dtype is known and [0] <= capacity, else 0: the batched
 * kernels then do nothing, [2..5] the number of tensors at width 1, 2, 4, 8) and the tensor of every block.
 * One small launch; nothing is read back.  No counterpart in the reference. */
int gact_batch_plan(gact_batch_entry* table, const int32_t* bits, int64_t L, int64_t total_blocks,
                    int64_t capacity, void* workspace, void* stream);

/* gact_batch_plan for up to GACT_BATCH_ARGS tensors whose addresses and seeds lie on the host (x[L], seeds[L]) and go to the GPU in the
 * launch's own arguments: writes all of `table` - `geometry`, a table in device memory of which x, seed and packed_offset are not
 * looked at, completed by them and by the offsets - and, where they are not null, a copy of the widths to `kept` and header words
 * [0] and [1] to `verdict` (two int64, device memory or pinned host memory, 8-byte aligned), each written through as soon as it is
 * known: a host that has put -1 there before the call may look for the change.  GACT_ELIMIT beyond GACT_BATCH_ARGS tensors. */
#define GACT_BATCH_ARGS 192
int gact_batch_plan_args(const gact_batch_entry* geometry, const void* const* x, const uint64_t* seeds, gact_batch_entry* table,
                         const int32_t* bits, int32_t* kept, int64_t L, int64_t total_blocks, int64_t capacity, void* workspace,
                         int64_t* verdict, void* stream);

/* Quantize / dequantize all L tensors of the table, each at its own bits[i] read from device memory: one
 * launch over the grid of blocks per element type (quantize) or for all of them (dequantize), the width of
 * a block's tensor selecting the code path.  Scale and min of tensor i
 * are written at byte offset 4*stats_offset of their arenas (keep stats_offset a multiple of 8 so that
 * the rows stay 32-byte aligned).  Results equal a loop of
 * gact_quantize / gact_dequantize over the tensors (gact/gact/quantizer.py:95-142 drives the reference
 * one tensor at a time).  `workspace` is what gact_batch_plan filled for the same table, bits, L and
 * total_blocks.  `dtypes` says which element types
 * occur in the table, which the host that built it knows: bit 0 float, bit 1 half, bit 2 bfloat16 (GACT_DTYPES_*); quantize
 * launches only the kernels of those types, so a tensor whose type is missing from the mask is left unquantized. */
#define GACT_DTYPES_F32 1
#define GACT_DTYPES_F16 2
#define GACT_DTYPES_BF16 4
#define GACT_DTYPES_ALL 7
int gact_quantize_batched(const gact_batch_entry* table, const int32_t* bits, int64_t L, int64_t total_blocks,
                          int noise_mode, int dtypes, const void* workspace, void* packed_arena,
                          void* scale_arena, void* min_arena, void* stream);
int gact_dequantize_batched(const gact_batch_entry* table, const int32_t* bits, int64_t L,
                            int64_t total_blocks, const void* workspace, const void* packed_arena,
                            const void* scale_arena, const void* min_arena, void* stream);

/* gact_dequantize_batched where the host knows which element types the table holds (the same mask; 0 or GACT_DTYPES_ALL: any): the
 * launch is shaped for them, the results are the same. */
int gact_dequantize_batched_types(const gact_batch_entry* table, const int32_t* bits, int64_t L, int64_t total_blocks, int dtypes,
                                  const void* workspace, const void* packed_arena, const void* scale_arena, const void* min_arena,
                                  void* stream);

/* The same for up to GACT_BATCH_ARGS tensors into x[L] (host array of device addresses, 16-byte aligned), with the table and the workspace
 * of the batch's quantize call: no plan of its own.  A width written over since then is looked at: a tensor whose codes would end past
 * the plan's bytes is left out.  GACT_ELIMIT beyond GACT_BATCH_ARGS tensors. */
int gact_dequantize_batched_to(const gact_batch_entry* table, void* const* x, const int32_t* bits, int64_t L, int64_t total_blocks, int dtypes,
                               const void* workspace, const void* packed_arena, const void* scale_arena, const void* min_arena,
                               void* stream);

/* gact_batch_plan followed by gact_quantize_batched, with the workspace in a device array that is part of
 * the library (1 MB per GPU the library runs on, held until the process ends) instead of memory the
 * caller brings: nothing is allocated, by the library or on its behalf.  No counterpart in the reference; it
 * is for callers that cannot allocate - code under HIP graph capture, tight serving loops, harnesses that
 * forbid it.  Same results as the two calls it stands for (packed_offset of every table entry is filled, the
 * arenas are written).  The plan's verdict lives in the library's array, out of the caller's reach, so the plan
 * also writes it to `verdict` (two int64 in device memory, 8-byte aligned; may be null): [0] the arena bytes the
 * table needs, [1] 1 when the launch went ahead, 0 when it was void (a width outside {1,2,4,8}, an unknown
 * element type, or [0] > capacity: the arenas are then left untouched).  Read it whenever the caller may
 * synchronise.  Limit: total_blocks <= 262144 (33.5 M groups, 8.6 G elements),
 * GACT_ELIMIT beyond.  All calls on one GPU share the array: calls that overlap on one GPU (two streams, two
 * threads) race, the caller serialises them.  The first call on a GPU looks the array's address up; make it
 * outside a stream capture.  Dequantize with gact_batch_plan + gact_dequantize_batched as usual. */
int gact_quantize_batched_static(gact_batch_entry* table, const int32_t* bits, int64_t L, int64_t total_blocks,
                                 int64_t capacity, int noise_mode, int dtypes, void* packed_arena,
                                 void* scale_arena, void* min_arena, int64_t* verdict, void* stream);

/* ---- Layers that train on 8-bit checkpoints.  No counterpart in the reference, whose layers save whole tensors through the hooks. ----
 *
 * A checkpoint of a matrix [rows, cols] of any element type: codes (one byte each, rows `ldc` bytes apart, ldc a multiple of 16
 * and at least cols, 16-byte aligned), and a float scale and minimum per row and group of 256 columns, [rows, ceil(cols/256)], the last
 * group of a row being shorter.  Codes, scale and minimum are those of gact_quantize of the values widened to float at 8 bit with
 * GACT_NOISE_CONST (equal to it where 256 divides cols); a code stands for code / scale + min.  As there, a NaN is passed over by minimum and
 * maximum and gets code 0, which stands for the minimum; a group of NaN alone, or of a range that no float holds (an infinity's), stands for NaN.
 * `ld...` are elements from one row to the next.  Rows up to GACT_LAYER_MAX_ROWS, columns up to GACT_LAYER_MAX_COLS. */
#define GACT_LAYER_MAX_ROWS 0x40000000
#define GACT_LAYER_MAX_COLS 262144
#define GACT_NORM_MAX_COLS 16384
#define GACT_LINEAR_FEW_ROWS 64
#define GACT_ACT_NONE 0
#define GACT_ACT_GELU 1      /* z Phi(z)                                            */
#define GACT_ACT_GELU_TANH 2 /* 0.5 z (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3)))     */
#define GACT_ACT_SILU 3      /* z / (1 + exp(-z))                                    */

/* x [rows, cols] -> its checkpoint, and back to values of `dtype` in a contiguous [rows, cols] (16-byte aligned). */
int gact_checkpoint(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* codes, int64_t ldc, float* scale, float* mn,
                    void* stream);
int gact_restore(const void* codes, int64_t ldc, const float* scale, const float* mn, int dtype, int64_t rows, int64_t cols, void* out,
                 void* stream);

/* x [rows, cols] copied to rows `ldo` apart (a multiple of 8, 16-byte aligned), columns behind the last one zero: what the products below
 * take of matrices whose rows are no whole 16-byte pieces. */
int gact_pad_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* out, int64_t ldo, void* stream);

/* Layer norm over the last dimension, cols <= GACT_NORM_MAX_COLS: y = (x - mean) / sqrt(var + eps) weight + bias (either may be null),
 * y contiguous.  With `codes`: also the checkpoint of x, and mean and 1 / sqrt(var + eps) of each row in stats [rows, 2]. */
int gact_norm_forward(const void* x, int64_t ldx, const void* weight, const void* bias, int dtype, int64_t rows, int64_t cols, float eps,
                      void* y, void* codes, int64_t ldc, float* scale, float* mn, float* stats, void* stream);
/* Its backward pass from the checkpoint: dx (contiguous), and dweight and dbias where they are not null, which need `workspace`
 * (gact_norm_workspace_bytes(), float aligned).  rows > 0. */
int64_t gact_norm_workspace_bytes(int64_t rows, int64_t cols);
int gact_norm_backward(const void* dy, int64_t lddy, const void* weight, const void* codes, int64_t ldc, const float* scale,
                       const float* mn, const float* stats, int dtype, int64_t rows, int64_t cols, void* dx, void* dweight, void* dbias,
                       float* workspace, void* stream);

/* y [rows, outer] = act(x [rows, inner] weight [outer, inner]^T + bias) + residual, y contiguous; bias and residual may be null.  With
 * `codes` (and an activation): also the checkpoint of z = x weight^T + bias.  x and weight: 16-byte aligned rows of whole 16-byte pieces (else
 * GACT_EALIGN), except for up to GACT_LINEAR_FEW_ROWS rows.  workspace: gact_linear_workspace_bytes() of the same sizes (codes: whether they
 * are asked for), 16-byte aligned; may be null where that is 0. */
int64_t gact_linear_workspace_bytes(int dtype, int64_t rows, int64_t inner, int64_t outer, int codes);
int gact_linear(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr,
                int activation, int dtype, int64_t rows, int64_t inner, int64_t outer, void* y, void* codes, int64_t ldc, float* scale,
                float* mn, void* workspace, void* stream);

/* dz [rows, cols] = dy act'(z) with z from its checkpoint (codes null and activation GACT_ACT_NONE: dz = dy), rows lddz apart (cols rounded up to a
 * multiple of 8, the columns behind the last one zero); dbias [cols] = the column sums of dz before rounding, through `workspace`
 * (gact_activation_workspace_bytes()).  Either output may be null.  rows > 0. */
int64_t gact_activation_workspace_bytes(int64_t rows, int64_t cols);
int gact_activation_backward(const void* dy, int64_t lddy, const void* codes, int64_t ldc, const float* scale, const float* mn,
                             int activation, int dtype, int64_t rows, int64_t cols, void* dz, int64_t lddz, void* dbias, float* workspace,
                             void* stream);

/* out [rows, cols] = a [rows, depth] b [depth, cols], and out [outer, inner] = grad [rows, outer]^T times the values, rounded to `dtype`, of a
 * checkpoint [rows, inner] (rows > 0); out contiguous.  Operands: 16-byte aligned rows of whole 16-byte pieces, `ld` leaving room for the
 * last one, and rows (of codes, too) at most 4 GACT_LAYER_MAX_COLS apart; what lies behind the last column of `a` up to its piece's end must be
 * zero.  workspace: gact_product_workspace_bytes() of (rows, cols, depth), or (outer, inner, rows); 16-byte aligned. */
int64_t gact_product_workspace_bytes(int dtype, int64_t rows, int64_t cols, int64_t depth);
int gact_product(const void* a, int64_t lda, const void* b, int64_t ldb, int dtype, int64_t rows, int64_t depth, int64_t cols, void* out,
                 void* workspace, void* stream);
int gact_checkpoint_product(const void* grad, int64_t ldg, const void* codes, int64_t ldc, const float* scale, const float* mn, int dtype,
                            int64_t rows, int64_t outer, int64_t inner, void* out, void* workspace, void* stream);

/* ---- Attention.  No counterpart in the reference. ----
 *
 * s_ij = scale q_i.k_j + bias[j - i + queries - 1], out_i = sum over j of softmax(s_i)_j v_j, for every batch entry and head; head h reads key head
 * h / (heads / kv_heads).  A key is hidden from a query where its mask byte is 0, where `causal` is set and j > i + keys - queries, and where the
 * bias is -1e30 or less; a query that sees nothing gets zeros, and its gradient, whatever it is, is nobody's.  What absent keys (mask byte 0) and
 * values hold does not matter; a NaN or infinity of a key that is hidden in another way may show.
 *
 * Rows: [batch, heads, rows, width] of `dtype`, elements from one batch entry, head and row to the next; a row's values lie side by side, in whole
 * 16-byte pieces, rows at least a row and at most GACT_ATTENTION_MAX_STRIDE bytes apart (GACT_EALIGN for addresses, widths and strides that are no
 * multiples of 16 bytes).  batch, queries and keys may be 0. */
#define GACT_ATTENTION_MAX_LENGTH 0x1000000
#define GACT_ATTENTION_MAX_WIDTH 128
#define GACT_ATTENTION_MAX_STRIDE 0x1000000
typedef struct gact_rows {
  const void* p;
  int64_t batch, head, row;
} gact_rows;
typedef struct gact_attention {
  int32_t dtype, causal;
  int64_t batch, heads, kv_heads, queries, keys, width;
  float scale;          /* above 0; times log2(e) a float */
  float reserved;
  const float* bias;    /* [heads, queries + keys - 1], may be null */
  const uint8_t* mask;  /* [batch, keys], rows mask_stride bytes apart; may be null */
  int64_t mask_stride;
  gact_rows q, k, v;
} gact_attention;
/* lse [batch, heads, queries], which the backward pass reads (the logarithm of base 2 of each query's sum; infinite where it sees nothing), and rest
 * [batch, queries, heads, width], 8-byte aligned, what rounding the result to 16 bits has left out of it, in eight bits each: either may be null, and rest is
 * not written for GACT_F32.  workspace: gact_attention_workspace_bytes(), 16-byte aligned; may be null where that is 0. */
int64_t gact_attention_workspace_bytes(const gact_attention* a);
int gact_attention_forward(const gact_attention* a, const gact_rows* out, float* lse, int8_t* rest, void* workspace, void* stream);
/* Recomputes the probabilities from q, k and lse; without rest (null) the result counts as it was rounded.  dq, dk, dv and dbias ([heads, queries + keys - 1]) may each be null.  Sums are made in one order:
 * results are repeatable. */
int64_t gact_attention_backward_workspace_bytes(const gact_attention* a, int dbias);
int gact_attention_backward(const gact_attention* a, const gact_rows* out, const float* lse, const int8_t* rest, const gact_rows* d_out,
                            const gact_rows* dq, const gact_rows* dk, const gact_rows* dv, float* dbias, void* workspace, void* stream);

/* A bias for each head and distance d = key - query, at d + keys - 1 of [heads, queries + keys - 1], out of table [buckets, heads]; and the table's
 * gradient.  `both`: half of the buckets for d > 0, half for the others; else all for d < 0, and those above in bucket 0.  Of one direction's buckets the
 * first half has one distance each, bucket k behind them begins where (|d| / half)^(steps) >= (max_distance / half)^k, and the last one has no end.
 * 2 to GACT_MAX_BUCKETS buckets, two at least to a direction; max_distance above half of a direction's. */
#define GACT_MAX_BUCKETS 512
int gact_position_bias(const void* table, int dtype, int64_t buckets, int64_t heads, int64_t queries, int64_t keys, int both, int64_t max_distance,
                       float* out, void* stream);
int gact_position_bias_backward(const float* grad, int dtype, int64_t buckets, int64_t heads, int64_t queries, int64_t keys, int both,
                                int64_t max_distance, void* d_table, void* stream);

/* ---- AdamW over many tensors.  No counterpart in the reference. ----
 *
 * m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g^2, p = p (1 - lr decay) - lr / (1 - beta1^step) m / (sqrt(v / (1 - beta2^step)) + eps), in
 * floats; g and p of `dtype`, the betas and 1 - beta rounded to float.  bits 32: m and v are floats.  bits 8: m int8 and v uint8 codes of groups of
 * 256 elements, the last one shorter, and scale [groups, 2] the largest |m| and v of each; a code c of m stands for c |c| (scale / 127^2), one of v
 * for c^4 (scale / 255^4), with the quotients and c^4 rounded to float (255^4 to 4228250624).  A value x of m gets the code nearest to the
 * root of |x| (127^2 / scale), one of v the nearest to its fourth root, and no v above 0 the code 0; a group whose largest |m| is below 1e-30
 * has scale and codes 0, one whose largest v is above 0 and below 1e-28 the scale 1e-28.  A group with an infinity or NaN is not finite afterwards.
 * p and g: any address that their type may have; m, v and scale 16-byte aligned.  Tensors must not overlap. */
typedef struct gact_adamw_tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* scale;
  int64_t numel;
} gact_adamw_tensor;
typedef struct gact_adamw_options {
  double lr, beta1, beta2, eps, decay;
  int64_t step;              /* from 1 on */
  const float* lr_at;        /* device memory: the kernel reads lr, and step, there where these are not null */
  const int64_t* step_at;
} gact_adamw_options;
int gact_adamw(const gact_adamw_tensor* tensors, int64_t count, int dtype, int bits, const gact_adamw_options* options, void* stream);
/* What the codes of `count` states stand for, one after the other, into m and v (either may be null); p, g unused. */
int gact_adamw_values(const gact_adamw_tensor* tensors, int64_t count, float* m, float* v, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GACT_HIP_H */
