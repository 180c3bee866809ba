/* nsfps -- MI355X-native farthest point sampling (NS-FPS semantics).
 *
 * C ABI of the drop-in boundary.  Plain pointers and sizes only; every entry
 * point returns an nsfps_status and, on failure, leaves a message readable with
 * nsfps_last_error() (thread-local).  The library never falls back to a CPU
 * path: without a usable HIP device, compute entry points fail with
 * NSFPS_EDEVICE.
 *
 * Reference interfaces replaced (paths relative to the reference tree):
 *   nsfps_range_derive   SpaceRange derived fields + make_range()
 *                        (src/yuezu_fps.h:56-83, src/yuezu_fps.cpp:7-161)
 *   nsfps_bbox           compute_bbox()          (src/yuezu_fps.cpp:643-670)
 *   nsfps_fps            yuezu_fps() behind fps_numpy()
 *                        (src/yuezu_fps.h:211-212, src/yuezu_fps.cpp:676-730,
 *                         yuezu_fps/yuezu_fps_pybind.cpp:67-86)
 *   nsfps_fps_bbox       fps_with_bbox()  (yuezu_fps/yuezu_fps_pybind.cpp:88-101)
 *   nsfps_fps_batched    no single counterpart: B independent yuezu_fps() calls
 *                        (the batched set-abstraction use of fps_numpy)
 *   nsfps_fps_device     yuezu_fps() on device-resident input (cf. the
 *                        reference GPU driver's FpsGPU::sample,
 *                        eval/src_gpu/yuezu_fps_gpu.h:90-126)
 *   nsfps_plan_create / _sample / _destroy
 *                        the reference GPU driver's FpsGPU::initialize /
 *                        sample and its teardown (eval/src_gpu/yuezu_fps_gpu.h:
 *                        90-126): build once, sample many times
 *   nsfps_gather_points, nsfps_ball_query (and _device)
 *                        no counterpart: the grouping step the reference's
 *                        callers run on its output (see their declarations)
 *   nsfps_embed_*, nsfps_conv_*, nsfps_scan_*
 *                        no counterpart: sequence operators over the samples
 *                        (see "Sequence operators")
 *   nsfps_fps_device_noalloc
 *                        no counterpart: nsfps_fps_device for callers that
 *                        cannot allocate device memory (see its declaration)
 */
#ifndef NSFPS_H
#define NSFPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  NSFPS_OK = 0,
  NSFPS_EINVAL = 1,      /* invalid argument (shape, range, non-finite input) */
  NSFPS_EDEVICE = 2,     /* HIP runtime / device failure, or no device */
  NSFPS_ENOMEM = 3,      /* device allocation failed */
  NSFPS_EUNSUPPORTED = 4 /* valid input outside what this build handles: more than
                            1024 blocks on an axis (cells are packed 10 bits per
                            axis), more than 2^31-1 points or samples, a cloud
                            needing more than 4096 level-1 nodes when the tree
                            engine is asked for (NSFPS_ENGINE=tree; the default
                            engine has no such limit), or a layout beyond the
                            allocation-free entry point's array, or a sequence
                            operator's size beyond its limits */
} nsfps_status;

/* The nine primary SpaceRange fields (src/yuezu_fps.h:56-60).  Derived fields
 * are always recomputed from these, so a range edited field by field can never
 * carry stale derived values. */
typedef struct {
  float min_x, max_x;
  float min_y, max_y;
  float min_z, max_z;
  uint32_t x_blocks, y_blocks, z_blocks;
} nsfps_range;

/* Number of cube half-width thresholds per axis in nsfps_range_info. */
#define NSFPS_CUBE_THRESHOLDS 8

/* Derived SpaceRange values (src/yuezu_fps.cpp:7-40, 136-161). */
typedef struct {
  float inv_bs[3];     /* 1.0f / ((max - min) / (float)blocks) */
  float block_size[3]; /* (max - min) / blocks */
  uint32_t bits[3];    /* ceil(log2(blocks)), at least 1 */
  uint32_t total_bits;
  uint64_t total_blocks;
  /* cube_thr[a][k]: the smallest squared distance D >= 0 whose cube
   * half-width on axis a, min((int)ceilf(sqrtf(D) / block_size[a]),
   * blocks - 1) (get_morton_codes_in_range, src/yuezu_fps.cpp:564-570, cells
   * beyond the grid being clipped), is at least k + 1; INFINITY when it never
   * is.  The half-width is monotone in D, so it equals the number of
   * thresholds <= D below the last one. */
  float cube_thr[3][NSFPS_CUBE_THRESHOLDS];
} nsfps_range_info;

/* Per-call measurements of the last compute call on this thread. */
typedef struct {
  double build_ms;   /* device time: cell keys, sorts, leaves (hipEvents) */
  double sample_ms;  /* device time: the sampling loop (hipEvents) */
  double wide_ms;    /* part of sample_ms spent in grid-wide iterations */
  double late_ms;    /* the single-workgroup loop kernel alone, or all rounds of runs */
  double device_ms;  /* build_ms + sample_ms */
  double e2e_ms;     /* host wall time of the whole call incl. copies */
  uint64_t n_points;
  uint64_t n_clouds;
  uint64_t n_leaves;
  uint64_t wide_iters;  /* iterations run by the grid-wide kernel */
  uint64_t samples;     /* samples produced (sum over clouds) */
  uint32_t padded;      /* 1 when the single cloud used the padded cell layout */
  uint32_t lds_bytes;   /* dynamic LDS of the single-workgroup loop */
  uint64_t rounds;      /* sampling rounds of the runs engine (max over clouds; 0 for the tree loop) */
  uint32_t engine;      /* 1: runs (rounds), 0: grid-wide steps + tree loop */
  uint32_t update_split; /* workgroups per level-1 node of the runs engine's update pass
                           (1, or 4 when the call has few level-1 nodes) */
  uint32_t mixed;       /* 1 when leaves were runs of 64 slots that may hold several buckets */
  uint32_t hot_set;     /* density class of the clouds: 128 when every one fills at least 6,912
                           buckets and no cells share buckets, else 64; always 64 where one
                           workgroup sampled each cloud, which counts no buckets, and 0 for the
                           tree loop.  Earlier versions' hot sets had that many copies; no
                           kernel depends on it now */
} nsfps_stats;

/* Library constants mirrored from src/yuezu_fps.h:19-50. */
#define NSFPS_DEFAULT_X_BLOCKS 16
#define NSFPS_DEFAULT_Y_BLOCKS 16
#define NSFPS_DEFAULT_Z_BLOCKS 16
#define NSFPS_MORTON_BLOCK_SIZE 16
#define NSFPS_CACHE_BLOCK_SIZE 16

const char *nsfps_last_error(void);
const char *nsfps_version(void);

/* Number of visible HIP devices (0 when none); never fails. */
int nsfps_device_count(void);

/* Prepares the current device for the library's calls: loads its kernels
 * (the runtime loads code on a kernel's first use), creates the stream and
 * events the host-buffer calls use, and makes one copy each way through a
 * pinned buffer (the runtime sets its copy path up on first use).  No
 * counterpart in the reference (a CPU library).  Optional: the first call on
 * a device does the same; calling this first keeps that one-time work (tens
 * of milliseconds, most of it the runtime's own start) out of the first
 * call.  NSFPS_EDEVICE when no device is visible.  The sequence operators'
 * kernels are loaded by nsfps_init_sequence_device. */
nsfps_status nsfps_init_device(void);

/* Derived fields and Morton LUTs of a range.  luts receives the x, y and z
 * LUTs back to back (2^bits[0] + 2^bits[1] + 2^bits[2] entries) when non-NULL
 * and lut_cap is large enough.  Replaces make_range()/make_uniform_range()'s
 * derivation (src/yuezu_fps.cpp:98-161). */
nsfps_status nsfps_range_derive(const nsfps_range *range, nsfps_range_info *info,
                                uint32_t *luts, uint64_t lut_cap);

/* compute_bbox(): exact fp32 bounds -/+ 1e-6 and the given block counts
 * (src/yuezu_fps.cpp:648-670).  n == 0 gives [0,1]^3 with 1x1x1 blocks. */
nsfps_status nsfps_bbox(const float *xyz, uint64_t n, uint32_t x_blocks,
                        uint32_t y_blocks, uint32_t z_blocks, nsfps_range *out);

/* compute_bbox of device-resident points (d_xyz, n x 3 float32) on the
 * device: the same bounds as nsfps_bbox over the finite points (minimum and
 * maximum do not depend on the order; +-0 differ only before the -/+ 1e-6),
 * and, when info is non-NULL, the range's derived fields as the sampling
 * calls derive them on the device (nsfps_range_derive gives the same bits on
 * the host).  This is the range nsfps_fps, nsfps_fps_bbox and the batched
 * calls use when they are given none.  stream: a hipStream_t (NULL = default
 * stream); the call returns after the stream work completes. */
nsfps_status nsfps_bbox_device(const float *d_xyz, uint64_t n, uint32_t x_blocks,
                               uint32_t y_blocks, uint32_t z_blocks, nsfps_range *out,
                               nsfps_range_info *info, void *stream);

/* FPS of one cloud.  xyz: host pointer, n x 3 float32, C order.  range == NULL
 * selects compute_bbox with the default 16^3 blocks.  out: host buffer of at
 * least n_samples int32 entries; *out_len receives the sample count (smaller
 * than n_samples when the maximum min-distance reaches 0).  Start index 0,
 * n_samples >= n returns 0..n-1, n == 0 or n_samples == 0 returns nothing. */
nsfps_status nsfps_fps(const float *xyz, uint64_t n, uint64_t n_samples,
                       const nsfps_range *range, int32_t *out, uint64_t *out_len);

/* fps_with_bbox(): compute_bbox with the given block counts, then FPS. */
nsfps_status nsfps_fps_bbox(const float *xyz, uint64_t n, uint64_t n_samples,
                            uint32_t x_blocks, uint32_t y_blocks,
                            uint32_t z_blocks, int32_t *out, uint64_t *out_len);

/* B independent clouds of n points each (xyz: B x n x 3, host).  ranges: B
 * ranges, or NULL for a per-cloud compute_bbox with blocks3 (NULL -> 16^3),
 * found on the device.  out: B x n_samples int32 (row b holds cloud b's
 * samples; entries past out_lens[b] are unspecified); out_lens: B.  The
 * reference samples one cloud per call (yuezu_fps, src/yuezu_fps.cpp:676-730,
 * with compute_bbox for range=None, yuezu_fps/yuezu_fps_pybind.cpp:74-76);
 * this is B such calls in one. */
nsfps_status nsfps_fps_batched(const float *xyz, uint64_t batch, uint64_t n,
                               uint64_t n_samples, const nsfps_range *ranges,
                               const uint32_t *blocks3, int32_t *out,
                               uint64_t *out_lens);

/* nsfps_fps_batched on device memory: d_xyz (B x n x 3 float32) and d_out
 * (B x n_samples int32, row b holding cloud b's samples) are device
 * pointers; ranges, blocks3 and out_lens are host memory as in
 * nsfps_fps_batched.  stream is a hipStream_t (NULL = default stream); the
 * call returns after the stream work completes. */
nsfps_status nsfps_fps_batched_device(const float *d_xyz, uint64_t batch, uint64_t n,
                                      uint64_t n_samples, const nsfps_range *ranges,
                                      const uint32_t *blocks3, int32_t *d_out,
                                      uint64_t *out_lens, void *stream);

/* FPS of one cloud whose points already live in device memory (d_xyz, n x 3
 * float32) writing device memory (d_out, n_samples int32).  stream is a
 * hipStream_t (NULL = default stream); the call returns after the stream work
 * completes.  range must be non-NULL. */
nsfps_status nsfps_fps_device(const float *d_xyz, uint64_t n, uint64_t n_samples,
                              const nsfps_range *range, int32_t *d_out,
                              uint64_t *out_len, void *stream);

/* nsfps_fps_device without any device allocation.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (tight
 * serving loops, harnesses that forbid hipMalloc).  The call's whole
 * workspace (cell keys, sorts, slots, leaves, tree and sampling state) lives
 * in a static device array of nsfps_noalloc_scratch_bytes() bytes (64 MiB)
 * per device, reserved on every device by the library's code object in each
 * process that loads the library, whether or not this call is used, and
 * held until the process ends.  A cloud whose layout needs more fails with
 * NSFPS_EUNSUPPORTED and a message giving both sizes: for samples of a
 * sixteenth the limits are 451,444 points on a 32^3 grid, 460,480 on 16^3 and
 * 430,720 on 64x64x16; for nearly all points 439,456, 448,540 and 419,312.
 * Same arguments, samples and guards as nsfps_fps_device; no hipMalloc,
 * hipFree, stream or event creation, and no memset nodes (fill kernels clear
 * what must start at zero).  Like every call here it cannot be captured into
 * a HIP graph (it reads results back between batches of rounds and waits for
 * the stream): on a capturing stream it returns NSFPS_EUNSUPPORTED before
 * enqueuing anything.  The array keeps the last call's contents; calls are
 * serialised by the library's lock, and a call on one device must not
 * overlap another use of that device's array (the library makes none).
 * Statistics report e2e_ms only (no device events). */
nsfps_status nsfps_fps_device_noalloc(const float *d_xyz, uint64_t n, uint64_t n_samples,
                                      const nsfps_range *range, int32_t *d_out,
                                      uint64_t *out_len, void *stream);
uint64_t nsfps_noalloc_scratch_bytes(void);

/* A cloud built once and sampled many times, the split of the reference GPU
 * driver's FpsGPU::initialize / FpsGPU::sample (eval/src_gpu/yuezu_fps_gpu.h:
 * 90-126).  nsfps_plan_create builds the structure of n points (xyz: host
 * pointer, or a device pointer when on_device != 0; read during the call
 * only) on the current device, in device memory the plan owns.
 * nsfps_plan_sample restores the points' min-distances and keys and runs the
 * sampling alone: the samples of nsfps_fps on the same points and range, for
 * any n_samples, written to device memory d_out (n_samples int32) on stream
 * (a hipStream_t, NULL = default stream); it returns after the stream work
 * completes and must be called with the plan's device current.  Calls on one
 * plan, or on several, are serialised by the library's lock.
 * nsfps_plan_destroy frees the plan (NULL is ignored). */
typedef struct nsfps_plan_s nsfps_plan;
nsfps_status nsfps_plan_create(const float *xyz, uint64_t n, const nsfps_range *range,
                               int on_device, nsfps_plan **plan);
nsfps_status nsfps_plan_sample(nsfps_plan *plan, uint64_t n_samples, int32_t *d_out,
                               uint64_t *out_len, void *stream);
void nsfps_plan_destroy(nsfps_plan *plan);

/* The step after sampling: set-abstraction grouping on the samples.  No
 * counterpart in the reference, which stops at the indices; the next step of
 * its callers is PointNet++'s sample-and-group (query_ball_point).
 *
 * nsfps_gather_points: out[i] = xyz[idx[i]], m x 3 float32.  An index outside
 * [0, n) fails with NSFPS_EINVAL (checked on the host for host pointers; the
 * device variant zeroes that row and reports it after the stream work).
 *
 * nsfps_ball_query: out is m x nsample int32; row j holds, in input order,
 * the first nsample indices i whose ((dx*dx + dy*dy) + dz*dz) to center j is
 * below radius*radius (float32, no contraction: the FPS distance); a row with
 * fewer hits repeats its first hit, a row with none is all zeros.  radius
 * must be finite and >= 0, nsample >= 1.
 *
 * The _device variants take device pointers and a hipStream_t (NULL = default
 * stream) and return after the stream work completes. */
nsfps_status nsfps_gather_points(const float *xyz, uint64_t n, const int32_t *idx, uint64_t m,
                                 float *out);
nsfps_status nsfps_gather_points_device(const float *d_xyz, uint64_t n, const int32_t *d_idx,
                                        uint64_t m, float *d_out, void *stream);
nsfps_status nsfps_ball_query(const float *xyz, uint64_t n, const float *centers, uint64_t m,
                              float radius, uint32_t nsample, int32_t *out);
nsfps_status nsfps_ball_query_device(const float *d_xyz, uint64_t n, const float *d_centers,
                                     uint64_t m, float radius, uint32_t nsample, int32_t *d_out,
                                     void *stream);

/* ------------------------------------------------------------------------
 * Sequence operators: what follows sampling in a model that reads a cloud's
 * samples as tokens.  The samples in the order of their grid cells are a
 * sequence; a sample's cell is its token (a vocabulary of total_blocks rows);
 * a selective state space scan with its short causal convolution mixes the
 * sequence.  No counterpart in the reference, which stops at the indices.
 *
 * All pointers are device pointers of the current device (d_..., and the p
 * of nsfps_rows); the argument structs live in host memory and are read
 * during the call only.  The calls only enqueue kernels on the stream (a
 * hipStream_t, NULL = default stream): they do not wait, allocate or copy, so
 * they can be captured into a HIP graph, and calls on several streams run
 * side by side.  Work that the kernels need beside their outputs is the
 * caller's: a call with a _workspace_bytes companion needs that many bytes
 * at workspace (aligned to 256), whose contents need not be kept, and which
 * calls that may overlap must not share.  The first call of an operator on a
 * device loads its kernels (seven and a half milliseconds for all of them);
 * nsfps_init_sequence_device does that ahead, before a capture for instance.
 * No output may overlap an input or another output, but those of norms and
 * dropout may be their own inputs' very rows (below).  Convolution, norms,
 * dropout and loss refuse other overlaps where the strides show them.  A
 * workspace that is too small, a size or stride that does not fit and a null
 * pointer are NSFPS_EINVAL; sizes beyond the limits named below are NSFPS_EUNSUPPORTED.
 * Nothing is enqueued by a refused call.
 *
 * Types: NSFPS_F32 and NSFPS_BF16 for inputs and outputs; sums, states and
 * the gradients of parameters are float32 with both.  In bfloat16 calls of the
 * scan and its gradient, computed factors of a product whose sum becomes a
 * bfloat16 output (scores, states in y, state gradients in db) hold 16 bits
 * there, those of other sums 24.  Results do not depend on the order in which
 * workgroups run: the same call gives the same bits. */
typedef enum { NSFPS_F32 = 0, NSFPS_BF16 = 1 } nsfps_dtype;

/* Loads the sequence operators' kernels on the current device.  Optional. */
nsfps_status nsfps_init_sequence_device(void);

/* A tensor of batch x length rows: row t of sequence b starts at
 * p + (b * batch_stride + t * row_stride) elements.  A row's elements are
 * contiguous.  Any strides that keep rows apart will do; the widest loads
 * need rows aligned to 16 bytes. */
typedef struct {
  void *p;
  uint64_t batch_stride, row_stride;
} nsfps_rows;

/* Embedding lookup: out[i] = scale * table[tokens[i]], tokens x width; a
 * token outside [0, rows) gives a row of zeros (the -1 that pads a batch's
 * index rows, say).
 *
 * Its gradient (d_out is then the input and d_table the output): every row v
 * of d_table is written, scale times the sum of the rows of d_out whose
 * token is v, zeros where no token is.  The tokens are sorted, and each
 * row's terms are added in float32 (in float64 where a row has more than 16) in
 * an order that the tokens alone decide.
 * d_out has type dtype, d_table grad_dtype.  At most 2^31 - 1 tokens and
 * rows (both calls), width at most 65,536. */
typedef struct {
  uint64_t tokens, rows;
  uint32_t width;
  uint32_t dtype;      /* lookup: table and out; gradient: out */
  uint32_t grad_dtype; /* gradient: table */
  float scale;
  uint64_t table_stride, out_stride; /* elements from row to row, >= width */
  void *d_table;
  const int32_t *d_tokens;
  void *d_out;
  void *workspace; /* gradient only */
  uint64_t workspace_bytes;
} nsfps_embed_args;
nsfps_status nsfps_embed_device(const nsfps_embed_args *args, void *stream);
nsfps_status nsfps_embed_grad_workspace_bytes(const nsfps_embed_args *args, uint64_t *bytes);
nsfps_status nsfps_embed_grad_device(const nsfps_embed_args *args, void *stream);

/* Ragged batches and caches, for the convolution and the scan alike:
 *   d_lengths    tokens of each sequence, at most length (NULL: all length);
 *                more count as length, fewer than 0 as 0.  Input rows past
 *                them are not read, output rows past them are zeros.
 *   d_positions  tokens that each sequence has had before this call (NULL:
 *                none).  0 starts it anew, whatever its caches hold; above 0
 *                continues from them.
 *   d_slots      each sequence's place in the caches (NULL: b); a negative
 *                one has none: it starts anew and leaves nothing.  No two
 *                sequences of a call may have the same place.
 * Convolution cache: [slots][width][channels] of type dtype; the input of
 * the token at position t is entry t modulo width.  Scan cache: [slots]
 * [heads][head_dim][state_dim] float32, the state after the last token. */

/* Short causal convolution over time with SiLU, each channel on its own:
 * y[t] = silu(bias + sum over k < width of weight[k] * x[t - (width-1) + k]).
 * width 2 to 4, weight [channels][width], bias [channels] (or NULL) of type
 * dtype.  d_cache (or NULL) is read where positions are above 0 and receives
 * the last inputs.  batch * length at most 2^31 - 1, channels at most 2^24.
 * y must not overlap x, nor dx x or dy (a tile of tokens reads those beside
 * it); where the strides show it, the call is refused.
 *
 * The gradient starts every sequence anew (d_positions, d_slots, d_cache
 * must be NULL; y is not read): dx of type dtype, d_dweight [channels][width]
 * and d_dbias [channels] (or NULL) in float32, all written. */
typedef struct {
  uint64_t batch, length;
  uint32_t channels, width, dtype;
  nsfps_rows x, y;
  const void *d_weight, *d_bias;
  const int32_t *d_lengths, *d_positions, *d_slots;
  void *d_cache;
  void *workspace; /* gradient only */
  uint64_t workspace_bytes;
} nsfps_conv_args;
typedef struct {
  nsfps_rows dy, dx;
  float *d_dweight, *d_dbias;
} nsfps_conv_grads;
nsfps_status nsfps_conv_device(const nsfps_conv_args *args, void *stream);
nsfps_status nsfps_conv_grad_workspace_bytes(const nsfps_conv_args *args, uint64_t *bytes);
nsfps_status nsfps_conv_grad_device(const nsfps_conv_args *args, const nsfps_conv_grads *grads,
                                    void *stream);

/* Selective state space scan.  Per head, with step = softplus(dt + dt_bias):
 *   state = exp(step * a) * state + step * x b^T   (head_dim x state_dim)
 *   y     = state c + d * x
 * x and y: rows of heads * head_dim; b and c: rows of groups * state_dim
 * (group g serves heads g * heads / groups onwards); dt: rows of heads; all
 * of type dtype; a, d and dt_bias: [heads] float32 (d and dt_bias may be
 * NULL).  a is not positive: exp(step * a) is a decay; an a of -infinity
 * forgets the state at every token, an a of NaN spoils its head.  A dt of
 * -infinity is a step of 0: the token leaves the state as it is.  Non-finite
 * inputs elsewhere spoil their sequence, and no other.  d_state (or NULL) is the
 * scan cache.  groups divides heads; head_dim and state_dim at most 128;
 * batch * heads at most 2^20; batch * length at most 2^31 - 1.
 *
 * The gradient starts every sequence anew (d_positions, d_slots and d_state
 * must be NULL; y is not read) and takes no gradient of the last state.  All
 * of dx, db, dc, ddt (type dtype) and d_da, d_dd, d_ddt_bias ([heads] float32;
 * the last two may be NULL) are written. */
typedef struct {
  uint64_t batch, length;
  uint32_t heads, groups, head_dim, state_dim, dtype;
  nsfps_rows x, b, c, dt, y;
  const float *d_a, *d_d, *d_dt_bias;
  const int32_t *d_lengths, *d_positions, *d_slots;
  float *d_state;
  void *workspace;
  uint64_t workspace_bytes;
} nsfps_scan_args;
typedef struct {
  nsfps_rows dy, dx, db, dc, ddt;
  float *d_da, *d_dd, *d_ddt_bias;
} nsfps_scan_grads;
nsfps_status nsfps_scan_workspace_bytes(const nsfps_scan_args *args, uint64_t *bytes);
nsfps_status nsfps_scan_device(const nsfps_scan_args *args, void *stream);
nsfps_status nsfps_scan_grad_workspace_bytes(const nsfps_scan_args *args, uint64_t *bytes);
nsfps_status nsfps_scan_grad_device(const nsfps_scan_args *args, const nsfps_scan_grads *grads,
                                    void *stream);

/* One token of every request, convolution and scan in one launch over the
 * caches that both leave: xbc (rows of heads * head_dim + 2 * groups *
 * state_dim channels: x, b, c) goes through the convolution, and x, b, c of
 * its result with dt through one step of the scan.  Between the two nothing
 * is rounded.  d_positions (required): tokens that each request has had; the
 * caller adds one after the call.  d_slots as above (NULL: b); a request
 * whose slot is negative gets a row of zeros and touches no cache.  width 2
 * to 4; head_dim and state_dim at most 128. */
typedef struct {
  uint64_t batch;
  uint32_t heads, groups, head_dim, state_dim, width, dtype;
  uint64_t xbc_stride, dt_stride, y_stride; /* elements from request to request */
  const void *d_xbc, *d_weight, *d_bias, *d_dt;
  const float *d_a, *d_d, *d_dt_bias;
  const int32_t *d_positions, *d_slots;
  void *d_cache;
  float *d_state;
  void *d_y;
} nsfps_step_args;
nsfps_status nsfps_scan_step_device(const nsfps_step_args *args, void *stream);

/* Norms of queries and keys, head by head, and the rotation by their position,
 * in one pass; of the scan's c and b say, between convolution and scan.  Per
 * head, with x its head_dim values:
 *   n = weight * x / sqrt(mean(x^2) + eps)
 * and of n's first rotary_dim values the pair (u, v) number i becomes
 *   u cos(w) - v sin(w), u sin(w) + v cos(w),  w = position * freq[i];
 * the values behind them stay.  Pairs are (i, i + rotary_dim / 2), with
 * neighbours != 0 (2i, 2i + 1).  A token's position is the one of its sequence
 * (d_positions, below 0 as 0; NULL: 0) plus its row's number; angles are exact
 * to 2^-22 at any position, for frequencies of up to 2^40.  Rows past a sequence's length are zeros.
 *
 * q and q_out: rows of q_heads * head_dim; k and k_out: rows of k_heads *
 * head_dim, all of type dtype (one of the two may have no heads).  Weights
 * [head_dim] of type dtype, or NULL (ones); freq [rotary_dim / 2] float32.
 * head_dim at most 256, rotary_dim even and at most head_dim (0: no
 * rotation), eps above 0; (q_heads + k_heads) * head_dim at most 2^24; batch *
 * length at most 2^31 - 1.  A head whose sum of squares passes float32 (values
 * near 10^19) becomes zeros, and so does its gradient.  In place: q_out may be
 * q's rows and k_out k's, and of the gradient dq those of q or dq_out, dk those
 * of k or dk_out.
 *
 * The gradient takes those of q_out and k_out and writes all of dq and dk
 * (type dtype), and d_dq_weight and d_dk_weight ([head_dim] float32, or NULL),
 * whose sums are off by 2^-16 of the terms' sizes at most, however many tokens;
 * q_out and k_out are not read. */
typedef struct {
  uint64_t batch, length;
  uint32_t q_heads, k_heads, head_dim, rotary_dim, neighbours, dtype;
  float eps;
  nsfps_rows q, k, q_out, k_out;
  const void *d_q_weight, *d_k_weight;
  const float *d_freq;
  const int32_t *d_lengths, *d_positions;
  void *workspace; /* gradient only */
  uint64_t workspace_bytes;
} nsfps_norm_args;
typedef struct {
  nsfps_rows dq_out, dk_out, dq, dk;
  float *d_dq_weight, *d_dk_weight;
} nsfps_norm_grads;
nsfps_status nsfps_norm_device(const nsfps_norm_args *args, void *stream);
nsfps_status nsfps_norm_grad_workspace_bytes(const nsfps_norm_args *args, uint64_t *bytes);
nsfps_status nsfps_norm_grad_device(const nsfps_norm_args *args, const nsfps_norm_grads *grads,
                                    void *stream);

/* Dropout onto a residual, the mask made where it is used and never stored:
 *   y = residual + (kept ? x / (1 - p) : 0)
 * (residual.p NULL: no residual).  Its gradient by x is the same call on dy
 * without residual; that by residual is dy inside the sequences and 0 past their
 * ends, which the same call with p = 0 makes.  Of a row's channels the eight from
 * 8 k on take 16 bits each, low half first, of the four words of Philox 4x32-10
 * (Salmon, Moraes, Dror, Shaw, 2011) at counter (k, row's number b * length +
 * t, d_seed[1] low, high) and key (d_seed[0] low, high); a value is dropped
 * where they are below p * 65536, rounded, and the factor is that of the
 * rounded p.  So the mask hangs on sizes and seed alone, not on types, strides
 * or lengths.  d_seed: two words in device memory, a key and the number of the
 * call (a captured graph's caller changes it between replays).  0 <= p <= 1 (1:
 * all is dropped); channels at most 2^24, batch * length at most 2^31 - 1.  Rows
 * past a sequence's length are zeros, their inputs are not read.  In place: y may
 * be the rows of x or of residual. */
typedef struct {
  uint64_t batch, length;
  uint32_t channels, dtype;
  float p;
  nsfps_rows x, residual, y;
  const uint64_t *d_seed;
  const int32_t *d_lengths;
} nsfps_dropout_args;
nsfps_status nsfps_dropout_device(const nsfps_dropout_args *args, void *stream);

/* Softmax cross entropy of tokens over a vocabulary of table rows, the logits
 * of which are never held at once:
 *   z[i][v] = scale * x[i] . table[v]   (x: tokens x width, table: rows x width)
 *   lse[i] = log(sum over v of exp(z[i][v])),  loss[i] = lse[i] - z[i][targets[i]]
 * A token whose target is outside [0, rows) has a loss of 0 and no gradient,
 * whatever its row of x holds (its lse is that row's).  d_loss and d_lse: [tokens]
 * float32, all written.
 *
 * The gradient needs d_lse as the call left it (d_loss is not read) and
 * d_dloss, the gradient of each token's loss: d_dx (type dtype, rows dx_stride
 * apart) and d_dtable (type grad_dtype, rows dtable_stride apart) are all
 * written.  exp(z - lse) - (v is the target), times dloss and scale, enters the
 * products in bfloat16 where the result is bfloat16, with 16 bits for a float32
 * table gradient of bfloat16 inputs, with 24 in float32 calls.
 *
 * scale and scale * log2(e) have to be finite.  A row of the table that is not
 * finite spoils every token.  At most 2^30
 * tokens, 2^31 - 1 rows, width at most 65,536.  The gradient takes the
 * vocabulary in pieces, whose products live in the workspace, beside copies of
 * rows that the kernels cannot take as they are; its size goes by sizes and types
 * alone.  bfloat16 rows of a multiple of 64 values at 16-byte boundaries are the
 * fastest. */
typedef struct {
  uint64_t tokens, rows;
  uint32_t width, dtype;
  float scale;
  uint64_t x_stride, table_stride; /* elements from row to row, >= width */
  const void *d_x, *d_table;
  const int32_t *d_targets;
  float *d_loss, *d_lse;
  void *workspace;
  uint64_t workspace_bytes;
} nsfps_loss_args;
typedef struct {
  const float *d_dloss;
  uint64_t dx_stride, dtable_stride;
  uint32_t grad_dtype;
  void *d_dx, *d_dtable;
} nsfps_loss_grads;
nsfps_status nsfps_loss_workspace_bytes(const nsfps_loss_args *args, uint64_t *bytes);
nsfps_status nsfps_loss_device(const nsfps_loss_args *args, void *stream);
nsfps_status nsfps_loss_grad_workspace_bytes(const nsfps_loss_args *args,
                                             const nsfps_loss_grads *grads, uint64_t *bytes);
nsfps_status nsfps_loss_grad_device(const nsfps_loss_args *args, const nsfps_loss_grads *grads,
                                    void *stream);

/* Measurements of the last compute call made on this thread. */
nsfps_status nsfps_get_stats(nsfps_stats *stats);

/* Phase clocks and work counters of the single-workgroup sampling loop of the
 * last call on this thread (cloud 0), recorded only when the environment
 * variable NSFPS_PROFILE is set (all zero otherwise).  Words 0-8: s_memtime
 * cycles spent between the loop's barriers (0 cube, 1 cell enumeration + scan,
 * 2 flatten, 3 fast phase A: candidate + sibling loads, 4 fast phase B,
 * 5 fast phase C / slow rounds, 6 slow level-1 rebuild, 7 level 2, 8 root);
 * 16 iterations, 17 fast iterations, 18 cube cells, 19 candidate leaves,
 * 20 dirty level-1 nodes on fast iterations, 21 elapsed s_memrealtime ticks
 * (100 MHz).  No counterpart in the reference (it has no instrumentation). */
nsfps_status nsfps_get_loop_profile(uint64_t *words, uint32_t nwords);

/* Releases the cached device workspace of the calling process, and the pinned
 * host buffer that host-buffer inputs are staged through. */
void nsfps_release_workspace(void);

#ifdef __cplusplus
}
#endif

#endif
