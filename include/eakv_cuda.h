/* eakv_cuda.h - extension entry points of libeakv_b200.so.
 *
 * Everything in eakv.h keeps the reference's host-pointer contract. The
 * calls below add what a GPU-resident cache needs and the reference has no
 * counterpart for: device-pointer variants (no host copies, asynchronous on
 * the cache's CUDA stream), the fused softmax attention the reference
 * ships only as an unexposed kernel (reference kernels/fused_attention.ea:
 * 10-373), a batched decode step over many caches and all layers, and the
 * sequence-split partial + log-sum-exp combine used across GPUs.
 *
 * All functions return EAKV_OK or a negative EAKV_ERR_* code unless noted;
 * the reason of the last failure on the calling host thread is available
 * from eakv_last_error_string(). Pointer arguments named d_* are device
 * pointers on the cache's device; "stream" arguments are cudaStream_t
 * (NULL selects the first cache's own stream).
 */
#ifndef EAKV_CUDA_H
#define EAKV_CUDA_H

#include <stddef.h>
#include <stdint.h>
#include "eakv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- errors and device state ---------------------------------------- */

/* Code of the last failed call on this host thread, EAKV_OK if none. The
 * void attention functions of eakv.h (reference src/attention.c:3-63 has no
 * error channel) report through this. */
int         eakv_last_error(void);
const char *eakv_last_error_string(void);

/* Sticky device status word of the library's kernels on `device`: 0 when
 * clean, else a bitmask (1 = a pipeline wait ran out of its bound, 2 = a
 * decode work item failed its index check and was skipped, 4 = a decode
 * CTA found a copy still in flight at its end and drained it). reset != 0
 * clears it. Synchronizes the device.
 * Returns the status, or a negative EAKV_ERR_* code. */
int eakv_device_status(int device, int reset);

/* ---- placement ------------------------------------------------------- */

/* Device on which this host thread's later eakv_cache_create / load calls
 * place caches (the library keeps its own CUDA runtime state, so a device
 * chosen through another runtime, e.g. a framework, is not seen here). */
int    eakv_set_device(int device);

int    eakv_cache_device(const eakv_cache_t *cache);         /* -1 for NULL */
/* HBM held by the cache: its page slab plus the scratch that host-buffer
 * calls, split decodes and eakv_extend_attention grow on demand. */
size_t eakv_cache_device_bytes(const eakv_cache_t *cache);
/* Stream used by this cache's calls; NULL restores the cache's own. */
int    eakv_cache_set_stream(eakv_cache_t *cache, void *stream);
void  *eakv_cache_stream(const eakv_cache_t *cache);
int    eakv_cache_synchronize(const eakv_cache_t *cache);

/* ---- device-pointer variants of eakv.h ------------------------------- */

/* As eakv_cache_load_raw / eakv_cache_append with device input
 * (reference src/cache.c:60-151); asynchronous. */
int eakv_cache_load_raw_device(eakv_cache_t *cache, const float *d_data,
                               int seq_len);
int eakv_cache_append_device(eakv_cache_t *cache, const float *d_data,
                             int layer, int kv_idx, int n_tokens);
/* One launch for every layer and K/V: d_data is
 * f32[n_layers][2][n_kv_heads][n_tokens][head_dim]. Writes at seq_len and,
 * like eakv_cache_append, does not advance. */
int eakv_cache_append_step_device(eakv_cache_t *cache, const float *d_data,
                                  int n_tokens);

/* As eakv_attention_scores / eakv_attention_output (reference
 * src/attention.c:3-63) on device buffers; asynchronous. */
int eakv_attention_scores_device(const eakv_cache_t *cache,
                                 const float *d_queries, int layer,
                                 int n_q_heads, int n_kv_heads,
                                 float *d_scores);
int eakv_attention_output_device(const eakv_cache_t *cache,
                                 const float *d_weights, int layer,
                                 int n_q_heads, int n_kv_heads,
                                 float *d_output);

/* ---- fused softmax attention ----------------------------------------- */

/* output = softmax(Q K^T / sqrt(head_dim)) V for one layer, host buffers
 * (queries/output f32[n_q_heads*head_dim]); the device counterpart of
 * reference kernels/fused_attention.ea:190-373 for any head mapping. */
int eakv_attention_fused(const eakv_cache_t *cache, const float *queries,
                         int layer, int n_q_heads, int n_kv_heads,
                         float *output);
int eakv_attention_fused_device(const eakv_cache_t *cache,
                                const float *d_queries, int layer,
                                int n_q_heads, int n_kv_heads,
                                float *d_output);

/* Batched decode step: n_caches caches of identical shape (layers, KV
 * heads, head_dim, max_seq_len), each attended over its own seq_len, all
 * layers in one launch. d_queries / d_output are
 * f32[n_caches][n_layers][n_q_heads][head_dim]. n_caches <= 256. */
int eakv_decode_attention(const eakv_cache_t *const *caches, int n_caches,
                          const float *d_queries, int n_q_heads,
                          float *d_output, void *stream);
/* Same as eakv_decode_attention, for callers that cannot allocate device
 * memory: no counterpart in the reference, whose CPU path has no device
 * memory at all. A framework whose caching allocator owns the GPU, or a
 * decode loop that must not block on cudaMalloc/cudaFree, gets the
 * split-merge workspace from a fixed 4 MiB array in the library's device
 * image (held by every GPU that loads the library) instead of from cache
 * scratch grown with cudaMalloc. Calls needing more than 4 MiB of workspace
 * return EAKV_ERR_INVALID. All calls on a device share the array: calls
 * whose kernels overlap on the GPU race. The first call on a device looks
 * up the array's address and should come before any stream capture. */
int eakv_decode_attention_noalloc(const eakv_cache_t *const *caches,
                                  int n_caches, const float *d_queries,
                                  int n_q_heads, float *d_output, void *stream);
/* Same with host buffers; copies in, decodes, copies out, synchronizes.
 * From 256 KiB of queries on, the batch is cut into up to four chunks of
 * caches (or of layers, for one cache) whose copies overlap the other
 * chunks' decodes; every chunk keeps the whole batch's split plan, so the
 * outputs equal eakv_decode_attention's bit for bit. */
int eakv_decode_attention_host(const eakv_cache_t *const *caches,
                               int n_caches, const float *queries,
                               int n_q_heads, float *output, void *stream);

/* Number of kernel launches one eakv_decode_attention call over these
 * caches makes: 1 (rows cut into sequence splits are merged inside the same
 * launch by the last CTA of each row group); < 0 on error. */
int eakv_decode_launches(const eakv_cache_t *const *caches, int n_caches,
                         int n_q_heads);
/* Sequence splits per row the planner chooses for one eakv_decode_attention
 * call over these caches (1: rows are not split and no split workspace is
 * used); < 0 on error. */
int eakv_decode_splits(const eakv_cache_t *const *caches, int n_caches,
                       int n_q_heads);

/* ---- sequence-split partials and exact combine ----------------------- */

/* Attention restricted to positions [pos_begin, min(pos_end, seq_len)) of
 * every cache: d_output gets that range's normalized output and d_lse
 * (f32[n_caches][n_layers][n_q_heads]) its natural-log log-sum-exp of the
 * scaled scores (-inf when the range is empty). */
int eakv_decode_attention_partial(const eakv_cache_t *const *caches,
                                  int n_caches, const float *d_queries,
                                  int n_q_heads, int pos_begin, int pos_end,
                                  float *d_output, float *d_lse, void *stream);

/* Exact merge of n_parts partial results over disjoint position ranges:
 * d_parts f32[n_parts][n_rows][head_dim], d_lse f32[n_parts][n_rows] ->
 * d_output f32[n_rows][head_dim] (and d_lse_out f32[n_rows] if not NULL):
 * out = sum_p exp(lse_p - L) out_p with L = log sum_p exp(lse_p). */
int eakv_lse_combine(int n_parts, int n_rows, int head_dim,
                     const float *d_parts, const float *d_lse,
                     float *d_output, float *d_lse_out, void *stream);

/* ---- inspecting a resident cache ------------------------------------------ */

/* Device validate: the reference's q4_validate (kernels/validate.ea:14-71) as
 * its CLI runs it on every (layer, K/V) block (src/cli.c:39-98), without
 * copying the cache to the host. codes (host, n_layers*2 entries, index
 * layer*2 + kv) receive 0 (ok), 1 (NaN scale), 2 (NaN bias) or 3 (negative
 * scale) for the first failing group in the reference's order ([head]
 * [position][group], positions < seq_len). Returns EAKV_OK or an error. */
int eakv_cache_validate(const eakv_cache_t *cache, int32_t *codes);

/* Dequantize positions [pos_begin, pos_end) of one (layer, K/V) block into
 * f32 [n_kv_heads][pos_end - pos_begin][head_dim], value = nibble * scale +
 * bias with one rounding (reference kernels/dequantize_avx512.ea:10-89, whose
 * range form :52-89 this generalises). The _device form writes device
 * memory on `stream` (NULL: the cache's stream; d_out 16-byte aligned); the
 * other writes host memory and returns when done. EAKV_ERR_INVALID for a bad
 * block, range or alignment. */
int eakv_cache_dequantize_device(const eakv_cache_t *cache, int layer, int kv_idx, int pos_begin,
                                 int pos_end, float *d_out, void *stream);
int eakv_cache_dequantize(const eakv_cache_t *cache, int layer, int kv_idx, int pos_begin,
                          int pos_end, float *out);

/* ---- several tokens per call --------------------------------------------
 *
 * A model's layer loop over a batch of caches, with any number of new tokens
 * per cache: append the layer's K and V (rotated and quantized in one
 * launch), attend, and after the last layer advance (or keep only the
 * accepted tokens with eakv_cache_compact). The tokens of a call are packed:
 * cache 0's n_new[0] tokens first, then cache 1's, and so on; a count may be
 * 0. The caches of a call share a shape and a device, n_caches <= 256,
 * head_dim is 64 or 128. n_new and the other count arrays are host memory,
 * read before the call returns. All calls are asynchronous on `stream`
 * (NULL: the first cache's own stream) and can be captured into a graph,
 * which keeps the counts and sequence lengths of the captured call. */

/* Element types of device buffers. */
#define EAKV_F32  0
#define EAKV_F16  1
#define EAKV_BF16 2

/* Rows [token][head][head_dim] of a device buffer: element d of (token t,
 * head h) is at data + t*token_stride + h*head_stride + d (strides in
 * elements), so a slice of a fused q/k/v projection needs no copy. Rows that are
 * read may overlap (a stride of 0 broadcasts one); of rows that are written a stride
 * below head_dim is refused where there is more than one row along it. Rows that
 * do not start on a 4-element boundary are read and written one element at a
 * time. */
typedef struct {
    void     *data;
    int64_t   token_stride;
    int64_t   head_stride;
    int       dtype;        /* EAKV_F32, EAKV_F16 or EAKV_BF16 */
} eakv_rows_t;

/* Rotary positions. The first rot_dim dims of a head (a multiple of 8) are
 * rot_dim/2 pairs: (i, i + rot_dim/2), or (2i, 2i+1) when interleaved. Pair
 * i of a token turns by the angle whose cosine and sine are at
 * [position][i] of the f32 tables [n_rows][rot_dim/2] (16-byte aligned), with the token's
 * position on the axis that pair i follows: the first sections[0] pairs
 * follow axis 0, the next sections[1] axis 1, and so on (one axis for text;
 * time, height and width for images and video). positions is device
 * int32[n_axes][total tokens], axis a at positions + a*axis_stride. */
#define EAKV_MAX_AXES 4
typedef struct {
    const float   *cos_table;
    const float   *sin_table;
    int            n_rows;
    int            rot_dim;
    int            interleaved;
    const int32_t *positions;
    int64_t        axis_stride;
    int            n_axes;
    int            sections[EAKV_MAX_AXES];
} eakv_rotary_t;

/* Quantizes the new tokens' K and V rows of one layer into the pages of
 * their caches, at positions seq_len .. seq_len + n_new - 1 (seq_len is not
 * changed, as with eakv_cache_append), K turned by `rotary` first (NULL: not
 * turned); and writes the turned q rows (n_q_heads heads; q NULL: none) to
 * q_out, which may be q itself. k, v, q and q_out have one element type. The
 * turned K is rounded once, to f32, and then quantized like
 * eakv_cache_append's f32 input: the same groups, bit for bit. A token with a
 * position outside the table sets status bit 2 (eakv_device_status) and its
 * rows are not written. */
int eakv_append_rotary(eakv_cache_t *const *caches, int n_caches, int layer, const int *n_new,
                       const eakv_rows_t *k, const eakv_rows_t *v, const eakv_rows_t *q,
                       const eakv_rows_t *q_out, int n_q_heads, const eakv_rotary_t *rotary,
                       void *stream);

/* Attention of the new tokens of one layer over the caches. Token t of cache
 * i stands at position seq_len + t and attends positions 0 .. seq_len + t,
 * its own and the earlier new tokens' among them (they are appended, and not
 * yet advanced over); with window > 0 only the last `window` of those; with
 * tree (device uint64[total tokens], n_new <= 64) of the new tokens exactly
 * those j whose bit j is set in its word, within the window (of slots: the call
 * with depths below goes by positions). Query head h reads KV
 * head h / (n_q_heads / n_kv_heads). out gets softmax(scale q.k) v, scale
 * 1/sqrt(head_dim) when given as 0; lse (device f32[total tokens][n_q_heads],
 * or NULL) the natural-log log-sum-exp of the scaled scores. A token that
 * attends nothing gets zeros and -inf. What is not attended has no influence,
 * NaN among it. q and out have one element type, and out may be q itself (a
 * row is read by all its parts before it is written). Sums are f32. f32 runs on
 * split operands that keep 22 bits, at any number of rows; a 16-bit type on one
 * f16 operand each: with up to 32 rows (new tokens x query heads) per KV head
 * the cache's values enter exactly, with more each is rounded to f16, which puts
 * f16 outputs 0.7e-3 of their size off in the mean (0.3e-3 with few rows) and
 * bf16 ones 1.8e-3, of which 1.7e-3 are the output's own rounding. A caller who
 * needs more bits there passes f32 rows. workspace (device, 16-byte aligned)
 * holds the records of long rows' sequence splits: at least eakv_extend_workspace bytes, zeroed once before
 * its first use, and not shared by calls that may overlap; NULL takes one that
 * the first cache keeps for this call, which then must not be in use on another
 * stream. A captured call takes a workspace of its own, since the cache's moves
 * when a later call needs more of it. (What the cache keeps for its decodes
 * stays where it is.) */
int eakv_extend_attention(const eakv_cache_t *const *caches, int n_caches, int layer,
                          const int *n_new, const eakv_rows_t *q, const eakv_rows_t *out,
                          int n_q_heads, float scale, int window, const uint64_t *tree, float *lse,
                          void *workspace, size_t workspace_bytes, void *stream);
/* The same for a tree under a sliding window, which goes by positions: token t of a
 * cache stands at seq_len + depth[t], not at its slot seq_len + t (depth: device
 * int32[total tokens], the number of its ancestors, 0 <= depth[t] <= t), and
 * attends what its mask names and the cached positions, of these the last
 * `window` up to its own: what it attends once the accepted branch is kept by
 * eakv_cache_compact. Another depth sets status bit 2 and counts as t. depth NULL
 * is eakv_extend_attention; depth needs a tree. */
int eakv_extend_attention_depths(const eakv_cache_t *const *caches, int n_caches, int layer,
                                 const int *n_new, const eakv_rows_t *q, const eakv_rows_t *out,
                                 int n_q_heads, float scale, int window, const uint64_t *tree,
                                 const int32_t *depth, float *lse, void *workspace,
                                 size_t workspace_bytes, void *stream);
/* Bytes of workspace such a call needs (0: none); tree is 0 without masks, 1 with
 * them, 2 with depths too. */
int eakv_extend_workspace(const eakv_cache_t *const *caches, int n_caches, const int *n_new,
                          int dtype, int n_q_heads, int window, int tree, size_t *bytes);

/* Copies positions [src_pos, src_pos + n) of every layer and head to
 * [dst_pos, dst_pos + n) of n_dst other caches in one launch, as they are
 * (nibbles, scales and biases), and sets their seq_len to dst_pos + n:
 * dst_pos <= their seq_len, src_pos + n <= src's. The caches agree in layers,
 * heads and head_dim; their max_seq_len may differ. n_dst <= 256. Here and in
 * eakv_cache_gather a stream of NULL is src's; what runs on the destinations'
 * own streams has to be ordered behind it by the caller. */
int eakv_cache_copy(eakv_cache_t *const *dsts, int n_dst, int dst_pos, const eakv_cache_t *src,
                    int src_pos, int n, void *stream);
/* A new cache of max_seq_len positions on src's device with src's first n, copied on
 * src's own stream, behind which the new cache's starts. Not for stream capture
 * (it allocates). */
int eakv_cache_fork(const eakv_cache_t *src, int n, int max_seq_len, eakv_cache_t **out);
/* Position dst_pos + j of (layer l, KV head h) of dst becomes position
 * index[l*layer_stride + h*head_stride + j] of src, j < n, for K and V; sets
 * dst's seq_len to dst_pos + n. index is device int32; a stride of 0 shares
 * one list between layers or heads; with n == 0 it may be NULL. An index outside [0, src's seq_len) sets
 * status bit 2 and leaves its position as it was. */
int eakv_cache_gather(eakv_cache_t *dst, int dst_pos, const eakv_cache_t *src, const int32_t *index,
                      int64_t layer_stride, int64_t head_stride, int n, void *stream);
/* The same within one cache: position begin + j becomes index[..+ j], and
 * seq_len begin + n; keeps a drafted branch, or evicts. index may reach up to
 * max_seq_len (appended tokens not yet advanced over), and no entry is below
 * its own place (index >= begin + j, as in every ascending list); one that is,
 * sets status bit 2 and leaves its position as it was. */
int eakv_cache_compact(eakv_cache_t *cache, int begin, const int32_t *index, int64_t layer_stride,
                       int64_t head_stride, int n, void *stream);

/* The values (nibble * scale + bias, rounded once to f32 and from there to the
 * rows' type) of positions [begin[i], begin[i] + n[i]) of cache i, i <
 * n_caches, for layers layer0 .. layer0 + n_layers - 1: rows packed like the
 * tokens of eakv_append_rotary, K of layer l at k->data + l*layer_stride
 * elements, V at v->data + the same (either may be NULL). Positions up to
 * max_seq_len may be read. */
int eakv_cache_read(const eakv_cache_t *const *caches, int n_caches, int layer0, int n_layers,
                    const int *begin, const int *n, const eakv_rows_t *k, const eakv_rows_t *v,
                    int64_t layer_stride, void *stream);

/* ---- testing aid ------------------------------------------------------ */

/* Forces every later fused / decode call on this host thread to cut each
 * row (eakv_extend_attention: each tile of rows) into n sequence splits (0
 * restores the automatic choice), so tests can exercise the split + combine
 * path on small caches. */
int eakv_test_force_splits(int n);

/* The decode planner's split count, for tests of the planner without a GPU
 * (pure host code, no CUDA call): `items` rows of max_pages pages, searched
 * in [lo, hi], per_sm CTAs resident on each of `sms` SMs. The planner itself
 * takes lo and hi from the precision cap and the two-page minimum, and
 * per_sm / sms from the device. */
int eakv_test_choose_splits(long long items, int max_pages, int lo, int hi, int per_sm,
                            int sms);

/* Kernel choice of later fused / decode calls on this host thread, for tests
 * and side-by-side measurements: 1 the CUDA-core kernel even for shapes the
 * tensor-core kernels serve, 2 the mma.sync tensor-core kernel (the automatic
 * choice), 3 the tcgen05 tensor-core kernel (head_dim 128; other shapes keep
 * the automatic choice); 0 restores the automatic choice. For
 * eakv_extend_attention on 16-bit types 2 takes the mma.sync kernel and 3 the
 * tcgen05 kernel whatever the number of rows is. */
int eakv_test_force_path(int path);

/* Later eakv_extend_attention calls on this host thread take the tcgen05
 * kernel to have been built with n registers per thread (0: what it was built
 * with). It can only run with the number it was written for; with another, as
 * another compiler may give it, the mma.sync kernel serves every call. */
int eakv_test_extend_registers(int n);

/* on != 0 makes later decode calls on this host thread merge their sequence
 * splits in a second kernel launch after the decode, instead of in the
 * decode kernel's last CTA of each row group; 0 restores the default. The
 * arithmetic is the same; tests compare the two bit for bit. */
int eakv_test_separate_merge(int on);

/* Failure-detection test: later fused / decode calls on this host thread
 * never request page `page` of each (row, split) work item into the
 * pipeline (page < 0 restores normal operation; eakv_extend_attention's
 * tcgen05 kernel never announces the scores of tile `page` instead), and
 * every wait of those kernels gives up after `wait_budget` polls (0: the
 * default budget). The
 * wait for the missing page then runs out: the kernel sets bit 1 of the
 * device status word (eakv_device_status), waits for the copies it did
 * request, and returns without writing its outputs. Nothing faults; the
 * context stays usable. */
int eakv_test_stall(int page, unsigned wait_budget);

#ifdef __cplusplus
}
#endif

#endif /* EAKV_CUDA_H */
