/*
 * shk_cuda.h -- C ABI of the B200 (sm_100a) decode path for the Shukuchi engine.
 *
 * This library replaces the reference's Apple Metal backend
 * (engine/include/metal_ops.h:5-26) and adds device-side versions of the ops
 * (engine/include/ops.h:9-38), the Q8_0 KV cache (engine/include/kv_cache.h:5-37)
 * and the per-layer forward (engine/src/engine.c:76-229), so the C engine keeps
 * its model/layer API and CLI while all math runs as hand-written CUDA kernels.
 *
 * Conventions
 *  - Plain C types only.  Pointers named *_dev are device pointers; *_host are
 *    host pointers.  `stream` is a cudaStream_t passed as void* (NULL = the
 *    context's compute stream).
 *  - Every call returns an int status: 0 ok, negative SHK_E* on error.  There is
 *    NO CPU fallback: an error is returned to the caller.
 *  - Device-side waits are bounded; a wait that runs out records SHK_ETIMEOUT
 *    in the context's error word (shk_cuda_check).
 *  - One compute thread per context; shk_cuda_layer_stage may be called from a
 *    separate loader thread (it uses the context's own copy stream).
 *  - Weight tensors are in GGUF block layout: Q4_K (ggml type 12, 144-byte
 *    super-blocks) and Q6_K (type 14, 210-byte super-blocks), rows of k/256
 *    blocks.  Device weight pointers must be 16-byte aligned.
 */
#ifndef SHK_CUDA_H
#define SHK_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum shk_status {
    SHK_OK = 0,
    SHK_EINVAL = -1,       /* bad argument / shape */
    SHK_ENOMEM = -2,       /* device or pinned allocation failed */
    SHK_ECUDA = -3,        /* CUDA runtime error */
    SHK_EUNSUPPORTED = -4, /* dtype or shape not handled (e.g. Q5_K) */
    SHK_ETIMEOUT = -5,     /* a bounded device wait ran out */
    SHK_ENODEV = -6,       /* no usable CUDA device */
    SHK_ENCCL = -7,        /* collective failure */
    SHK_EDEVICE = -8       /* kernel reported an error (bad position/token) */
};

typedef struct shk_ctx shk_ctx;     /* device, streams, error word, counters */
typedef struct shk_kv shk_kv;       /* Q8_0 KV cache in HBM */
typedef struct shk_model shk_model; /* dims, scratch, captured decode step */

struct shk_cuda_config {
    int device;     /* CUDA ordinal; -1 = current device */
    uint32_t flags; /* SHK_CUDA_FLAG_*; 0 = defaults */
};
/* Run whole-token decode (shk_cuda_token_step / shk_cuda_decode_steps) in the
 * persistent decode kernel (one cooperative launch per call, grid-wide
 * barriers between phases) instead of captured graphs of per-projection
 * kernels.  Both give the same results within fp32 rounding. */
#define SHK_CUDA_FLAG_PERSISTENT 2u
/* Capture the decode-step graphs without programmatic dependent launch
 * (each kernel then starts only after its predecessor has finished). */
#define SHK_CUDA_FLAG_NO_PDL 4u

/* ---- context: replaces metal_ops_init/metal_ops_shutdown/metal_available/
 *      metal_ops_report (engine/include/metal_ops.h:5-6, 24-25) ---- */
shk_ctx *shk_cuda_init(const struct shk_cuda_config *cfg);
void shk_cuda_shutdown(shk_ctx *ctx);
int shk_cuda_available(void);
void shk_cuda_report(shk_ctx *ctx);
/* Synchronises the compute stream and returns SHK_ETIMEOUT / SHK_EDEVICE if a
 * kernel recorded a device-side error since the last call (which clears it). */
int shk_cuda_check(shk_ctx *ctx);
const char *shk_cuda_strerror(int status);
void *shk_cuda_stream(shk_ctx *ctx);       /* compute stream (cudaStream_t) */
int shk_cuda_num_sms(shk_ctx *ctx);

/* ---- memory helpers for the engine and loader ---- */
int shk_cuda_dev_alloc(shk_ctx *ctx, size_t bytes, void **out_dev);
int shk_cuda_dev_free(shk_ctx *ctx, void *p_dev);
int shk_cuda_host_alloc(shk_ctx *ctx, size_t bytes, void **out_host); /* pinned */
int shk_cuda_host_free(shk_ctx *ctx, void *p_host);
int shk_cuda_memcpy_h2d(shk_ctx *ctx, void *dst_dev, const void *src_host, size_t bytes, void *stream);
int shk_cuda_memcpy_d2h(shk_ctx *ctx, void *dst_host, const void *src_dev, size_t bytes, void *stream);
int shk_cuda_sync(shk_ctx *ctx, void *stream);

/* ---- dequantise-matvec: replaces metal_matmul_q4k_vec / metal_matmul_q6k_vec
 *      (engine/include/metal_ops.h:7-23) as called from op_matmul_q4_k /
 *      op_matmul_q6_k (engine/src/ops.c:266-314, 361-404).
 *      y[r] = sum_k dequant(W[r,k]) * x[k], W m x k, k % 256 == 0.  Async. ---- */
int shk_cuda_matmul_q4k_vec(shk_ctx *ctx, const void *w_dev, const float *x_dev, float *y_dev,
                            uint32_t m, uint32_t k, void *stream);
int shk_cuda_matmul_q6k_vec(shk_ctx *ctx, const void *w_dev, const float *x_dev, float *y_dev,
                            uint32_t m, uint32_t k, void *stream);
/* replaces metal_matmul_q5k_vec (engine/include/metal_ops.h:5-26) as called
 * from op_matmul_q5_k (engine/src/ops.c:316-359).  W is in the reference's
 * 176-byte Q5_K block layout {u16 d, u16 dmin, u8 scales[12], u8 qh[32],
 * u8 qs[128]}, element i of a block = low nibble (i even) / high nibble (i odd)
 * of qs[i/2] plus bit i%8 of qh[i/8] as the fifth bit (dequantize_row_q5_k,
 * :144-165), rows dense; w_dev and x_dev 16-byte aligned.  Async. */
int shk_cuda_matmul_q5k_vec(shk_ctx *ctx, const void *w_dev, const float *x_dev, float *y_dev,
                            uint32_t m, uint32_t k, void *stream);

/* ---- Q6_K weight layout in HBM.  No counterpart in the reference (its
 *      weights stay in the GGUF layout in host memory).  The staged GEMV reads
 *      Q6_K rows in a planar layout: the same 210 * k/256 bytes of a row
 *      regrouped as [ql of every block][qh][scales][d], each plane 16-byte
 *      aligned, with the 16-byte chunks of a block rotated by the block index
 *      (ql chunk c of block b at 128 b + 16 ((c + b) & 7), qh chunk c at
 *      128 nb + 64 b + 16 ((c + (b >> 1)) & 3), scales at 192 nb + 16 b, d at
 *      208 nb + 2 b).  Weights registered with a model as Q6_K must be in this
 *      layout and carry dtype SHK_DTYPE_Q6_K_PLANAR (output head: GGUF Q6_K is
 *      also accepted, on the plain-load kernel). ---- */
#define SHK_DTYPE_Q6_K_PLANAR 0x10Eu
/* Converts `rows` Q6_K rows of k elements, row_stride bytes apart (0 = 210 *
 * k/256; must be a multiple of 16 and at most 227 KB), in place: to the
 * planar layout (to_planar != 0) or back to GGUF blocks.  Async on stream. */
int shk_cuda_q6k_repack(shk_ctx *ctx, void *w_dev, uint32_t rows, uint32_t k, uint32_t row_stride,
                        int to_planar, void *stream);
/* ---- Row-tiled weight layout for the tensor-core matvec.  No counterpart in
 *      the reference (its weights stay GGUF blocks in host memory, read by
 *      op_matmul_q4_k / op_matmul_q6_k, engine/src/ops.c:266-314, 361-404).
 *      A matrix of `rows` rows and nb = k/256 super-blocks becomes ceil(rows/16)
 *      row tiles; tile (row tile t, block b) holds block b of rows 16t..16t+15
 *      (rows past `rows` are zero) at byte (t * nb + b) * tile_bytes, tile_bytes
 *      = 16 * 144 (Q4_K) or 16 * 210 (Q6_K).  Inside a tile the GGUF bytes are
 *      only moved, into the order the tensor-core fragments read them:
 *        Q4_K: [0,256) the 16 rows' 16-byte block headers (d, dmin, scales);
 *              [256,2304) [chunk j<4][lane<32][16]: row g = lane/4 quant bytes
 *              32j + 8(lane%4) .. +7, then row g+8's.
 *        Q6_K: [0,3072) [half n<2][lane<32][48]: row g ql bytes 64n + 8t..+7,
 *              ql 64n+32+8t..+7, qh 32n+8t..+7 (t = lane%4), then row g+8's;
 *              [3072,3328) int8 scales[16] per row; [3328,3360) fp16 d per row.
 *      Weights registered as SHK_DTYPE_Q4_K_TILED / SHK_DTYPE_Q6_K_TILED run on
 *      the tensor-core matvec (mma.sync int8 over fixed-point x limbs). ---- */
#define SHK_DTYPE_Q4_K_TILED 0x20Cu
#define SHK_DTYPE_Q6_K_TILED 0x20Eu
/* Bytes of the tiled form of a rows x k matrix of dtype 12/14 (or a tiled
 * dtype); 0 for other dtypes or k not a multiple of 256. */
size_t shk_cuda_tiled_bytes(uint32_t dtype, uint32_t rows, uint32_t k);
/* GGUF rows (dtype 12 or 14, src_row_stride bytes apart, 0 = dense) -> the
 * tiled layout at dst_dev (shk_cuda_tiled_bytes bytes, 16-byte aligned, not
 * overlapping src).  Async on stream. */
int shk_cuda_tile(shk_ctx *ctx, uint32_t dtype, const void *src_dev, uint32_t src_row_stride, uint32_t rows,
                  uint32_t k, void *dst_dev, void *stream);
/* ---- batched prefill matmul on the tensor cores.  No counterpart in the
 *      reference, which feeds prompt tokens one at a time
 *      (engine/src/engine.c:306-501); this is the contraction those n_tokens
 *      op_matmul_q4_k / op_matmul_q6_k calls (engine/src/ops.c:266-314,
 *      361-404) add up to: y[t][r] = sum_k W[r][k] * x[t][k] for t <
 *      n_tokens, x fp32 [n_tokens][k], y fp32 [n_tokens][m].  Weights are
 *      dequantised to f16 tiles, each token row of x is scaled by a power of
 *      two (largest magnitude to [2^14, 2^15)) and rounded to f16, and the
 *      product runs f16 x f16 -> fp32 on tcgen05.mma (accumulators in TMEM),
 *      the scale put back exactly: results carry the f16 rounding of the
 *      inputs (2^-11 relative each).  dtype 12 (Q4_K) or
 *      SHK_DTYPE_Q6_K_PLANAR; row_stride 0 = dense rows.  Async on stream. ---- */
int shk_cuda_prefill_matmul(shk_ctx *ctx, uint32_t dtype, const void *w_dev, uint32_t row_stride,
                            const float *x_dev, float *y_dev, uint32_t m, uint32_t k, uint32_t n_tokens,
                            void *stream);
/* dequantise-matvec by dtype: 12 (Q4_K), 13 (Q5_K), 14 (GGUF Q6_K),
 * SHK_DTYPE_Q6_K_PLANAR, SHK_DTYPE_Q4_K_TILED or SHK_DTYPE_Q6_K_TILED;
 * row_stride 0 = dense rows (ignored for tiled weights; Q5_K rows must be
 * dense). */
int shk_cuda_matvec(shk_ctx *ctx, uint32_t dtype, const void *w_dev, uint32_t row_stride,
                    const float *x_dev, float *y_dev, uint32_t m, uint32_t k, void *stream);
/* Same contract as metal_matmul_q{4,6}k_vec: HOST weights/x/y, synchronous
 * (copies in, computes, copies out).  For callers that keep the reference's
 * host-resident layer buffers unchanged. */
int shk_cuda_matmul_q4k_vec_host(shk_ctx *ctx, const void *w_host, const float *x_host,
                                 float *y_host, uint32_t m, uint32_t k);
int shk_cuda_matmul_q6k_vec_host(shk_ctx *ctx, const void *w_host, const float *x_host,
                                 float *y_host, uint32_t m, uint32_t k);
int shk_cuda_matmul_q5k_vec_host(shk_ctx *ctx, const void *w_host, const float *x_host,
                                 float *y_host, uint32_t m, uint32_t k);

/* ---- op-level glue on device (engine/include/ops.h:9-38) ---- */
/* op_rmsnorm, n = 1 (engine/src/ops.c:195-214) */
int shk_cuda_rmsnorm(shk_ctx *ctx, const float *x_dev, const float *w_dev, float *y_dev,
                     uint32_t d, void *stream);
/* op_rope (engine/src/ops.c:216-238); in place */
int shk_cuda_rope(shk_ctx *ctx, float *qk_dev, uint32_t n_heads, uint32_t head_dim, uint32_t pos,
                  float rope_theta, void *stream);
/* SwiGLU of op_mlp_swiglu (engine/src/ops.c:491-496) */
int shk_cuda_swiglu(shk_ctx *ctx, const float *gate_dev, const float *up_dev, float *h_dev,
                    uint32_t n, void *stream);
/* op_embed for one token, Q4_K (12) or F16 (1) table (engine/src/ops.c:533-577) */
int shk_cuda_embed(shk_ctx *ctx, const void *table_dev, uint32_t dtype, uint32_t n_vocab,
                   uint32_t token, float *out_dev, uint32_t n_embd, void *stream);
/* first-index argmax (engine/src/engine.c:424-431); result to host.
 * n must be 1..0xFFFFFFFE (SHK_ARGMAX_NOALLOC_MAX_N below); else SHK_EINVAL. */
int shk_cuda_argmax(shk_ctx *ctx, const float *x_dev, uint32_t n, uint32_t *out_host);

/* ---- Q8_0 KV cache in HBM (engine/include/kv_cache.h:11-37).  Quantisation
 *      is bit-identical to q8_quantize_vec (engine/src/kv_cache.c:28-55). ---- */
struct shk_kv_config {
    uint32_t n_layers;
    uint32_t n_kv_heads;
    uint32_t head_dim; /* 64 or 128 */
    uint32_t block_size; /* kept for API parity; storage is per position */
    uint32_t max_seq_len; /* not capped at 2048 */
};
shk_kv *shk_cuda_kv_create(shk_ctx *ctx, const struct shk_kv_config *cfg);
void shk_cuda_kv_destroy(shk_kv *kv);
/* kv_cache_append (engine/src/kv_cache.c:130-155); k/v: n_kv*head_dim fp32 */
int shk_cuda_kv_append(shk_kv *kv, uint32_t layer, uint32_t pos, const float *k_dev,
                       const float *v_dev, void *stream);
/* kv_cache_append for positions start..start+n-1 in one launch, as the
 * reference's prefill loop appends them one by one (engine/src/engine.c:352-380
 * via forward_layer_view :133); k/v: n rows of n_kv*head_dim fp32 */
int shk_cuda_kv_append_range(shk_kv *kv, uint32_t layer, uint32_t start, uint32_t n,
                             const float *k_dev, const float *v_dev, void *stream);
/* kv_cache_read_range (engine/src/kv_cache.c:175-199): fp32 [pos][n_kv*hd] */
int shk_cuda_kv_read_range(shk_kv *kv, uint32_t layer, uint32_t start, uint32_t end,
                           float *k_dev, float *v_dev, void *stream);
/* raw 36-byte {float scale; int8 q[32]} blocks, reference order
 * [pos][n_kv*hd/32] -- for byte-exact comparisons */
int shk_cuda_kv_read_blocks(shk_kv *kv, uint32_t layer, uint32_t start, uint32_t end,
                            void *k_dev, void *v_dev, void *stream);
/* kv_cache_read_range + op_attention over positions [0, seq_len) fused on the
 * Q8_0 cache (engine/src/engine.c:137-158, engine/src/ops.c:406-461).  If
 * k_new_dev/v_new_dev are non-NULL they are first appended at seq_len-1. */
int shk_cuda_kv_attend(shk_kv *kv, uint32_t layer, const float *q_dev, const float *k_new_dev,
                       const float *v_new_dev, float *out_dev, uint32_t n_heads, uint32_t seq_len,
                       float scale, void *stream);
/* shk_cuda_kv_attend for n_seq sequences in one launch -- the KV
 * microbenchmark's batch of decode streams (no counterpart in the reference,
 * which decodes one sequence): sequence z appends to and attends cache layer
 * layer0 + z with q / out rows at z * n_heads * hd floats and k_new / v_new
 * rows at z * n_kv * hd; every sequence at seq_len.  Scratch for the split
 * partials grows on the first call of a larger n_seq (make that call outside
 * graph capture). */
int shk_cuda_kv_attend_batch(shk_kv *kv, uint32_t layer0, uint32_t n_seq, const float *q_dev,
                             const float *k_new_dev, const float *v_new_dev, float *out_dev,
                             uint32_t n_heads, uint32_t seq_len, float scale, void *stream);
/* kv_cache_clear / kv_cache_get_seq_len (engine/src/kv_cache.c:230-248) */
void shk_cuda_kv_clear(shk_kv *kv);
uint32_t shk_cuda_kv_seq_len(shk_kv *kv, uint32_t layer);

/* ---- paged K/V pools in 8 bits, shared by the requests of a batch.  No
 *      counterpart in the reference, which decodes one sequence from one cache
 *      (engine/include/kv_cache.h:5-37).  A pool is cut into blocks of
 *      block_tokens positions; a request holds the blocks that its block table
 *      lists, so requests of different lengths share one pool without gaps.
 *      Values are held in 8 bits with one fp32 scale per block and head (K and
 *      V apart): value = scale * byte.  Buffers belong to the caller; one
 *      struct shk_pages describes one layer's.
 *
 *      A step of a batch: shk_cuda_pages_release (blocks of the requests that
 *      ended) or shk_cuda_pages_truncate (of those that were cut short as well),
 *      shk_cuda_pages_assign (blocks, slots, positions of the new tokens), per layer shk_cuda_pages_append and shk_cuda_pages_attend, then
 *      shk_cuda_sample on the logits.  All of it is stream-ordered and reads
 *      lengths on the device only, so a captured step can be replayed.
 *
 *      Lengths, slots, positions and block ids are int32, and every array of
 *      them or of floats is 4-byte aligned (else SHK_EINVAL).  A bad value (a block
 *      id outside the pool, a position outside the table, a slot outside the
 *      pool) is left out and recorded: shk_cuda_check returns SHK_EDEVICE. ---- */
#define SHK_PAGES_I8 0u   /* signed integers -127..127 */
#define SHK_PAGES_E4M3 1u /* 8-bit floating point: 4 exponent, 3 mantissa bits, largest value 448 */
#define SHK_PAGES_MAX_SEQ 16384u
#define SHK_PAGES_MAX_ROWS 65535u
/* types of activations (ggml's codes) */
#define SHK_DTYPE_F32 0u
#define SHK_DTYPE_F16 1u
#define SHK_DTYPE_BF16 30u
struct shk_pages {
    void *k_dev, *v_dev;              /* [n_blocks][n_kv_heads][block_tokens][head_dim] bytes, 16-byte aligned */
    float *k_scale_dev, *v_scale_dev; /* [n_blocks][n_kv_heads] */
    uint32_t type;                    /* SHK_PAGES_* */
    uint32_t n_blocks;                /* n_blocks * block_tokens < 2^31 */
    uint32_t n_kv_heads;              /* at most 1024 */
    uint32_t head_dim;                /* 64 or 128 */
    uint32_t block_tokens;            /* 16, 32, 64, 128 or 256 */
};
/* Block tables and slots from lengths.  Request r holds have[r] tokens in the
 * blocks table[r][0 ..], have[r] / block_tokens of them rounded up, and gets add[r] more.  Requests are served in order:
 * their rows (one per new token) are laid out one request after the other, and
 * a new block of theirs is taken from the top of the free stack
 * free_dev[0 .. *n_free_dev).  Row i: slots[i] = block * block_tokens + place in
 * the block, pos[i] = position in the request, seq[i] = request.  Rows that no
 * token takes get -1 in all three.  A request is refused whole -- lens[r] =
 * have[r], its rows -1, no block taken -- when its tokens outgrow table_stride
 * blocks, its rows outgrow n_rows, or its blocks and those asked for by the
 * requests before it outgrow the free stack; rows are counted as if every
 * request before it had been served.  A row whose block id (of the table or the
 * free stack) lies outside the pool gets -1 in all three arrays as well, and so
 * does last[r] where it is the request's last one; the table gets -1 for such a
 * new block, and lens[r] and the counts are as if the id were good.  lens_dev may
 * be have_dev, and counts_dev may be n_free_dev.  One launch; async on stream. */
struct shk_pages_assign {
    uint32_t n_seq;        /* request slots: 1 .. SHK_PAGES_MAX_SEQ */
    uint32_t block_tokens; /* 16 .. 256, a power of two */
    uint32_t n_blocks;     /* blocks in the pool */
    uint32_t table_stride; /* block ids per table row */
    uint32_t n_rows;       /* rows laid out, at most 2^30 - 1 */
    const int32_t *have_dev, *add_dev; /* [n_seq] */
    int32_t *table_dev;                /* [n_seq][table_stride]: read for the blocks held, new ones written */
    const int32_t *free_dev;           /* [n_blocks], the stack; not changed */
    const int32_t *n_free_dev;         /* [1] its height */
    int32_t *lens_dev;                 /* [n_seq] out: tokens after the step */
    int32_t *counts_dev;               /* [3] out: free blocks left, rows taken, requests refused */
    int32_t *slots_dev, *pos_dev, *seq_dev; /* [n_rows] out */
    int32_t *last_dev;                 /* [n_seq] out: the request's last row (its next token's logits), or -1 */
};
int shk_cuda_pages_assign(shk_ctx *ctx, const struct shk_pages_assign *a, void *stream);
/* Gives the blocks of the requests with done[r] != 0 back: pushed on the free
 * stack in request and table order, lens[r] = 0 (have[r] for the others), the
 * new height to n_free_out_dev.  lens_dev may be have_dev, n_free_out_dev may be
 * n_free_dev.  Ids outside the pool are left out, the others close up (what
 * free_dev holds above the new height is of no account); a request whose have[r]
 * is negative or more than its table row holds keeps it and gives nothing back.
 * Where the stack would outgrow n_blocks (a block given back twice) nothing is
 * given back at all.  shk_cuda_check returns SHK_EDEVICE after each of these. */
int shk_cuda_pages_release(shk_ctx *ctx, uint32_t n_seq, uint32_t block_tokens, uint32_t n_blocks,
                           uint32_t table_stride, const int32_t *table_dev, const int32_t *done_dev,
                           const int32_t *have_dev, int32_t *lens_dev, int32_t *free_dev,
                           const int32_t *n_free_dev, int32_t *n_free_out_dev, void *stream);
/* Requests cut short, as after rejected draft tokens: r keeps its first keep[r]
 * tokens (all where keep[r] >= have[r], 0: as if it had ended), lens[r] =
 * min(keep[r], have[r]), and the blocks that hold none of them go back, like
 * shk_cuda_pages_release's; a negative keep[r] counts as a bad length.  lens_dev
 * may be have_dev or keep_dev.  shk_cuda_pages_assign takes a request's blocks
 * from have[r] alone: a length lowered in any other way loses the blocks behind
 * it.  The scales of a block that is kept stay what its dropped tokens made them. */
int shk_cuda_pages_truncate(shk_ctx *ctx, uint32_t n_seq, uint32_t block_tokens, uint32_t n_blocks,
                            uint32_t table_stride, const int32_t *table_dev, const int32_t *keep_dev,
                            const int32_t *have_dev, int32_t *lens_dev, int32_t *free_dev,
                            const int32_t *n_free_dev, int32_t *n_free_out_dev, void *stream);
/* Quantise-and-store n_tokens rows of K and V (dtype F32, F16 or BF16; row i at
 * i * row_stride elements, 0 = n_kv_heads * head_dim) at slots_dev[i]; a
 * negative slot is a padding row and is skipped.  Per block and head the scale
 * is max|x| / 127 (E4M3: / 448) over the tokens it has taken since its first
 * place was last written: a token that raises it has the block's earlier
 * places rounded again to the new scale.  Quotients are formed in fp32 and
 * rounded half to even; NaN counts for nothing and is stored as 0; an infinity
 * makes the scale infinite (the block then reads as NaN).  The rows of one
 * block must be consecutive in the call and rising by one, as
 * shk_cuda_pages_assign lays them out: a block's second run in one call is not
 * stored, and shk_cuda_check returns SHK_EDEVICE.  (The search for such runs grows
 * with the square of n_tokens: better several calls above 100000.)  Calls that
 * append to one block must be ordered (one stream).  Async on stream. */
int shk_cuda_pages_append(shk_ctx *ctx, const struct shk_pages *pages, uint32_t n_tokens, const void *k_dev,
                          const void *v_dev, uint32_t dtype, size_t row_stride, const int32_t *slots_dev,
                          void *stream);
/* The values at slots_dev[0 .. n_tokens) as fp32 rows of n_kv_heads * head_dim;
 * rows of negative slots are left as they were. */
int shk_cuda_pages_read(shk_ctx *ctx, const struct shk_pages *pages, uint32_t n_tokens, const int32_t *slots_dev,
                        float *k_dev, float *v_dev, void *stream);
/* Attention of n_rows query rows: row i belongs to request seq[i] (seq_dev NULL:
 * request i) and sees its positions 0 .. pos[i], so a decode row, the draft
 * rows of one request and the rows of a prompt all have the causal mask that
 * pos gives.  Query head h reads KV head h % n_kv_heads, as op_attention does
 * (engine/src/ops.c:423).  pos < 0: the row sees nothing and becomes zeros;
 * seq < 0: no row (padding), out left as it was.  q and out are dtype F32, F16
 * or BF16 rows of n_heads * head_dim, q_stride / out_stride elements apart (0 =
 * dense); out may not overlap q (rows of one stride may lie between one another,
 * with two strides the whole ranges count).  Sums and softmax in fp32; a
 * position's weight times its V scale enters the output to 2^-22 of itself or
 * 2^-39 of the row's largest such product, whichever is more.  Rows of one request
 * that follow one another read its blocks together; how many may is chosen from
 * n_rows and n_seq, so padding rows and idle request slots far beyond the live
 * ones make the call slower (up to 1.7 times).  What no row of the call
 * sees may hold anything; between a row's last position and that of a
 * neighbour in its request, E4M3 bytes have to be numbers, as shk_cuda_pages_append
 * writes them.  ws_dev:
 * shk_cuda_pages_attend_ws bytes, 16-byte aligned, contents of no account
 * before and after; calls that may run at the same time need one each. */
struct shk_pages_rows {
    uint32_t n_rows;  /* at most SHK_PAGES_MAX_ROWS */
    uint32_t n_heads; /* a multiple of n_kv_heads, at most 4096 */
    uint32_t dtype;
    const void *q_dev;
    void *out_dev;
    size_t q_stride, out_stride;
    const int32_t *seq_dev, *pos_dev; /* [n_rows] */
    const int32_t *table_dev;         /* [n_seq][table_stride] */
    uint32_t n_seq, table_stride;
    float scale;
    void *ws_dev;
    size_t ws_bytes;
};
/* 0 for heads or a head_dim that shk_cuda_pages_attend does not take. */
size_t shk_cuda_pages_attend_ws(uint32_t n_rows, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim);
int shk_cuda_pages_attend(shk_ctx *ctx, const struct shk_pages *pages, const struct shk_pages_rows *rows,
                          void *stream);

/* ---- sampling: one token per row of logits from given random numbers (the
 *      reference only takes the argmax, engine/src/engine.c:424-431).  Row i of
 *      the logits (dtype F32, F16 or BF16) is at i * row_stride elements (0 =
 *      n_vocab).  temperature, top_k, top_p, min_p: one value per row, or NULL
 *      for off.  u_dev: one number in [0, 1) per row.
 *       - weights w = exp((z - z_max) / T); T <= 0 or NaN: the first index of
 *         the maximum, as shk_cuda_argmax; NaN and -inf logits have weight 0;
 *       - top_k > 0: the k largest logits stay, equal ones by lower index;
 *       - top_p < 1: of those, from the largest down, each stays while the
 *         weights before it sum to less than top_p of them all (one always does);
 *       - min_p > 0: tokens with w < min_p go (w is 1 for the largest);
 *       - the first token, in index order, at which the running sum of the
 *         weights that stay exceeds u of their total.
 *      out_dev[i] = its index, prob_dev[i] (if not NULL) = its weight over that
 *      total.  A row without a logit above -inf gives SHK_SAMPLE_NONE and 0.
 *      Weights are summed as whole multiples of 2^-40: the same inputs give the
 *      same token on every run, and weights below 2^-40 count for nothing.
 *      Async on stream; no workspace. ---- */
#define SHK_SAMPLE_NONE 0xFFFFFFFFu
#define SHK_SAMPLE_MAX_VOCAB 262144u /* larger: SHK_EUNSUPPORTED */
int shk_cuda_sample(shk_ctx *ctx, const void *logits_dev, uint32_t dtype, uint32_t n_rows, uint32_t n_vocab,
                    size_t row_stride, const float *temperature_dev, const int32_t *top_k_dev,
                    const float *top_p_dev, const float *min_p_dev, const float *u_dev, uint32_t *out_dev,
                    float *prob_dev, void *stream);

/* ---- model: per-layer forward, embed, lm_head+argmax, captured decode step ---- */
struct shk_model_desc {            /* struct model_info (model_loader.h:66-74) + resident */
    uint32_t n_layers, n_embd, n_heads, n_kv_heads, head_dim, n_ff, n_vocab;
    float rope_theta;              /* 0 -> 10000, as engine/src/engine.c:86 */
    const void *tok_embd_dev;      /* token_embd, resident */
    uint32_t tok_embd_dtype;
    const void *output_dev;        /* output (lm_head), resident */
    uint32_t output_dtype;
};
struct shk_layer_desc {            /* struct layer_view (model_loader.h:28-56), DEVICE pointers */
    const float *attn_norm, *ffn_norm;
    const void *attn_q, *attn_k, *attn_v, *attn_o, *ffn_gate, *ffn_up, *ffn_down;
    uint32_t attn_q_dtype, attn_k_dtype, attn_v_dtype, attn_o_dtype;
    uint32_t ffn_gate_dtype, ffn_up_dtype, ffn_down_dtype;
    uint32_t row_stride_v, row_stride_down; /* 0 = dense rows; else padded row bytes */
};
shk_model *shk_cuda_model_create(shk_ctx *ctx, const struct shk_model_desc *desc, shk_kv *kv);
void shk_cuda_model_destroy(shk_model *m);
/* Registers device weights of a layer for the captured whole-token step. */
int shk_cuda_model_set_layer(shk_model *m, uint32_t layer, const struct shk_layer_desc *lv);
/* forward_layer_view (engine/src/engine.c:76-229) on device-resident weights:
 * hidden_dev (n_embd fp32) is updated in place; K/V appended at pos. */
int shk_cuda_forward_layer(shk_model *m, const struct shk_layer_desc *lv, uint32_t layer,
                           uint32_t pos, float *hidden_dev, void *stream);
/* op_embed(token) into the model's hidden state */
int shk_cuda_model_embed(shk_model *m, uint32_t token, void *stream);
/* lm_head on the raw residual (no final norm, engine/src/engine.c:403-422) and
 * first-index argmax.  logits_host may be NULL. */
int shk_cuda_model_lm_head(shk_model *m, uint32_t *token_host, float *logits_host, void *stream);
/* A token drawn from the logits of the model's last output head (shk_cuda_token_step
 * or shk_cuda_prefill with the next token wanted, shk_cuda_model_lm_head), as
 * shk_cuda_sample draws one, in place of that call's argmax.  u in [0, 1);
 * temperature <= 0 gives the argmax, top_k <= 0, top_p >= 1 and min_p <= 0 are
 * off.  *prob_host (may be NULL): the token's share of the weights that stayed.
 * Before the model's first output head the token is SHK_SAMPLE_NONE, its share 0.
 * Synchronous.  Single GPU (a tensor-parallel rank: SHK_EUNSUPPORTED). */
struct shk_sampling {
    float temperature;
    int32_t top_k;
    float top_p, min_p;
};
int shk_cuda_model_sample(shk_model *m, const struct shk_sampling *s, float u, uint32_t *token_host,
                          float *prob_host, void *stream);
float *shk_cuda_model_hidden(shk_model *m); /* device pointer to hidden[n_embd] */
/* One whole token through embed -> all layers (-> lm_head -> argmax when
 * want_next) as one captured CUDA graph.  token and pos come from the host;
 * the next token (and logits if logits_host != NULL) are copied back.  All
 * layers must be registered with shk_cuda_model_set_layer. */
int shk_cuda_token_step(shk_model *m, uint32_t token, uint32_t pos, int want_next,
                        uint32_t *next_host, float *logits_host);
/* Device-only decode steps: token and position stay on the device (argmax
 * feeds the next embed, position auto-increments).  Used for throughput. */
int shk_cuda_decode_steps(shk_model *m, uint32_t first_token, uint32_t first_pos, uint32_t n_steps,
                          void *stream);
int shk_cuda_model_token(shk_model *m, uint32_t *token_host); /* last argmax */
/* Batched prompt prefill: tokens[0..n) (host) at positions pos0.. run through
 * every layer as T = n rows at a time -- the projections on the tensor-core
 * matmul (shk_cuda_prefill_matmul: f16 operands, fp32 accumulation), RMSNorm,
 * RoPE, SwiGLU and residuals row-batched, the n K/V rows appended to the
 * Q8_0 cache in one launch per layer and every row's causal attention over
 * [0, pos0 + row] -- then the output head on the last row: its argmax to
 * *next_host (and its logits to logits_host when non-NULL).  The reference
 * feeds the prompt one token at a time (engine/src/engine.c:343-394); this is
 * the same computation with f16 rounding of the matmul inputs, so logits
 * differ from the token-by-token path by that rounding.  Weights must be
 * Q4_K or planar Q6_K (else SHK_EUNSUPPORTED: feed the prompt through
 * shk_cuda_token_step); single GPU. */
int shk_cuda_prefill(shk_model *m, const uint32_t *tokens_host, uint32_t n, uint32_t pos0,
                     uint32_t *next_host, float *logits_host, void *stream);
/* Timeline of the persistent decode kernel, for profiling (no counterpart in
 * the reference, whose CPU loop has no phases).  shk_cuda_model_trace_enable
 * (m, n) makes the following token_step / decode_steps launches record, on
 * CTA 0, %globaltimer (ns) at the start and at the arrival at / departure from
 * the grid barrier after each of the first n phases (n = 0 turns it off).
 * shk_cuda_model_trace_read copies up to cap values of the last launch
 * ([start, arrive_0, leave_0, arrive_1, ...]) and returns how many it wrote, or
 * a negative status.  Phases per token: embed, 5 per layer (QKV, attention, O,
 * gate/up, down), lm_head, argmax. */
int shk_cuda_model_trace_enable(shk_model *m, uint32_t n_phases);
int shk_cuda_model_trace_read(shk_model *m, uint64_t *out_host, uint32_t cap);
/* Profiling hook: enqueue one part of a registered layer's step at the device
 * position of the last step (part 0 RMSNorm+QKV+RoPE GEMV, 1 append+attention,
 * 2 O-proj+residual, 3 RMSNorm+gate/up+SwiGLU, 4 down+residual; 5 = lm_head
 * GEMV, layer ignored).  Returns the algorithmic bytes of that launch's
 * weights in *bytes_out (nullable). */
int shk_cuda_model_launch_part(shk_model *m, uint32_t layer, uint32_t part, void *stream,
                               uint64_t *bytes_out);

/* ---- layer streaming: pinned staging -> HBM on the context's copy stream
 *      (replaces the host-only prefetch ring, engine/src/prefetch.c:39-280) ---- */
/* Queue an async H2D copy of a staged layer blob into dst_dev and record the
 * completion event of `slot`.  Callable from the loader thread. */
int shk_cuda_layer_stage(shk_ctx *ctx, uint32_t slot, void *dst_dev, const void *pinned_src,
                         size_t bytes);
/* Strided variant: rows of src_row_bytes copied to rows of dst_row_bytes
 * (pads Q6_K rows to 16-byte multiples). */
int shk_cuda_layer_stage_rows(shk_ctx *ctx, uint32_t slot, void *dst_dev, size_t dst_row_bytes,
                              const void *pinned_src, size_t src_row_bytes, size_t rows);
/* General strided copy: `rows` runs of `width` bytes, src_pitch apart in the
 * pinned blob, to dst_pitch apart in HBM -- a tensor-parallel rank's column
 * shard of a matrix (its block range of every row) or its row range.  No
 * counterpart in the reference (it has no tensor parallelism). */
int shk_cuda_layer_stage_2d(shk_ctx *ctx, uint32_t slot, void *dst_dev, size_t dst_pitch,
                            const void *pinned_src, size_t src_pitch, size_t width, size_t rows);
/* Converts Q6_K rows just staged into dst_dev (rows x k elements, row_stride
 * bytes apart, 0 = dense) to the planar layout, in place, on the copy stream
 * after the slot's copies; the slot's commit covers it.  Callable from the
 * loader thread.  No counterpart in the reference. */
int shk_cuda_layer_stage_q6k_planar(shk_ctx *ctx, uint32_t slot, void *dst_dev, uint32_t rows, uint32_t k,
                                    uint32_t row_stride);
/* Marks the end of a slot's staging sequence (records its event). */
int shk_cuda_layer_commit(shk_ctx *ctx, uint32_t slot);
/* 1 if the slot's copies completed, 0 if still in flight (wait = 0), or block
 * until complete (wait != 0). */
int shk_cuda_layer_ready(shk_ctx *ctx, uint32_t slot, int wait);
/* Make `stream` wait (on the device) for the slot's copies. */
int shk_cuda_layer_wait(shk_ctx *ctx, uint32_t slot, void *stream);
/* Device-slot reuse (prefetcher_release, engine/src/prefetch.c:262-280): the
 * next staging into `slot` first waits, on the copy stream, for the work
 * queued on `stream` so far -- the kernels that read the slot's old layer. */
int shk_cuda_layer_release(shk_ctx *ctx, uint32_t slot, void *stream);

/* ---- failure detection.  No counterpart in the reference (its only device
 *      path is synchronous Metal).  Every device wait in this library is
 *      bounded; on expiry the kernel records a timeout and returns, and the
 *      next status check reports SHK_ETIMEOUT.  This launches one wait that
 *      nothing satisfies (an mbarrier that never completes) with a budget of
 *      budget_us microseconds (at most 1 s): it returns SHK_ETIMEOUT and the
 *      context stays usable. ---- */
int shk_cuda_selftest_wait_timeout(shk_ctx *ctx, uint32_t budget_us);

/* ---- tensor parallelism over the GPUs of one node: NCCL all-reduce over
 *      NVLink after the O and down projections (layout: Wq/Wk/Wv/
 *      gate/up split by output rows, Wo/down by input columns, KV heads local
 *      to a rank).  No counterpart in the reference (single device). ---- */
#define SHK_TP_ID_BYTES 128
/* Rank 0 creates the communicator id (returns its size); the caller passes
 * it to every rank, which then calls shk_cuda_tp_init before creating its
 * model.  NCCL is loaded at first use (libnccl.so.2). */
int shk_cuda_tp_unique_id(void *out, size_t cap);
int shk_cuda_tp_init(shk_ctx *ctx, int rank, int world, const void *id);
/* Ranks in the context's NCCL communicator (ncclCommCount): world after
 * shk_cuda_tp_init, 1 without one; negative on error.  No counterpart in the
 * reference (which has no tensor parallelism). */
int shk_cuda_tp_comm_size(shk_ctx *ctx);
/* This rank computes rows [o_lo, o_hi) of the O projection (its attn_o
 * weights have o_hi - o_lo rows; ranks that share attention heads split the
 * rows) and rows [v_lo, v_hi) of the output head (its output weights have
 * v_hi - v_lo rows).  The head is either replicated (0, n_vocab) or split in
 * equal slices in rank order (v_lo = rank * n_vocab / world); a split head's
 * argmax is merged over the ranks, and a logits copy to the host gathers the
 * slices first, so every rank must ask for logits on the same steps.
 * Default: all rows.  Call after shk_cuda_tp_init and before
 * shk_cuda_model_set_layer. */
int shk_cuda_model_set_tp_rows(shk_model *m, uint32_t o_lo, uint32_t o_hi, uint32_t v_lo, uint32_t v_hi);

/* Tensor-parallel all-reduce over NVLink peer memory instead of NCCL: the O
 * and down GEMVs send their partial output rows straight into every rank's
 * exchange buffer (plain peer stores) and raise a per-rank flag; the next
 * GEMV waits for the flags (bounded), adds the residual and the partials in
 * rank order and proceeds -- no collective kernel between them.  Setup, after
 * shk_cuda_model_set_tp_rows and before shk_cuda_model_set_layer: every rank
 * exports its buffer's IPC handle (64 bytes, returned size), the caller
 * gathers them in rank order and every rank imports the set together with
 * every rank's O rows (o_ranges: world x {o_lo, o_hi}).  The ranks must run
 * on separate GPUs of one node, one process per GPU (CUDA IPC).  NCCL is
 * still used for the vocabulary-split argmax.  No counterpart in the
 * reference. */
int shk_cuda_model_tp_p2p_export(shk_model *m, void *handle_out, size_t cap);
int shk_cuda_model_tp_p2p_import(shk_model *m, const void *handles, const uint32_t *o_ranges);

/* Tensor-parallel all-reduce over NVLink peer memory with the flags in the
 * data words, replacing the NCCL all-reduce after O and down: every rank
 * stores its partial row as 8-byte {value, step} words into every rank's
 * exchange buffer, then sums the ranks' rows from its own buffer in rank
 * order once each word carries the current step (bounded waits).  One small
 * kernel per all-reduce, inside the captured decode step.  Setup, after
 * shk_cuda_model_set_tp_rows and before the first token step: every rank
 * exports its buffer's IPC handle (64 bytes), the caller gathers them in rank
 * order and every rank imports the set.  One process per GPU of one node.  No
 * counterpart in the reference (which has no tensor parallelism). */
int shk_cuda_model_tp_ll_export(shk_model *m, void *handle_out, size_t cap);
int shk_cuda_model_tp_ll_import(shk_model *m, const void *handles);

/* ---- argmax without any device allocation.  No counterpart in the reference:
 *      it exists for callers that cannot call cudaMalloc (a sampler inside a
 *      host runtime that has already reserved the device's memory in its own
 *      pool, or code that holds only device pointers and a stream, no shk_ctx).
 *
 * Writes the first index of the maximum of x_dev[0..n) to *out_dev (device
 * memory), on `stream` (a cudaStream_t; NULL = the legacy default stream), on
 * the CURRENT device.  Same result as shk_cuda_argmax.  Asynchronous: read
 * *out_dev after the stream has been synchronised.
 *  - Scratch is a fixed 2304-byte array in the library's device image (block
 *    partials + merge ticket); every GPU that loads the library holds it until
 *    the process exits.  No cudaMalloc / cudaFree is called.
 *  - The first call in each CUDA context (one per device for runtime-API
 *    callers; a new one after cudaDeviceReset or under a caller's own driver
 *    context) looks up the array's device address in that context (set-up
 *    under a lock, cached by the context's unique id); make that first call
 *    before any stream capture.
 *  - All calls on a device share the array: calls whose kernels overlap on the
 *    GPU (e.g. on two streams at once) race and give wrong results.
 *  - n must be 1..SHK_ARGMAX_NOALLOC_MAX_N; larger or zero n returns
 *    SHK_EINVAL without launching anything. ---- */
#define SHK_ARGMAX_NOALLOC_MAX_N 0xFFFFFFFEu
int shk_cuda_argmax_noalloc(const float *x_dev, uint32_t n, uint32_t *out_dev, void *stream);

#ifdef __cplusplus
}
#endif
#endif
