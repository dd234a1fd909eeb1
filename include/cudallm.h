/*
 * cudallm.h: C ABI of the B200 (sm_100a) Llama-3.2-1B decode engine.
 *
 * Drop-in replacement for wasiqnauman/cudallm's include/cudallm/cudallm.h:1-62. Every symbol, struct
 * layout, return code and ownership rule of that header is kept, so its ctypes wrapper
 * (python/cudallm/engine.py:39-66) and its tests bind this library unchanged when CUDALLM_LIB points
 * at it. Entry points after the "additive" marker are new and change none of the originals.
 *
 * Conventions (reference src/capi/cudallm_capi.cpp:24-44): every entry point returns a CUDALLM_*
 * code (except destroy / default_options / pos / last_error); no C++ exception crosses the ABI;
 * the message of the last failure on the calling thread is returned by cudallm_last_error().
 * One engine per thread; engines own all device memory, callers own all host buffers.
 */
#ifndef CUDALLM_B200_CUDALLM_H
#define CUDALLM_B200_CUDALLM_H

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes: reference include/cudallm/cudallm.h:8-14. */
#define CUDALLM_OK 0
#define CUDALLM_ERR_INVALID_ARG 1
#define CUDALLM_ERR_IO 2
#define CUDALLM_ERR_FORMAT 3
#define CUDALLM_ERR_CUDA 4
#define CUDALLM_ERR_STATE 5
#define CUDALLM_ERR_INTERNAL 6

typedef struct cudallm_engine cudallm_engine;

/* Engine options, 24 bytes: reference include/cudallm/cudallm.h:18-25.
 * matvec_impl/attn_impl: 0 naive, 1 opt. fuse: 1 selects the fused decode path (the persistent
 * decode-step kernel when matvec and attention are both opt). cuda_graph: replay the step as a CUDA
 * graph. max_seq_len: 0 = the file header's value, else a positive multiple of 128 not above it.
 * matvec_rpb: 0 = default, else 1, 2, 4 or 8 = the most weight rows a consumer warp takes per tile. */
typedef struct {
    int matvec_impl;
    int attn_impl;
    int fuse;
    int cuda_graph;
    int max_seq_len;
    int matvec_rpb;
} cudallm_options;

/* Model description: reference include/cudallm/cudallm.h:27-32. weight_bytes = sum of the nbytes of
 * every tensor in the file, each counted once (the bytes one decode step streams). */
typedef struct {
    int weight_dtype; /* 1 bf16, 3 int8, 4 int4 */
    int hidden, inter, n_layers, n_heads, n_kv_heads, head_dim, vocab, max_seq_len, group_size;
    float rms_eps;
    unsigned long long weight_bytes;
} cudallm_config_info;

/* Replaces reference cudallm.h:34 (thread-local message of the last failure). */
const char* cudallm_last_error(void);
/* Replaces reference cudallm.h:35: fills opt, opt, fuse 1, graph 1, 0, 0. */
void cudallm_default_options(cudallm_options* out);
/* Replaces reference cudallm.h:36: loads a .cudallm file; *out = NULL on failure. */
int cudallm_create(const char* path, const cudallm_options* opts, cudallm_engine** out);
/* Replaces reference cudallm.h:37; NULL-safe. */
void cudallm_destroy(cudallm_engine* e);
/* Replaces reference cudallm.h:38. */
int cudallm_get_config(cudallm_engine* e, cudallm_config_info* out);
/* Replaces reference cudallm.h:39: position back to 0 (KV contents are overwritten as it advances). */
int cudallm_reset(cudallm_engine* e);
/* Replaces reference cudallm.h:40: host mirror of the position; -1 for a NULL engine. */
int cudallm_pos(cudallm_engine* e);
/* Replaces reference cudallm.h:41. token >= 0 is fed; -1 feeds the previous step's device argmax.
 * logits_out: host [vocab] or NULL; next_token_out: host or NULL. With both NULL the call does not
 * synchronise (steps queue asynchronously on the engine's stream). */
int cudallm_step(cudallm_engine* e, int token, float* logits_out, int* next_token_out);
/* Replaces reference cudallm.h:42. Never uses a CUDA graph; residuals_out: host [(n_layers+1)*hidden],
 * the residual stream after the embedding and after each layer. */
int cudallm_step_debug(cudallm_engine* e, int token, float* residuals_out, float* logits_out, int* next_token_out);

/* ---- single-kernel test hooks: host pointers in/out; each call allocates, uploads, runs on the
 * default stream, synchronises, downloads and frees (reference cudallm.h:44-56, cudallm_capi.cpp:179-316). */

/* Replaces reference cudallm.h:45-48. impl 0 naive (bf16, STORE, no norm), 1 opt. weight_dtype 1/3/4;
 * epilogue 0 STORE, 1 ADD (y += W x), 2 SWIGLU (y[r] = silu(g_r) u_r, rows/2 outputs). */
int cudallm_kernel_matvec(int impl, int weight_dtype, int epilogue, int fuse_norm, int rpb,
                          const void* w, unsigned long long w_bytes, const void* scales, unsigned long long scales_bytes,
                          const float* x, const float* norm_w, float eps,
                          float* y /* in/out (ADD reads it) */, int rows, int cols);
/* Replaces reference cudallm.h:49. */
int cudallm_kernel_rmsnorm(const float* x, const float* w, float eps, float* y, int n);
/* Replaces reference cudallm.h:50-52. Caches are fp16 bits [nkv][max_seq][hd]. */
int cudallm_kernel_rope_kv(int fused, float* qkv /* in/out */, const float* inv_freq, int pos,
                           unsigned short* k_cache, unsigned short* v_cache, int nh, int nkv, int hd, int max_seq);
/* Replaces reference cudallm.h:53-54. impl 1 requires max_seq % 128 == 0, nh == 4*nkv, hd == 64. */
int cudallm_kernel_attention(int impl, const float* q, const unsigned short* k_cache, const unsigned short* v_cache,
                             int ctx, float* out, int nh, int nkv, int hd, int max_seq);
/* Replaces reference cudallm.h:55. */
int cudallm_kernel_silu_mul(const float* gu, float* act, int inter);
/* Replaces reference cudallm.h:56. Lowest index wins ties. */
int cudallm_kernel_argmax(const float* logits, int n, int* out_idx);

/* ================================ additive (no counterpart in the reference ABI) ================ */

#define CUDALLM_KV_FP16 0
#define CUDALLM_KV_BF16 1

#define CUDALLM_PATH_AUTO 0       /* persistent decode-step kernel when fuse=1 and both impls are opt */
#define CUDALLM_PATH_PERSISTENT 1 /* force the persistent decode-step kernel (needs fuse=1, opt/opt) */
#define CUDALLM_PATH_PER_OP 2     /* one kernel per operation, as the reference sequences them */

/* Extended creation options. struct_size must be sizeof(cudallm_options_ex). */
typedef struct {
    int struct_size;
    int kv_dtype; /* CUDALLM_KV_FP16 (reference default, engine.cpp:51-52) or CUDALLM_KV_BF16 */
    int device;   /* CUDA device ordinal; -1 = the calling thread's current device */
    int path;     /* CUDALLM_PATH_* */
    int reserved[4];
} cudallm_options_ex;

/* Fills kv fp16, device -1, path auto. */
void cudallm_default_options_ex(cudallm_options_ex* out);
/* cudallm_create with extended options (ex may be NULL = defaults). */
int cudallm_create_ex(const char* path, const cudallm_options* opts, const cudallm_options_ex* ex, cudallm_engine** out);
/* Waits for every queued step; reports a device-side failure (e.g. a timed-out inter-block wait). */
int cudallm_synchronize(cudallm_engine* e);
/* Prompt prefill: feeds tokens[0..n) (host) at positions pos .. pos+n-1, with the results of n calls of
 * cudallm_step(e, tokens[i], NULL, NULL) up to fp32 summation order, 64 tokens per batched tensor-core step
 * (a batched engine with its own copy of the weights is created on the first call and writes this engine's
 * KV cache; int8 weights step the tokens through the decode path). Afterwards cudallm_pos advanced by n,
 * *next_token_out (or NULL) is the argmax after tokens[n-1], logits_out (host [vocab], or NULL) its logits,
 * and cudallm_step(e, -1, ...) continues from that argmax. n must fit in max_seq_len (else STATE).
 * Synchronises. No counterpart in the reference, which feeds prompts one cudallm_step at a time. */
int cudallm_prefill(cudallm_engine* e, const int* tokens, int n, float* logits_out, int* next_token_out);
/* Which decode path the engine runs: CUDALLM_PATH_PERSISTENT or CUDALLM_PATH_PER_OP. */
int cudallm_engine_path(cudallm_engine* e);
/* The engine's CUDA stream (a cudaStream_t) and device, so callers can order or time work against the
 * steps it enqueues; NULL / -1 for a NULL engine. */
void* cudallm_engine_stream(cudallm_engine* e);
int cudallm_engine_device(cudallm_engine* e);
/* Step tracing (persistent path only): enable = 1 makes every following step record, per CTA, the
 * %globaltimer value (ns) at each operation's dependency-wait begin / end, its end, and when the
 * producer warp starts streaming its weights; 0 turns it off. */
int cudallm_debug_trace(cudallm_engine* e, int enable);
/* Copies the last traced step: grid x slots per-CTA values followed by 256 x 5 stamps of 256 consecutive
 * tiles of CTA 0 (from the first tile of the weight operation the "trace_tile_op" knob names, by default the
 * lm_head); count >= grid*slots + 1280. *grid_out, *slots_out get the shape. Waits for queued work. */
int cudallm_debug_read_trace(cudallm_engine* e, unsigned long long* out, unsigned long long count, int* grid_out,
                             int* slots_out);
/* Sets a tuning or test knob of the persistent decode path by name; CUDALLM_ERR_INVALID_ARG for an unknown
 * name, a value out of range, or a per-op engine. Knobs: "wait_limit_ns" (bound of every inter-block wait of
 * the step, 1 .. 1e10; default 1e9; a step whose wait runs out returns CUDALLM_ERR_STATE and leaves the
 * position unchanged), "prefetch_tiles" (L2 prefetch distance of the weight stream, 0 .. 1024),
 * "whole_head_max_tiles" (contexts up to this many 64-token tiles attend with one block per KV head, longer
 * ones split each head's context over many blocks, 0 .. max_seq_len/64; default 6, int4 weights 8), "trace_tile_op" (weight operation whose tiles the trace stamps, 0 .. 64),
 * "stall_op" (for tests of the failure path: the blocks computing weight operation k, 1 .. 64, wait for an
 * input that is never written, so every such wait runs out after wait_limit_ns and the step fails with
 * CUDALLM_ERR_STATE; -1 = off, the default). */
int cudallm_debug_set(cudallm_engine* e, const char* knob, long long value);

/* Next-token rule of the following steps (no counterpart in the reference, which decodes greedily:
 * src/kernels/argmax.cu). temperature 0 (the default) = argmax, lowest index on ties. temperature > 0 =
 * sampling: the top_k largest logits (1 .. 64; 0 = 64; ties to the lower index) are weighted by
 * exp((logit - max) / temperature); the nucleus is the shortest prefix of them, in descending order, whose
 * weight reaches top_p (0 < top_p <= 1) of their total; the token is drawn from it with a uniform number
 * that depends only on (seed, position), so a rerun reproduces the tokens. The `next` output of
 * cudallm_step and the token fed by cudallm_step(e, -1, ...) are the drawn token; logits are unchanged.
 * Persistent decode path only (INVALID_ARG on a per-op engine with temperature > 0). */
int cudallm_set_sampling(cudallm_engine* e, float temperature, int top_k, float top_p, unsigned long long seed);

/* ---- batched decode (no counterpart in the reference, whose engine holds one sequence): up to 64
 * independent sequences decoded together on one GPU, one token each per step; every row runs the
 * reference engine's per-token sequence (src/engine/engine.cpp:181-237) on its own token, position and KV
 * cache, with the weight matvecs as tensor-core GEMMs (bf16 or int4 weights). Several GPUs: one batch engine per
 * device (device field), each on its own sequences; no communication between them. */
typedef struct cudallm_batch cudallm_batch;

typedef struct {
    int struct_size; /* sizeof(cudallm_batch_options) */
    int n_seq;       /* 1..64 */
    int max_seq_len; /* 0 = the file header's value, else a positive multiple of 128 not above it */
    int kv_dtype;    /* CUDALLM_KV_FP16 or CUDALLM_KV_BF16 */
    int device;      /* CUDA device ordinal; -1 = the calling thread's current device */
    int cuda_graph;  /* 1: replay the step as a CUDA graph */
    int attn_mode;   /* 0 choose by size; 1 one block per (KV head, sequence) streaming the context;
                        2 split over 64-token tiles, merged by a second kernel */
    int reserved[3];
} cudallm_batch_options;

/* Fills n_seq 64, max_seq_len 0, kv fp16, device -1, cuda_graph 1, attn_mode 0. */
void cudallm_default_batch_options(cudallm_batch_options* out);
/* Loads a .cudallm file (bf16 or int4 weights; int8 returns INVALID_ARG) for n_seq sequences; *out = NULL on failure. */
int cudallm_batch_create(const char* path, const cudallm_batch_options* opts, cudallm_batch** out);
/* NULL-safe. */
void cudallm_batch_destroy(cudallm_batch* e);
/* As cudallm_get_config; max_seq_len is the engine's. */
int cudallm_batch_get_config(cudallm_batch* e, cudallm_config_info* out);
/* seq in [0, n_seq): that sequence's position back to 0; seq = -1: every sequence. */
int cudallm_batch_reset(cudallm_batch* e, int seq);
/* Host mirror of sequence seq's position; -1 for a NULL engine or an index out of range. */
int cudallm_batch_pos(cudallm_batch* e, int seq);
/* One decode step of every sequence. tokens: host [n_seq], tokens[b] >= 0 is fed to sequence b, -1 feeds
 * b's previous argmax; NULL = all -1. next_out: host [n_seq] (each row's argmax, lowest index on ties) or
 * NULL; logits_out: host [n_seq][vocab] or NULL. With both outputs NULL the call does not synchronise.
 * Every sequence must have room (pos < max_seq_len), else CUDALLM_ERR_STATE and nothing runs. */
int cudallm_batch_step(cudallm_batch* e, const int* tokens, int* next_out, float* logits_out);
/* Waits for every queued step; reports a device-side failure. */
int cudallm_batch_synchronize(cudallm_batch* e);
/* Prompt prefill of sequence seq (engines of n_seq 64): tokens[0..n) at that sequence's positions pos ..
 * pos+n-1, 64 per batched step, every row of a step one position of that sequence. The other sequences keep
 * their positions and previous argmax. next_token_out / logits_out (host, or NULL) as in cudallm_prefill.
 * Synchronises. */
int cudallm_batch_prefill(cudallm_batch* e, int seq, const int* tokens, int n, float* logits_out, int* next_token_out);
/* The engine's CUDA stream (a cudaStream_t); NULL for a NULL engine. */
void* cudallm_batch_stream(cudallm_batch* e);
/* Tuning knobs of the batched step by name (CUDALLM_ERR_INVALID_ARG when unknown or out of range): "pdl"
 * (0/1: programmatic dependent launch between the step's kernels), "ksplit_qkv", "ksplit_wo",
 * "ksplit_gate_up", "ksplit_down" (K split of that GEMM, 1 .. min(16, k/64); int4 k/128). The next step
 * captures its graph again. _get reads them back, and "attn_stream" (1 = streaming attention in use). */
int cudallm_batch_debug_set(cudallm_batch* e, const char* knob, long long value);
int cudallm_batch_debug_get(cudallm_batch* e, const char* knob, long long* value_out);

/* Test hook of the batched path (no counterpart in the reference): tensor-core GEMM y[b][j] (+)= sum_k
 * (x[b][k] + x_lo[b][k]) * w[j][k] for b < batch (1..64), w [n][k], x and x_lo [batch][k] bf16 bits (x_lo
 * may be NULL = zeros; the engine passes an fp32 activation as its bf16 rounding plus the bf16 rounding of
 * the remainder), fp32 result, the 64-column K chunks split evenly over `ksplit` CTA rows (k a multiple of
 * 64, ksplit <= k / 64). epilogue 0 stores, 1 adds to y, 2 applies SwiGLU (y is [batch][n/2]: silu(gate) *
 * up, gate rows first). Host pointers; allocates, runs on the default stream and synchronises like the
 * other hooks. */
int cudallm_kernel_gemm(const unsigned short* w, const unsigned short* x, const unsigned short* x_lo, float* y, int n, int k,
                        int batch, int ksplit, int epilogue);

/* No counterpart in the reference. Split-K decode attention (the kernels behind
 * cudallm_kernel_attention impl 1) for callers that cannot allocate device memory: code whose device
 * memory is owned by another runtime's pool, or loops that must not enter the driver's allocator.
 * Every argument is caller-owned DEVICE memory: q [nh*hd] fp32, k_cache / v_cache [nkv][max_seq][hd]
 * fp16 bits (16-byte aligned), out [nh*hd] fp32; ctx in [1, max_seq]; stream a cudaStream_t (NULL = the
 * legacy default stream). The call only enqueues work on stream; it allocates nothing. The split-K
 * partials live in one fixed device array of 1.03 MiB that every GPU loading the library holds until
 * exit, so nh <= 32 and max_seq <= 8192 (and nh == 4*nkv, hd == 64, max_seq % 128 == 0); larger sizes
 * return CUDALLM_ERR_INVALID_ARG. All calls share that array and it keeps the last call's contents, so
 * calls whose GPU work overlaps (other streams or threads, same device) race: order them on one stream.
 * The first call on each device, with that device current, looks up the array's device address
 * (cudaGetSymbolAddress) and keeps it for the life of the process; make that first call before any stream
 * capture that includes this function. A cudaDeviceReset of that device invalidates the kept address:
 * call this function no more on a device that was reset while the library stayed loaded. */
int cudallm_attention_noalloc(const float* q, const unsigned short* k_cache, const unsigned short* v_cache, int ctx,
                              float* out, int nh, int nkv, int hd, int max_seq, void* stream);

/* ---- paged key-value cache and beam search (no counterpart in the reference, whose engine keeps one contiguous
 * cache and decodes greedily). Every pointer inside these argument structs is caller-owned DEVICE memory; the
 * calls only enqueue work on `stream` (a cudaStream_t of the current device, NULL = the legacy default stream),
 * allocate nothing and can be captured in a CUDA graph. Argument errors are INVALID_ARG and enqueue nothing.
 * What the host cannot see (lengths, tables, positions, parents) is bounded inside the kernels as stated below,
 * so no content of those arrays leads to an access outside of the caller's buffers.
 *
 * Workspaces: `workspace` points to at least cudallm_*_workspace_bytes() bytes, 256-byte aligned; its contents do not matter (but for
 * cudallm_beam_select's, see there). One may serve the cudallm_paged_* calls one after the other on one stream; calls that may overlap (on
 * other streams, or from other host threads: a call may be two launches) need their own. */

#define CUDALLM_BEAM_COUNTER_BYTES 16384

#define CUDALLM_X_FP32 0
#define CUDALLM_X_FP16 1
#define CUDALLM_X_BF16 2

/* A pool of pages: k and v are [n_layers][n_pages][n_kv_heads][page_size][head_dim] with the strides below (in
 * elements, the same for both, multiples of 8; head_dim is contiguous), 16-byte aligned. head_dim: a multiple of 8,
 * 8 .. 256. A table row lists the pages of one sequence's tokens 0 .. page_size-1, page_size .. and so on; an entry
 * outside [0, n_pages) holds no page: attention treats its tokens as masked, append stores nothing there. */
typedef struct {
    int struct_size; /* sizeof(cudallm_pages) */
    int kv_dtype;    /* CUDALLM_KV_FP16 or CUDALLM_KV_BF16 */
    int n_layers, n_pages, n_kv_heads, page_size, head_dim, reserved;
    void* k;
    void* v;
    long long layer_stride, page_stride, head_stride, token_stride;
} cudallm_pages;

/* Attention of one new token per sequence over its pages: out[b][h] = softmax_t(scale q.k_t) v over the cached
 * positions max(0, lens[b] - window) <= t < lens[b] (window 0: all; lens outside [0, table_width * page_size] are
 * clamped to it) whose page exists; n_heads / n_kv_heads query heads share a key head. lse (or NULL): the natural
 * logarithm of the sum of the exponentials. No position left: out 0, lse -inf; a score that is not a number: out and
 * lse of its head are not numbers either. Scores, statistics and sums are fp32.
 * q [n_seq][n_heads][head_dim] has its own strides, out and lse are contiguous; out has q's type; out and
 * lse must not overlap the inputs or each other. Values in unused slots of a page do not matter; keys and values of used ones must be finite. */
typedef struct {
    int struct_size; /* sizeof(cudallm_attend_args) */
    int layer, x_dtype, n_seq, n_heads, table_width, window;
    float scale;
    const void* q;
    long long q_seq_stride, q_head_stride; /* elements */
    const int* tables;                     /* [n_seq][table_width] */
    long long table_stride;                /* elements */
    const int* lens;                       /* [n_seq] */
    void* out;                             /* [n_seq][n_heads][head_dim] */
    float* lse;                            /* [n_seq][n_heads] or NULL */
    void* workspace;
    unsigned long long workspace_bytes;
} cudallm_attend_args;

int cudallm_paged_attend(const cudallm_pages* pages, const cudallm_attend_args* args, void* stream);
/* Workspace of cudallm_paged_attend for any arguments (a constant). */
unsigned long long cudallm_attend_workspace_bytes(void);

/* Rotary positions of n_tokens new tokens: q_out = rotated q (may be q itself); rotated k and v are stored in the
 * slots of their positions. Token i belongs to table row rows[i] (rows NULL: row i) at positions[i]. Pair j < rotary
 * / 2 of a head turns by the angle (float)position * inv_freq[j], rounded to fp32 as in the decode step, with cos and
 * sin multiplied by `factor`; the pair is dims (j, j + rotary / 2), or (2j, 2j + 1) with interleaved != 0; dims from
 * `rotary` on are copied. A negative position is padding: q_out is 0 there and nothing is stored; nothing is stored
 * either for a row outside [0, n_rows), a position beyond the table or an entry without a page. Two tokens of one call
 * must not share a slot. rotary 0 stores without rotation. q may be NULL (keys and values only). q_out must not overlap any
 * other input (heads of one packed projection may lie between each other), nor q, k and v the pages. */
typedef struct {
    int struct_size; /* sizeof(cudallm_append_args) */
    int layer, x_dtype, n_tokens, n_heads, n_rows, table_width, rotary, interleaved;
    float factor;
    const void* q;
    const void* k;
    const void* v;
    long long q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    const float* inv_freq; /* [rotary / 2] */
    const int* positions;  /* [n_tokens] */
    const int* rows;       /* [n_tokens] or NULL */
    const int* tables;     /* [n_rows][table_width] */
    long long table_stride;
    void* q_out;           /* [n_tokens][n_heads][head_dim], strides below */
    long long out_token_stride, out_head_stride;
} cudallm_append_args;

int cudallm_paged_append(const cudallm_pages* pages, const cudallm_append_args* args, void* stream);

/* The next step's sequences: row i of tables_out continues row parents[i] of tables (a parent outside [0, n_rows):
 * row i is empty, which is how sequences are freed). Full pages are shared. The first child (lowest i) of a
 * parent also takes over the parent's pages from the first not full one on, if no other row refers to that one; any
 * other child gets a page of its own with a copy of the tokens in that page, in every layer. Then every row gets the
 * pages that `room` more tokens need. New pages are the lowest-numbered ones with refs 0, handed out in row order;
 * refs_out counts each page's references after the call (references that are not in `tables` stay counted).
 * A row's entries end at the first one without a page at or after its full pages. lens are clamped to
 * [0, table_width * page_size]. *missing = how many pages were wanted and not found (0 = success); their entries are
 * -1. The inputs stay as they are (outputs must not overlap them), so after a shortage the caller frees rows and calls
 * again on the same inputs. Layers' pages with refs > 0 are not written. */
typedef struct {
    int struct_size; /* sizeof(cudallm_fork_args) */
    int n_rows, n_out, table_width, room, reserved;
    const int* tables; /* [n_rows][table_width] */
    long long table_stride;
    const int* lens;    /* [n_rows] */
    const int* refs;    /* [n_pages] */
    const int* parents; /* [n_out] */
    int* tables_out;    /* [n_out][table_width] */
    long long table_out_stride;
    int* lens_out; /* [n_out] */
    int* refs_out; /* [n_pages] */
    int* missing;  /* [1] */
    void* workspace;
    unsigned long long workspace_bytes;
} cudallm_fork_args;

int cudallm_paged_fork(const cudallm_pages* pages, const cudallm_fork_args* args, void* stream);

/* Moves the *live pages with refs > 0 to the front of the pool: the k-th lowest unused page among the first *live takes
 * content (all layers), references and table entries of the k-th lowest used page after them. Table entries without a
 * page become -1. tables and refs stay as they are (outputs must not overlap them); pages from *live on may be
 * given back or reused afterwards. */
typedef struct {
    int struct_size; /* sizeof(cudallm_compact_args) */
    int n_rows, table_width, reserved;
    const int* tables;
    long long table_stride;
    const int* refs; /* [n_pages] */
    int* tables_out;
    long long table_out_stride;
    int* refs_out; /* [n_pages] */
    int* live;     /* [1] */
    void* workspace;
    unsigned long long workspace_bytes;
} cudallm_compact_args;

int cudallm_paged_compact(const cudallm_pages* pages, const cudallm_compact_args* args, void* stream);
/* Workspace of cudallm_paged_fork and cudallm_paged_compact for pools of n_pages pages and calls of up to `rows`
 * rows (the larger of n_rows and n_out); 0 for sizes that the calls refuse. */
unsigned long long cudallm_pages_workspace_bytes(int n_pages, int rows);

/* Beam search's selection. Candidate (w, t) of group g: scores[g][w] + (x[t] - logsumexp(x)) with x = row g * beams +
 * w of logits, or, where finished[g][w] != 0 (finished may be NULL), x = 0 at eos and -inf elsewhere. A candidate that
 * is not a number counts as -inf. The `keep` best of each group, in order: larger candidate, then lower beam, then
 * larger logit (one that is not a number: -inf), then lower token. out_parents are rows of logits (as
 * cudallm_paged_fork takes them). beams 1 .. 64, keep 1 .. 64 and at most beams * vocab, vocab at most 2^24. Outputs
 * must not overlap inputs or each other, but out_scores may be scores where keep equals beams. */
typedef struct {
    int struct_size; /* sizeof(cudallm_beam_args) */
    int x_dtype, n_groups, beams, keep, vocab, eos, reserved;
    const void* logits; /* [n_groups * beams][vocab] */
    long long row_stride;
    const float* scores;  /* [n_groups][beams] */
    const int* finished;  /* [n_groups][beams] or NULL */
    float* out_scores;    /* [n_groups][keep] */
    int* out_parents;     /* [n_groups][keep] */
    int* out_tokens;      /* [n_groups][keep] */
    void* workspace;
    unsigned long long workspace_bytes;
} cudallm_beam_args;

int cudallm_beam_select(const cudallm_beam_args* args, void* stream);
/* Workspace of cudallm_beam_select for up to `rows` = n_groups * beams rows of up to vocab logits; 0 for sizes that
 * the call refuses. Unlike the others' it must have its first CUDALLM_BEAM_COUNTER_BYTES bytes zero before the first call with
 * it; every call leaves them zero. So it is not shared with the calls above. */
unsigned long long cudallm_beam_workspace_bytes(int rows, int vocab, int keep);

#ifdef __cplusplus
}
#endif

#endif /* CUDALLM_B200_CUDALLM_H */
