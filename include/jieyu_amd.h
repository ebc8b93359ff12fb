/*
 * jieyu_amd.h — C ABI of the MI355X (gfx950) decode path: HBM-resident
 * weights and int8 KV cache, hand-written HIP kernels, one GPU.
 *
 * These entry points are the device-resident counterparts of jieyu's
 * model_libs forward-step interface.  All take plain pointers and sizes, return
 * an int status (0 / count on success, -1 on error) or a handle (NULL on
 * error); jyhip_last_error() gives the calling thread's last error text.  No
 * C++ exception crosses this boundary.
 *
 * Arithmetic: every kernel reproduces the reference CPU path's operation order
 * and rounding, so outputs are bit-identical to jieyu's AVX2+FMA build on the
 * same inputs (token ids, KV cache bytes, hidden states).
 */
#ifndef JIEYU_AMD_H
#define JIEYU_AMD_H

#include <stddef.h>
#include <stdint.h>

#include "jieyu_model.h"

#ifdef __cplusplus
extern "C" {
#endif

#define JYHIP_API __attribute__((visibility("default")))

typedef struct jyhip_model jyhip_model;
typedef struct jyhip_kv jyhip_kv;

/* token_cb of libs/model_libs/generate.h:8 — return nonzero to stop */
typedef int (*jyhip_token_cb)(int id, void* ud);

typedef struct jyhip_stats {
    double prefill_ms;      /* prompt forward + first token, device time */
    double decode_ms;       /* every later token, device time             */
    int prompt_len;
    int decoded;            /* tokens produced after the first            */
    double upload_ms;       /* host->device weight copy + repack (model)  */
} jyhip_stats;

/* Thread-local text of the last error ("" when none). */
JYHIP_API const char* jyhip_last_error(void);
/* Number of visible HIP devices (0 when none; never an error). */
JYHIP_API int jyhip_device_count(void);
/* Select the device used by subsequent calls of this thread. */
JYHIP_API int jyhip_set_device(int device);

/* Upload a model and precompute its RoPE table for positions [0, max_seq).
 * Mirrors what jieyu's bind_model + RoPETable::init produce
 * (libs/model_libs/pipeline.h:63-153, libs/date_libs/date.h:52-66); 2-D weights
 * must all be JY_Q8_0 or all JY_F32. */
JYHIP_API jyhip_model* jyhip_model_upload(const jy_model_desc* m, int max_seq);
JYHIP_API void jyhip_model_free(jyhip_model* model);
/* Arithmetic mode of a model's kernels (no counterpart in the reference).
 * JYHIP_MODE_EXACT (the default) reproduces the reference's operation order and rounding
 * bit for bit.  The other bits trade that for speed where the specification allows a
 * tolerance (per-layer fp32 hidden states within 1e-3 relative, identical greedy ids):
 *   JYHIP_MODE_SPLIT_ATTN  decode attention split across workgroups over the keys
 *                          (flash-decoding): exact int8 quantisation and int32 q.k, the
 *                          softmax sum and p.v accumulated per slice and merged; up to
 *                          1024 keys one kernel whose workgroups each take all the keys
 *                          and 16 output dims (the sum and p.v per wave, merged in the
 *                          workgroup); prompt rows in the same arithmetic, one workgroup
 *                          per kv head and row;
 *   JYHIP_MODE_SPLIT_MV    decode Q8_0 matvecs of fewer than JYHIP_SPLIT_MV_ROWS rows with
 *                          each row's dot split across waves; larger matrices keep the exact
 *                          kernel's dot order, which measured faster there (e.g. 4096 x
 *                          14336: 15.7 vs 18.9 us; 896 x 4864: 7.2 vs 5.1 us the other way);
 *                          both apply the RMSNorm scale after the dot (linearity);
 *   JYHIP_MODE_MFMA_PREFILL Q8_0 prompt GEMMs (m > 1) on the matrix cores: each activation
 *                          row scaled by a power of two and split into fp16 high + low parts
 *                          (22 significant bits), int8 weights exact in fp16, one fp32 MFMA
 *                          sum per 32-weight block times its scale.  Enabling it builds a
 *                          second copy of every layer's Q8_0 matrices in the matrix-core
 *                          operand order (about 1.13 bytes per weight; kept until the model
 *                          is freed); other weight types keep the exact tiles.
 * Int8 KV bytes and ids are the reference's wherever the fp32 values they come from are. */
#define JYHIP_MODE_EXACT 0
#define JYHIP_MODE_SPLIT_ATTN 1
#define JYHIP_MODE_SPLIT_MV 2
#define JYHIP_MODE_MFMA_PREFILL 4
#define JYHIP_MODE_FAST (JYHIP_MODE_SPLIT_ATTN | JYHIP_MODE_SPLIT_MV | JYHIP_MODE_MFMA_PREFILL)
#define JYHIP_SPLIT_MV_ROWS 2048
/* With both split bits: each decode row of every layer (and, in a session's greedy step, the
 * head) as one persistent kernel whose workgroups hand activations to each other through
 * grid barriers, instead of about six kernels per layer.  Same arithmetic as the split
 * forms; opt-in (measured slower than the separate kernels at the benchmark shapes). */
#define JYHIP_MODE_PERSIST 8
#define JYHIP_MODE_ALL (JYHIP_MODE_SPLIT_ATTN | JYHIP_MODE_SPLIT_MV | JYHIP_MODE_MFMA_PREFILL | JYHIP_MODE_PERSIST)
/* Set the mode (a combination of the bits above) for later calls on the model; sessions
 * capture their decode graphs again after a change.  Returns 0 / -1. */
JYHIP_API int jyhip_model_set_mode(jyhip_model* model, int mode);
JYHIP_API int jyhip_model_mode(const jyhip_model* model);

/* Bytes of 2-D weights (incl. lm_head) one decode step streams. */
JYHIP_API size_t jyhip_model_weight_bytes(const jyhip_model* model);
JYHIP_API double jyhip_model_upload_ms(const jyhip_model* model);

/* __KVcache::init (libs/date_libs/date.h:99-111): zero-filled int8 K/V and fp32
 * scales for num_layers x max_seq x num_kv_heads x head_dim. */
JYHIP_API jyhip_kv* jyhip_kv_create(const jyhip_model* model, int max_seq);
JYHIP_API void jyhip_kv_free(jyhip_kv* kv);
JYHIP_API int jyhip_kv_len(const jyhip_kv* kv);
JYHIP_API int jyhip_kv_set_len(jyhip_kv* kv, int current_len);
/* Copy positions [pos0, pos0+npos) of one layer in jieyu's host layout:
 * k, v int8 [npos][num_kv_heads][head_dim]; ks, vs float [npos][num_kv_heads]. */
JYHIP_API int jyhip_kv_write(jyhip_kv* kv, int layer, int pos0, int npos, const int8_t* k, const float* ks,
                             const int8_t* v, const float* vs);
JYHIP_API int jyhip_kv_read(const jyhip_kv* kv, int layer, int pos0, int npos, int8_t* k, float* ks, int8_t* v,
                            float* vs);

/* forward_cached (libs/model_libs/forward.h:47-96).  X: host [seq][hidden], the
 * embeddings of positions [start_pos, start_pos+seq) on entry, the final-normed
 * hidden states on exit.  layer_out (optional, host [num_layers][seq][hidden])
 * receives X after every layer.  Sets the cache length to start_pos+seq. */
JYHIP_API int jyhip_forward_cached(jyhip_model* model, jyhip_kv* kv, float* X, int seq, int start_pos,
                                   float* layer_out);

/* The same with the hidden states to `out` (host [seq][hidden], X itself or apart from it),
 * for a caller that keeps X or would copy it only to have it overwritten. */
JYHIP_API int jyhip_forward_cached_to(jyhip_model* model, jyhip_kv* kv, const float* X, float* out, int seq,
                                      int start_pos, float* layer_out);

/* Bytes of the static per-GPU workspace of jyhip_forward_cached_noalloc. */
#define JYHIP_NOALLOC_SCRATCH_BYTES (16u << 20)

/* jyhip_forward_cached (layer_out aside) without any device allocation.  It has no
 * counterpart in the reference: it is for callers that cannot allocate device memory
 * (tight serving loops, harnesses that forbid hipMalloc).  Like jyhip_forward_cached it
 * copies X from and back to the host and waits for the model's stream, so it cannot be
 * recorded into a caller's HIP graph: it allocates nothing, it is not capturable.  The
 * calling thread copies the rows itself, and nothing is allocated on the host for them (they
 * go through the model's pinned memory once a jyhip_forward_cached call of as many rows has
 * made it).
 * Same arguments, checks and results as jyhip_forward_cached with layer_out == NULL.
 * Its workspace is one static array of JYHIP_NOALLOC_SCRATCH_BYTES in each GPU's memory,
 * held until the process ends; a call whose rows and keys need more (a long prompt, a
 * long context) fails with an error that names the size.  Every call on a GPU shares
 * that GPU's array: calls that overlap on one GPU race. */
JYHIP_API int jyhip_forward_cached_noalloc(jyhip_model* model, jyhip_kv* kv, float* X, int seq, int start_pos);

/* generate / generate_cached (libs/model_libs/generate.h:9-112).  kv == NULL
 * uses a private max_seq cache.  Returns the sequence length written to
 * out_ids (prompt + generated), 0 for an empty / too long prompt, -1 on error.
 * out_ids needs max_seq entries.  logits_out (optional, [vocab_size]) receives
 * the logits of the last step. */
JYHIP_API int jyhip_generate(jyhip_model* model, jyhip_kv* kv, const int* prompt_ids, int prompt_len,
                             const int* eos_ids, int num_eos, int max_seq, int max_new, float temperature,
                             float repetition_penalty, int* out_ids, jyhip_token_cb cb, void* cb_ud,
                             float* logits_out, jyhip_stats* stats);

/* The same generation driven step by step (no counterpart in the reference; the
 * decode loop of generate_cached, generate.h:39-87, split so a caller can time
 * or interleave steps).  begin runs the prompt and picks the first token;
 * step produces up to n more (returns how many, 0 when finished); ids copies the
 * sequence so far.  begin returns a finished session (len = what generate()
 * would return) when the prompt is empty/too long or max_new <= 0.  A model holds
 * one generation's token ids and length on the device: once another session (or
 * jyhip_generate) begins on the same model, step on the earlier session returns -1
 * with an error.  forward_cached calls between steps are allowed. */
typedef struct jyhip_session jyhip_session;
JYHIP_API jyhip_session* jyhip_session_begin(jyhip_model* model, jyhip_kv* kv, const int* prompt_ids,
                                             int prompt_len, const int* eos_ids, int num_eos, int max_seq,
                                             int max_new, float temperature, float repetition_penalty);
/* A generation over a cache that already holds kv's current length (c) positions of
 * ids[0 .. n_ids): ids[c .. n_ids) run as one chunk at start_pos c, as forward_cached
 * does (libs/model_libs/forward.h:95), then decoding continues as in begin; the
 * repetition penalty covers only the tokens generated here.  Needs 0 <= c < n_ids.
 * The reference has no such entry (generate_cached, generate.h:31, always starts the
 * cache at 0); it serves decoding after a cache filled by other means (long-context
 * measurement, a conversation's earlier turns). */
JYHIP_API jyhip_session* jyhip_session_resume(jyhip_model* model, jyhip_kv* kv, const int* ids, int n_ids,
                                              const int* eos_ids, int num_eos, int max_seq, int max_new,
                                              float temperature, float repetition_penalty);
JYHIP_API int jyhip_session_step(jyhip_session* s, int n);
JYHIP_API int jyhip_session_remaining(const jyhip_session* s);
JYHIP_API int jyhip_session_len(const jyhip_session* s);
JYHIP_API int jyhip_session_ids(const jyhip_session* s, int* out, int cap);
JYHIP_API int jyhip_session_stats(jyhip_session* s, jyhip_stats* stats);
/* Diagnostics of a session's captured decode graph `which` (0: the graph for lengths past
 * the short-context threshold, 1: up to it); no counterpart in the reference.  Each graph is
 * checked when it is captured (kernel nodes only, one dependency chain, launch shapes within
 * the device's limits, every device buffer the step can address a live allocation on the
 * model's device) and before each jyhip_session_step (no such buffer replaced since capture).
 * Writes info[0] = nodes, info[1] = edges, info[2] = buffers checked; returns 1, 0 when that
 * graph has not been captured, -1 on error (a failed check). */
JYHIP_API int jyhip_session_graph_info(const jyhip_session* s, int which, long long* info);
JYHIP_API void jyhip_session_end(jyhip_session* s);

/* Isolated Q8_0 matvec (decode kernel): y[n] = W[n][:] . x for a [rows][cols/32]x34
 * jieyu matrix.  jyhip_q8_upload keeps `copies` identical device copies so timed
 * runs can rotate through more bytes than the 256 MiB last-level cache. */
typedef struct jyhip_q8mat jyhip_q8mat;
JYHIP_API jyhip_q8mat* jyhip_q8_upload(const void* w, int rows, int cols, int copies);
JYHIP_API void jyhip_q8_free(jyhip_q8mat* m);
JYHIP_API int jyhip_q8_matvec(jyhip_q8mat* m, const float* x, float* y);
/* jyhip_q8_matvec's kernel: JYHIP_MODE_EXACT (the default) or with JYHIP_MODE_SPLIT_MV the
 * split-dot form at any size; with JYHIP_MODE_MFMA_PREFILL jyhip_q8_gemm runs the matrix-core kernel
 * (the first such call builds its copies of the matrix).  Returns 0 / -1. */
JYHIP_API int jyhip_q8_set_mode(jyhip_q8mat* m, int mode);
/* Time `iters` launches (rotating copies) with HIP events on the launch stream:
 * *avg_us = mean kernel-to-kernel time per launch.  variant 0 is the plain
 * matvec; variant 1 is the decode step's gate/up launch of the same kernel
 * (RMSNorm over x, SwiGLU epilogue over interleaved row pairs); variants 2 and 3
 * are the same two launches of the split-dot kernel (JYHIP_MODE_SPLIT_MV); variant 4 is
 * the gate/up launch of the first kernel with the RMSNorm applied after the dot, the form
 * JYHIP_MODE_SPLIT_MV gives the matrices it leaves in the 32-lane order. */
JYHIP_API int jyhip_q8_matvec_time(jyhip_q8mat* m, const float* x, int variant, int iters, double* avg_us);
/* C[mr][rows] = A[mr][cols] W^T (row-major fp32) through the prompt GEMM of the
 * matrix's mode: the exact tiles, or with JYHIP_MODE_MFMA_PREFILL the matrix-core kernel
 * (the generic m > 1 matmul of libs/matmul_libs/matmul_q.h:145-161).  Returns 0 / -1. */
JYHIP_API int jyhip_q8_gemm(jyhip_q8mat* m, int mr, const float* A, float* C);
/* Mean device time in microseconds of `iters` such GEMMs (A uploaded once, the launches
 * cycling through the matrix's copies), the activation split included.  Returns 0 / -1. */
JYHIP_API int jyhip_q8_gemm_time(jyhip_q8mat* m, int mr, const float* A, int iters, double* avg_us);

/* One weight matrix of any bound type in HBM: matmul_w (libs/model_libs/wmat_kernel.h:9-16)
 * with B = w, n output rows, k inputs (f32 / f16 [k][n]; Q8_0 / k-quants [n][k/block]).
 * jyhip_wmat_matmul computes C[m][n] = A[m][k] x B from host buffers in the
 * reference's order for w's type: m == 1 the decode kernel (dot_row_avx2 for
 * quantized rows, matmul_q.h:111-143), m > 1 the prompt GEMM (:145-161; dense
 * [k][n]: the fma chain of matmul.h / matmul_f16.h).  `copies` device copies let
 * jyhip_wmat_time rotate through more bytes than the last-level cache: it times
 * `iters` decode launches with HIP events on the launch stream (mean us). */
typedef struct jyhip_wmat jyhip_wmat;
JYHIP_API jyhip_wmat* jyhip_wmat_upload(const jy_wmat* w, int n, int k, int copies);
JYHIP_API void jyhip_wmat_free(jyhip_wmat* w);
JYHIP_API int jyhip_wmat_matmul(jyhip_wmat* w, int m, const float* A, float* C);
JYHIP_API int jyhip_wmat_time(jyhip_wmat* w, const float* x, int iters, double* avg_us);

/* ---- Operators of a decode step over several sequences at once: a paged
 * key/value cache written and read back, attention of one new token per sequence over it, and
 * sampling.  The reference decodes one sequence at a time over a contiguous int8 cache
 * (libs/date_libs/date.h:89-147, libs/model_libs/attention/attention_q8.h:12-184) and samples
 * by temperature alone on the host (libs/model_libs/generate.h:36, :50-77); these have no
 * counterpart there.
 *
 * All buffers are the caller's and in device memory.  Calls enqueue work on `stream` (a
 * hipStream_t, NULL for the device's default stream) and return without waiting; they allocate
 * nothing and can be recorded into a HIP graph.  A call's buffers, its workspace among them,
 * have to stay as they are until its work is done, and two calls that may run at the same time
 * need a workspace each.  Status 0, or -1 with the reason in jyhip_last_error(); a refused call
 * has enqueued nothing.  `device` is the device that the buffers are on; a stream of another
 * device is refused. */

/* element types */
enum { JYHIP_T_F32 = 0, JYHIP_T_F16 = 1, JYHIP_T_BF16 = 2, JYHIP_T_I8 = 3, JYHIP_T_I4 = 4 };

/* One layer's pool of pages, `page_size` positions each:
 *   k, v              [num_pages][num_kv_heads][page_size][head_dim] of `type`
 *   k_scale, v_scale  fp32 [num_pages][num_kv_heads][page_size] with JYHIP_T_I8, the groups'
 *                     numbers below with JYHIP_T_I4, else NULL
 * head_dim: a multiple of 16 up to 256; page_size: 16, 32, 64, 128 or 256; type: JYHIP_T_I8,
 * JYHIP_T_I4, JYHIP_T_F16 or JYHIP_T_BF16.  k and v are aligned to 16 bytes, as 4-bit pages' scales are.  An int8 vector holds
 * q * scale by the rule of jyhip_kv (libs/model_libs/attention/attention_q8.h:29-35): scale =
 * absmax / 127, q = rint(x * (127 / absmax)), both fp32; zeros where absmax <= 1e-8.  A vector
 * with an infinity or a NaN in it is held as NaN (scale NaN), all of it.
 *
 * A JYHIP_T_I4 vector is laid out in G groups of 32 elements, G = 2 for a head_dim up to 64, 4 up to 128,
 * 8 above: 16 G bytes, byte r G + g holding the numbers n of elements 32 g + 2 r (its low half) and
 * 32 g + 2 r + 1 (what lies past head_dim holds zeros); so k, v are [num_pages][num_kv_heads][page_size][16 G]
 * bytes.  k_scale, v_scale point to fp16 [num_pages][num_kv_heads][page_size][G][2], each group's step and
 * lowest value: an element is n * step + low, with low = fp16(min x), step = fp16(round7((max x - low) / 15)),
 * n = rint((x - low) * (1 / step)) in 0 .. 15 (0 where step is 0), in fp32; round7 rounds to seven significant
 * bits, ties to even.  A vector with an element that is not finite or past +-30000 is held as NaN, all of it.
 * Steps that are not of this kind (more than seven bits, over 4000) are within the rules of none of these calls. */
typedef struct jyhip_pages {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    int num_pages;
    int page_size;
    int num_kv_heads;
    int head_dim;
    int type;
    int device;
} jyhip_pages;

/* Which page holds a sequence's positions: position p of sequence s lies in slot p % page_size
 * of page tables[s * table_stride + p / page_size].  An id outside [0, num_pages) is a hole: its
 * positions do not exist (they are not written, read as zeros, and attention leaves them out).
 * The same page may stand in several sequences' tables (a shared prefix).  The tables are read on
 * the device. */
typedef struct jyhip_page_tables {
    const int* tables;
    int num_seqs;
    int table_stride; /* pages per sequence */
} jyhip_page_tables;

/* Vectors [row][head][head_dim]: element (r, h, i) at data[r * row_stride + h * head_stride + i]
 * (strides in elements, not negative). */
typedef struct jyhip_vectors {
    void* data;
    long long row_stride;
    long long head_stride;
} jyhip_vectors;

/* Write the keys and values k, v (elements of `type`: JYHIP_T_F32, _F16 or _BF16) of `rows`
 * positions: row r is position pos[r] of sequence seq[r] (seq NULL: of sequence r).  A row whose
 * sequence or position does not exist (negative, past the table, a hole) is skipped: so the idle
 * rows of a padded batch have position -1.  The rows of one call are different positions; where
 * two name the same slot, that slot's contents are unspecified.  rows x num_kv_heads is at most
 * 2^28 - 16. */
JYHIP_API int jyhip_pages_write(const jyhip_pages* pages, const jyhip_page_tables* tables, int rows, const int* seq,
                                const int* pos, const jyhip_vectors* k, const jyhip_vectors* v, int type,
                                void* stream);

/* Read the same positions back as values of `type` (zeros for a row that does not exist). */
JYHIP_API int jyhip_pages_read(const jyhip_pages* pages, const jyhip_page_tables* tables, int rows, const int* seq,
                               const int* pos, const jyhip_vectors* k, const jyhip_vectors* v, int type, void* stream);

/* Attention of one query row per sequence over the first lens[s] positions of every sequence s of
 * `tables`: out[s][h] = sum_j softmax_j(scale q[s][h] . k_j) v_j, head h reading kv head
 * h / (num_heads / num_kv_heads).  q and out are of `type` (JYHIP_T_F32, _F16, _BF16); scores,
 * softmax and sums are held in fp32 (against int8 keys a query vector under 2^-104 counts as zeros).  A
 * sequence without any position (lens[s] <= 0, only holes) gives zeros.  max_len, at most 2^30, is an upper
 * bound of lens known on the host: it sizes the launch, and a longer lens[s] is cut to it; a loose one costs
 * some time, as it sizes the pieces that the sequences are taken in, too.  The workspace
 * needs jyhip_pages_attend_workspace() bytes, aligned to 16 (0 for arguments that are refused).
 *
 * What is not finite: a query vector with an infinity or a NaN gives NaN.  A score of -infinity has no
 * weight (a row of nothing else gives zeros), one of +infinity or NaN makes its row NaN, and a value that is
 * not finite is so in its dim of every row that reads it, NaN where its weight is 0.  There a query's
 * element under 2^-39 of its vector's largest and a weight under 2^-39 of its row's largest may count as
 * 0.  Int8 scales are finite or NaN.  Scores of 2^127 and more, and sums of weights (the largest 1) times
 * values past fp32's range, are infinite. */
JYHIP_API int jyhip_pages_attend(const jyhip_pages* pages, const jyhip_page_tables* tables, const int* lens,
                                 int max_len, int num_heads, float scale, const jyhip_vectors* q,
                                 const jyhip_vectors* out, int type, void* workspace, size_t workspace_bytes,
                                 void* stream);
JYHIP_API size_t jyhip_pages_attend_workspace(const jyhip_pages* pages, int num_seqs, int num_heads, int max_len);

/* One token id for each of `rows` rows of `vocab` logits (of `type`, row r at logits + r *
 * row_stride elements), from the row's own settings and a given random number u[r] in [0, 1):
 *   temperature  T <= 0: the largest logit (the lowest index of equal ones), the rest unused;
 *                else token i has mass e_i = exp((x_i - max x) / T), and the tokens stand in order
 *                of falling logits, equal ones by index
 *   top_k        k > 0: the first k stay
 *   top_p        p < 1: of those, the ones before which less than p of their mass lies (the first
 *                always stays)
 *   min_p        m > 0: of those, the ones with e_i >= m (at most 1)
 * and the id is the lowest index at which the running sum of the staying tokens' masses, in order of
 * indices, exceeds u[r] times their total.  Masses are fp64, added up as whole numbers (a step is
 * at most 2^-40 of the largest mass), so a row's id does not depend on the order of additions.
 * A logit that is NaN or -infinity is never picked; a row of nothing else gives -1.  With +infinity
 * among the logits, those alone have mass.  Each of temperature, top_k, top_p and min_p may be
 * NULL: 1, off, off, off.  A NaN temperature counts as 0, a NaN top_p or min_p is off.  u outside [0, 1) counts
 * as the nearest value in it, NaN as 0.  A row with a top_k from 1024 on (and below vocab) takes about ten
 * times as long as others.  vocab is at most 2^22, rows less than 2^20.  The workspace needs jyhip_sample_workspace() bytes, aligned to 16. */
JYHIP_API int jyhip_sample(const void* logits, int type, int rows, int vocab, long long row_stride, const float* u,
                           const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                           int* ids, void* workspace, size_t workspace_bytes, int device, void* stream);
JYHIP_API size_t jyhip_sample_workspace(int rows, int vocab);

/* What else makes a score, beside scale q . k:
 *   cap     c > 0: a score s becomes c tanh(s / c), so it stays within +-c (0: as it is; over 2^64: 2^64)
 *   slopes  fp32 [num_heads]: then slope * |the row's position - the key's| is taken off (NULL: nothing)
 *   first   int32, one per row: positions before it are left out (NULL: none; a window, a document's start)
 *   last    int32, one per row: positions from it on are left out (NULL: those after the row's own; past it
 *           for a prefix that is seen whole) */
typedef struct jyhip_rules {
    float cap;
    const float* slopes;
    const int* first;
    const int* last;
} jyhip_rules;

/* jyhip_pages_attend with rules (NULL: none; `last` is not for it), the row of sequence s at position lens[s] - 1
 * over positions first[s] .. lens[s] - 1.  With `first`, max_len is an upper bound of lens[s] - first[s], and of
 * more positions the first max_len count.  With `weights`, fp32, the weights of position j, summed over the
 * query heads of a kv head, are added to weights[s * weights_seq_stride + kv head * weights_head_stride + j]
 * (strides in elements), for each position j < weights_len that s sees; each sequence and head has elements of its own (strides
 * that say otherwise are refused).  What is not finite: as in
 * jyhip_pages_attend, but that what a row's rules leave out never reaches it; with a cap a score of +-infinity is
 * +-cap. */
JYHIP_API int jyhip_pages_attend_ruled(const jyhip_pages* pages, const jyhip_page_tables* tables, const int* lens,
                                       int max_len, int num_heads, float scale, const jyhip_rules* rules,
                                       const jyhip_vectors* q, const jyhip_vectors* out, int type, float* weights,
                                       long long weights_seq_stride, long long weights_head_stride, int weights_len,
                                       void* workspace, size_t workspace_bytes, void* stream);
JYHIP_API size_t jyhip_pages_attend_ruled_workspace(const jyhip_pages* pages, int num_seqs, int num_heads, int max_len,
                                                    int has_first, int has_weights);

/* The same for runs of rows (prompts, drafted tokens): sequence s has the query rows starts[s] .. starts[s + 1] - 1 of
 * q and out (starts: int32 [num_seqs + 1], ascending, on the device), and row r stands at position pos[r] and sees
 * positions first[r] .. last[r] - 1 (0 and pos[r] + 1 without them) of its sequence, whose keys and values are in the
 * pages.  A row that sees nothing gives zeros; rows before starts[0] and from starts[num_seqs] on are left as they
 * are.  max_len is an upper bound of the positions that any row sees (last, or pos + 1): those past it are cut.
 * Long runs of 16-bit rows take a weight as one number of the second product's type: fp16 over fp16 and 4-bit pages
 * (under 2^-34 of its row's largest it may count as 0; a 4-bit value is rounded to fp16 there), else bf16, in two
 * parts where the outputs are fp16; sums are fp32.  Which runs are long is decided by the call's rows, query heads and
 * sequences.  What is not finite: as with single rows, for each row by what it sees.  rows x num_heads is less than 2^22. */
JYHIP_API int jyhip_pages_attend_rows(const jyhip_pages* pages, const jyhip_page_tables* tables, const int* starts,
                                      const int* pos, int rows, int max_len, int num_heads, float scale,
                                      const jyhip_rules* rules, const jyhip_vectors* q, const jyhip_vectors* out, int type,
                                      void* workspace, size_t workspace_bytes, void* stream);
JYHIP_API size_t jyhip_pages_attend_rows_workspace(const jyhip_pages* pages, int num_seqs, int rows, int num_heads,
                                                   int max_len, int type);

/* Evict what gets little attention: of the first n = min(lens[s], max_len) positions of every sequence (holes do not
 * count) each kv head keeps min(keep, their number): those from n - recent on, and of the others the ones with the
 * largest weights, equal ones by position (NaN counts as the least, a position past weights_len as 0).  weights: fp32,
 * position j of kv head h at weights[s * weights_seq_stride + h * weights_head_stride + j], as jyhip_pages_attend_ruled adds them up.
 * What stays moves, in order, to positions 0, 1, ... of the pages that `to` names, which are none that any of `tables`
 * names (their contents would be unspecified): the caller frees the old ones afterwards.  kept [num_seqs][kv heads][keep]
 * receives the old positions, -1 behind them; new_lens the new lengths (lens itself is not for it); new_weights, if not
 * NULL, the weights of what stayed and zeros behind them, new_weights_len a head; it may be `weights` itself with the same
 * strides and length.  0 <= recent <= keep, keep >= 1; sequences x kv heads x keep is at most 2^28 - 16. */
JYHIP_API int jyhip_pages_evict(const jyhip_pages* pages, const jyhip_page_tables* tables, const jyhip_page_tables* to,
                                const int* lens, int* new_lens, int max_len, int keep, int recent, const float* weights,
                                long long weights_seq_stride, long long weights_head_stride, int weights_len,
                                float* new_weights, long long new_seq_stride, long long new_head_stride,
                                int new_weights_len, int* kept, void* stream);

/* Rotary positions: turn the pairs of every head of `rows` rows of queries (q_heads heads) and keys (k_heads,
 * 0 with k and k_out NULL: none).  Pair i of a head of row r turns by the angle pos[r] * freq[i] (fp64):
 *   (x, y) -> (x c - y s, x s + y c),  c = factor * cos, s = factor * sin
 * with (x, y) elements (i, i + pairs) or, interleaved, (2 i, 2 i + 1); a head's elements from 2 pairs on are
 * copied.  q, k and the outputs hold elements of `type` (JYHIP_T_F32, _F16, _BF16); an output may be its own
 * input (the same data and strides), else they do not overlap.  Products are fp32, rounded once; angles are
 * good up to 2^40.  head_dim is at most 1024, 2 pairs at most head_dim, pairs at least 1. */
JYHIP_API int jyhip_rope(const jyhip_vectors* q, const jyhip_vectors* q_out, int q_heads, const jyhip_vectors* k,
                         const jyhip_vectors* k_out, int k_heads, int rows, int head_dim, const int* pos,
                         const double* freq, int pairs, int interleaved, float factor, int type, int device,
                         void* stream);

/* One pass of a model over `rows` tokens of several sequences whose keys and values lie in pages: row r
 * is position pos[r] of sequence seq[r] (seq NULL: of sequence r).  X and out: host [rows][hidden], the
 * tokens' embeddings and their final-normed hidden states, as in jyhip_forward_cached_to (out may be X).
 * pages: one pool per layer of the model (pages[0 .. num_layers)), of one number and size of pages (the types
 * may differ), on the model's device, its heads the model's.  tables, seq and pos are HOST arrays here ([num_seqs][table_stride],
 * [rows], [rows]).  Each layer writes the rows' keys and values into the pages, then every row attends
 * over positions 0 .. pos[r] of its sequence, so several new positions of one sequence may come in one
 * call (a prompt) as long as the earlier ones are in the pages or in the call; each row reads its positions
 * by itself, so a long prompt takes a time that grows with its square.
 * Refused before anything is enqueued: positions outside the RoPE table or the page table, page ids
 * outside the pool among those that a row attends over, two rows with the same slot.
 * The products are the model's (its mode's); the attention is jyhip_pages_attend's, which does not
 * round the query to int8 as the reference's does.  Waits for the model's stream; work on other streams
 * that the pages depend on has to be done before. */
JYHIP_API int jyhip_forward_paged(jyhip_model* model, const jyhip_pages* pages, const float* X, float* out, int rows,
                                  const int* tables, int num_seqs, int table_stride, const int* seq, const int* pos);

/* jyhip_session_step for a sampled session, the tokens drawn on the device by jyhip_sample with the
 * session's temperature, these filters (top_k <= 0, top_p >= 1, min_p <= 0: off) and the given numbers
 * u (host, n of them in [0, 1), one per step): the logits do not leave the device.  Returns how many
 * tokens were produced; -1, and the session ends, where a step's logits hold nothing but NaN and
 * -infinity.  Refuses a greedy session (temperature <= 0) and one with a repetition
 * penalty.  The session's first token came from jyhip_session_begin. */
JYHIP_API int jyhip_session_step_sampled(jyhip_session* s, int n, int top_k, float top_p, float min_p, const float* u);

#ifdef __cplusplus
}
#endif

#endif
