/*
 * xj_hip.h - the MI355X (gfx950) backend for the xiaoju-pipe token loop.
 *
 * Three layers, all C ABI (plain pointers and sizes):
 *
 *  1. The drop-in stage. xj_hip_stage_new returns a `struct xj_stage` whose
 *     vtable behaves like the Metal stage it replaces, so the reference's
 *     pipeline (xj_pipeline_eval/verify/rollback) and speculative driver run
 *     on it unchanged.
 *       xj_hip_stage_new    <- xj_metal_stage_new  src/xiaoju-pipe/core/xj_stage.h:46-47
 *       xj_hip_device_name  <- xj_metal_device_name src/xiaoju-pipe/core/xj_stage.h:48
 *       xj_hip_tune_note    <- xj_metal_tune_note  src/xiaoju-pipe/core/xj_stage.h:50
 *
 *  2. Host-side counterparts of the reference loader, needed because the
 *     reference sources do not ship with this library. They carry the xjh_
 *     prefix so that a program linking the reference's own core objects next to
 *     this library sees no duplicate symbols; a model built by either loader
 *     can be passed to xj_hip_stage_new (the struct layout is the same):
 *       xjh_model_load / xjh_model_free <- xj_model_load / xj_model_free
 *                                          src/xiaoju-pipe/core/xj_model.h:64,69
 *       xjh_model_load_layers           <- xj_model_load_layers  xj_model.h:66
 *       xjh_model_attach_mtp            <- xj_model_attach_mtp   xj_model.h:72
 *       xjh_model_mtp_range             <- xj_model_mtp_range    xj_model.h:74
 *                                          (takes a path instead of a gguf_file)
 *       xjh_model_ranges                <- xj_model_ranges       xj_model.h:78
 *       xjh_model_layer_bytes           <- xj_model_layer_bytes  xj_model.h:80
 *       xjh_row_bytes / xjh_type_block  <- xj_row_bytes / xj_type_block
 *       / xjh_type_name                    / xj_type_name  src/xiaoju-pipe/core/gguf.h:81-83
 *     plus a writer for synthetic qwen35 GGUF files and the Q4_K / Q6_K /
 *     Q8_0 quantizers it uses (the reference has none for K-quants).
 *
 *  3. Device-resident extensions with no Metal counterpart: a chain of HIP
 *     stages that keeps the hidden state in HBM between stages, embeds token
 *     ids and takes the greedy argmax on the device, and replays one decode
 *     step as a HIP graph; a speculative driver with a separate draft model;
 *     and one C entry point per kernel (dequant, GEMV, norms, RoPE, attention,
 *     DeltaNet, argmax) used by the parity tests and the benchmark.
 *
 * Errors: every function that can fail returns -1 (or NULL) and writes a
 * message into err[errlen], as the reference does.
 */
#ifndef XJ_HIP_H
#define XJ_HIP_H

#include "xj_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- stage -- */

/* Same contract as xj_metal_stage_new (xj_stage.h:46-47, semantics
 * xj_metal.m:554-663): validates the layer range and weight mapping, copies
 * the weights of [l0,l1) (and the head when has_head) into HBM, allocates the
 * fp16 KV cache of every attention layer ([n_ctx][n_head_kv*head_dim]) and the
 * fp32 conv/recurrent state of every DeltaNet layer. backend = "hip".
 * With a model that has an MTP layer, [n_layer, n_layer + 1) builds the MTP
 * stage (mtp = true, xj_cpu.c:378-379): forward takes T rows of
 * [embedding | hidden] (2 n_embd floats each; the result, n_embd per row, is
 * written to the first T * n_embd floats), each half RMS-normalised with
 * nextn.enorm / nextn.hnorm and mapped back by nextn.eh_proj before the layer
 * (xj_cpu.c:253-261); its head normalises with nextn.shared_head_norm
 * (xj_cpu.c:287). */
xj_stage   *xj_hip_stage_new(const xj_model *m, int l0, int l1, int n_ctx, int max_batch,
                             bool has_head, char *err, size_t errlen);
const char *xj_hip_device_name(void);
const char *xj_hip_tune_note(void);

/* Bytes of HBM a stage holds besides the repacked weights
 * (counterpart of xj_stage_state_bytes, xj_stage.h:57). A chain
 * (xjh_chain_new) over stages of max_batch <= 512 whose matrices are mostly
 * Q4_K and Q6_K adds a second set of scratch per stage, for prompts beyond
 * max_batch in pieces of up to min(n_ctx, 1024) tokens: when it is built if
 * max_batch >= 16, else on the first prompt of 16 tokens or more beyond two
 * chunks. Other prompts beyond max_batch run in chunks of max_batch, a single
 * stage's layers in up to XJ_STAGE_SPLIT parts, for which the chain adds up to
 * XJ_STAGE_SPLIT - 1 further sets of the stage's own scratch: when it is built
 * if max_batch >= 16 and there are no pieces, else on the first such prompt.
 * Without the memory for them, chunks run one after the other. */
uint64_t    xj_hip_stage_state_bytes(const xj_model *m, int l0, int l1, int n_ctx, int max_batch);

/* Copy the whole recurrent state (conv + DeltaNet state of every layer) of a
 * HIP stage into snapshot slot `slot` (0 <= slot < 8), and restore it while
 * setting n_past. Lets a draft model roll back across separate T=1 calls,
 * which the reference's keep/rollback (one forward call only) cannot. */
int xj_hip_stage_snapshot(xj_stage *s, int slot, char *err, size_t errlen);
int xj_hip_stage_restore(xj_stage *s, int slot, int n_past, char *err, size_t errlen);
/* Test hook, no counterpart in the reference: fill every attention layer's K
 * and V cache from position pos0 to n_ctx with the fp16 pattern `bits`
 * (e.g. 0x7E00, a NaN), standing for stale memory that a decode step must
 * never read before writing it. */
int xj_hip_stage_fill_kv(xj_stage *s, int pos0, uint16_t bits, char *err, size_t errlen);

/* -------------------------------------------------------- host loader -- */

int         xjh_type_block(uint32_t type, int *block_bytes);
uint64_t    xjh_row_bytes(uint32_t type, int64_t n);
const char *xjh_type_name(uint32_t type);
/* The whole file mapped; the model table as xj_model_load builds it
 * (xj_model.c:129-209): hparams, layer pattern, tensors, tied head, eos/eot,
 * fingerprint, and the MTP layer in layers[n_layer] when the file has one. */
xj_model   *xjh_model_load(const char *path, char *err, size_t errlen);
void        xjh_model_free(xj_model *m);
/* Partial load for a stage of layers [l0, l1) (xj_model.c:214-233):
 * only the GGUF header is read, then one mapping spans the merged byte ranges
 * of those layers (with_io: also token_embd, output_norm, output). Tensors
 * outside the mapping keep data = NULL, so a stage over other layers fails
 * ("weights are not mapped"); the file may be a partial download as long as
 * it reaches the end of that span. Error for an empty or out-of-range [l0, l1). */
xj_model   *xjh_model_load_layers(const char *path, int l0, int l1, bool with_io, char *err, size_t errlen);
/* Attach the MTP layer of another GGUF of the same model (xj_model.c:275-300):
 * only its header and the MTP layer's byte span need to be present in that
 * file. No-op when m already has one; error when the shapes differ or the
 * file has no MTP layer. The mapping is released by xjh_model_free(m). */
int         xjh_model_attach_mtp(xj_model *m, const char *path, char *err, size_t errlen);
/* Byte span [lo, hi) of the MTP layer (layer tensors and nextn.*) of the
 * GGUF at path, from its header alone (xj_model.c:262-273). */
int         xjh_model_mtp_range(const char *path, uint64_t *lo, uint64_t *hi, char *err, size_t errlen);
/* Byte ranges [lo, hi) of the file that layers [l0, l1) (and with include_embd
 * the embedding, output norm and untied head) occupy, sorted, ranges at most
 * 4096 bytes apart merged; returns their count, at most max (xj_model.c:315-328). */
int         xjh_model_ranges(const xj_model *m, int l0, int l1, bool include_embd, uint64_t (*ranges)[2], int max);
/* Total tensor bytes of layers [l0, l1) (xj_model.c:330-338). */
uint64_t    xjh_model_layer_bytes(const xj_model *m, int l0, int l1);

/* --------------------------------------------------- synthetic models -- */

/* Shape and quantization recipe of a random-weight qwen35 model. Matrices are
 * N(0, w_std); norm weights 1 + 0.1 N; ssm_a = -exp(0.5 N); ssm_dt = 0.5 N;
 * conv1d 0.5 N. Every value is a pure function of (seed, tensor name, row). */
typedef struct {
    int n_layer, n_embd, n_ff, n_vocab;
    int n_head, n_head_kv, head_dim, n_rot;
    float rope_base, eps;
    int conv_k, s_k, h_k, h_v;          /* d_inner = h_v * s_k */
    int full_attn_interval;
    uint32_t type_default;              /* every matrix not named below */
    uint32_t type_embd, type_out, type_v, type_down;
    float w_std;
    uint64_t seed;
    int nextn;                          /* 1: one MTP layer (blk.{n_layer}, nextn.*) */
    int32_t eos_id;                     /* >= 0: tokenizer.ggml.eos_token_id */
    int32_t eot_id;                     /* >= 0: a token list with "<|im_end|>" at this id */
} xjs_config;

/* Fill out[n] with N(0, std) from the build's generator: splitmix64 feeding
 * Box-Muller in double, rounded to float. */
void xjs_fill_normal(float *out, int64_t n, uint64_t seed, float std);
/* Per-tensor seed = seed ^ FNV-1a(name). */
uint64_t xjs_tensor_seed(uint64_t seed, const char *name);
/* Quantize n_rows rows of k floats into `out` (row_bytes(type, k) each). */
int  xjs_quantize(uint32_t type, const float *x, int64_t n_rows, int64_t k, void *out,
                  char *err, size_t errlen);
/* Write a qwen35 GGUF v3 file for cfg; returns total bytes or -1. */
int64_t xjs_write_model(const char *path, const xjs_config *cfg, char *err, size_t errlen);

/* ------------------------------------------ device chain (fast path) -- */

typedef struct xjh_chain xjh_chain;

/* A chain runs HIP stages in sequence on one stream with the hidden state
 * kept in HBM; the last stage must have the head. Mirrors the no-remote branch
 * of eval_once (xj_net.c:541-559) with embedding and argmax on the device. */
xjh_chain *xjh_chain_new(xj_stage **stages, int n_stages, char *err, size_t errlen);
void       xjh_chain_free(xjh_chain *c);
/* Feed n tokens: up to max_batch in one chunk, more in pieces of up to 1024
 * tokens or in chunks of max_batch (xj_hip_stage_state_bytes). When nlog > 0 the
 * logits of the last min(nlog, rows) rows, rows being what chunks of max_batch
 * leave for the last one, are computed: copied to `logits`
 * [nlog][n_vocab] when it is not NULL, and their greedy argmax (first maximum)
 * written to `argmax`. keep != 0 turns this call into a verify (xj_net.c:668):
 * all n tokens in one chunk, recurrent checkpoints kept for rollback. The
 * token the next decode step feeds is the last row's argmax or, with the
 * sampler on (xjh_chain_set_sampler), its draw (one number consumed). */
int  xjh_chain_eval(xjh_chain *c, const int32_t *tokens, int n, int nlog, int keep,
                    float *logits, int32_t *argmax, char *err, size_t errlen);
/* Up to n_steps steps entirely on the device. The first input token is the
 * one left by the previous eval/decode; out[i] receives the token chosen after
 * step i (so out[0] is the first step's argmax or, with the sampler on, its
 * draw with the next number). One step is one HIP graph launch. Generation stops at the model's end token
 * (hp.eos / hp.eot, xj_spec.c:29,139): it is the last token written and it is
 * not fed, so the state is that of the tokens before it. Returns the number of
 * tokens written (0 when the previous token already was an end token), or -1. */
int  xjh_chain_decode(xjh_chain *c, int n_steps, int32_t *out, char *err, size_t errlen);
/* The token that the next decode step would feed (the last argmax or draw). */
int  xjh_chain_last_token(xjh_chain *c);
/* The app's sampler on the device-resident path: with temperature > 0 every
 * token the chain produces - after xjh_chain_eval's last row, at each
 * xjh_chain_decode step, and the target's tokens in both speculative drivers -
 * is the draw of the app's top-k 40 / top-p 0.95 sampler from its logits row,
 * with the next of the n numbers rand30[] (each < 2^30) standing in for its
 * arc4random_uniform(1 << 30); numbers are consumed in order, one per token
 * produced, and a call that would need more than are left fails.
 * temperature <= 0 is greedy decoding (no number consumed, the app's rule).
 * Drafts stay greedy, as the reference's MTP drafts are. A chain reset keeps
 * the numbers and the count; this call restarts the count.
 * Replaces: the app's sample_cb passed to xj_spec_next
 * (src/xiaoju-pipe/ios/App/XJGlue.c:248-282, core/xj_spec.c:135,185). */
int  xjh_chain_set_sampler(xjh_chain *c, float temperature, const uint32_t *rand30, int n,
                           char *err, size_t errlen);
/* Numbers consumed since the last xjh_chain_set_sampler. */
int  xjh_chain_sampler_used(xjh_chain *c);
int  xjh_chain_rollback(xjh_chain *c, int n_past, char *err, size_t errlen);
void xjh_chain_reset(xjh_chain *c);
int  xjh_chain_n_past(xjh_chain *c);
/* Average GPU time of the last xjh_chain_decode, in ms per step, from HIP
 * events recorded on the chain's stream around the replayed graphs. */
double xjh_chain_last_decode_ms(xjh_chain *c);

/* Run only the GEMV launches of one T=1 decode step (same shapes and weights,
 * epilogues redirected to scratch so no state changes) `iters` times between
 * HIP events on the chain's stream. Reports the mean GPU ms per step, the
 * algorithmic HBM bytes of those launches per step, and the launch count. */
int  xjh_chain_time_gemv(xjh_chain *c, int iters, double *ms_per_step, double *bytes_per_step,
                         int *launches_per_step, char *err, size_t errlen);

/* Speculative decoding with a separate draft model (no reference
 * counterpart: the reference drafts with an MTP layer, xj_spec.c:131-209, and
 * the accept/rollback rule below is that function's). Each step feeds the
 * pending token t to the draft and lets it propose up to k tokens by greedy
 * T=1 steps, verifies [t, d1..dk] on the target in one batch, accepts the
 * longest prefix the target's token agrees with (its argmax, or with the
 * target's sampler on its draw, row i with the next number + i, so the output
 * is that of plain sampled decoding with the same numbers) and rolls both
 * models back. Greedy with k = 4, after rounds whose drafts were all
 * accepted, the draft makes the next round's drafts while the target
 * verifies (from the round's last draft: one step for the target's next
 * token, then k); they are used when the target accepts every draft and its
 * next token is the guessed one, so the tokens are those of the sequential
 * rounds (XJ_SPEC_PIPE=0: always sequential).
 * oracle (optional, n_oracle ids) replaces the drafts, with every
 * (g*7+j) % oracle_miss == 0 draft made wrong, as xj_spec.c:173-177; the
 * guess of the target's next token is then the oracle's. */
typedef struct {
    long n_steps, n_drafted, n_accepted;
    long acc_at[4];
    double t_total_ms, t_draft_ms;
    long n_overlap, n_overlap_held;   /* rounds drafted ahead during a verification; of them used */
} xjh_spec_stats;
/* Returns the number of tokens written to out (at most n_gen): generation
 * stops after an end token (hp.eos / hp.eot), which is written but not fed,
 * and an accepted end token cuts the accepted drafts there (xj_spec.c:139,
 * :193-194). -1 on error. */
int xjh_spec_generate(xjh_chain *target, xjh_chain *draft, int k, int n_gen,
                      const int32_t *oracle, int n_oracle, int oracle_miss,
                      int32_t *out, xjh_spec_stats *stats, char *err, size_t errlen);

/* Speculative decoding with the model's own MTP stage as the drafter, the
 * reference's algorithm (xj_spec.c:97-209, greedy or the chain's sampler: the MTP stage
 * takes every fed position with the token after it, drafts k <= 4 tokens, the
 * first from the pending positions and each further one from
 * [embedding(previous draft) | shared_head_norm(previous MTP output)]; the
 * target verifies [t, d1..dk] in one batch and keeps the agreeing prefix).
 * The target's hidden rows pass its output_norm before the MTP stage takes
 * them, and an MTP output passes shared_head_norm before it is fed back, both
 * as x * (sc * w) (the driver's defaults, XJ_MTP_MAIN_POST / XJ_MTP_CHAIN_POST
 * = 0 turn them off as in the reference).
 * Feeds the prompt itself (both models are reset first); out receives the
 * tokens of plain greedy decoding (with the target's sampler on: of plain
 * sampled decoding with the same numbers), end tokens handled as in xjh_spec_generate;
 * returns their count or -1. draft_log (optional) receives the first
 * draft_cap drafted tokens in order, before any oracle replacement. oracle /
 * oracle_miss as for xjh_spec_generate. mtp: xj_hip_stage_new(m, n_layer,
 * n_layer + 1, ..., has_head = true) of the target's model.
 * Replaces: xj_spec_feed / xj_spec_next with an MTP stage
 * (src/xiaoju-pipe/core/xj_spec.c:117-209) over the device chain. */
int xjh_spec_generate_mtp(xjh_chain *target, xj_stage *mtp, int k, const int32_t *prompt, int n_prompt,
                          int n_gen, const int32_t *oracle, int n_oracle, int oracle_miss,
                          int32_t *out, xjh_spec_stats *stats, int32_t *draft_log, int draft_cap,
                          char *err, size_t errlen);

/* ----------------------------------------------------- per-op kernels -- */

/* Device memory and stream helpers for tests and benchmarks. All per-op
 * entry points run on the library's own stream and return after the GPU
 * finished unless stated otherwise. */
void *xjh_malloc(size_t bytes);
void  xjh_free(void *p);
int   xjh_h2d(void *dst, const void *src, size_t bytes);
int   xjh_d2h(void *dst, const void *src, size_t bytes);
/* Device-to-device copy (the runtime's copy kernel): the known-size transfer
 * that calibrates the HBM byte counters of a profiler run. */
int   xjh_d2d(void *dst, const void *src, size_t bytes);
int   xjh_sync(void);
const char *xjh_last_error(void);

/* Repack a GGUF tensor (n_rows rows of k elements, GGUF block layout) into the
 * device layout the kernels read; returns the device pointer, NULL on error.
 * Q4_K and F32 keep the GGUF layout; Q6_K and Q8_0 are split into planes
 * (quants, high bits, scales, d) so every load is 16-byte aligned. */
void *xjh_upload_weight(uint32_t type, const void *host, int64_t n_rows, int64_t k,
                        char *err, size_t errlen);
/* Bit-exact dequantization of rows [r0, r0+n) of an uploaded weight into y. */
int xjh_dequant(uint32_t type, const void *dw, int64_t n_rows, int64_t k, int64_t r0, int64_t n,
                float *y, char *err, size_t errlen);
/* y[t][r] = W[r] . x[t] (add != 0: y += ...), T in 1..max, fp32 accumulate. */
int xjh_gemv(uint32_t type, const void *dw, int64_t n_rows, int64_t k, const float *x, int T,
             float *y, int add, char *err, size_t errlen);
/* xjh_gemv without any allocation: no counterpart in the reference. For
 * callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc). The same kernels and
 * results as xjh_gemv, bit for bit; the prepared activations go to a static
 * 1 MiB scratch array that each GPU holds from the library's load to the end
 * of the process, so T * (7.625 * k rounded up to 256 bytes) must fit in
 * 1 MiB (k = 9216: T <= 14), or the call fails with a message. Nothing in the
 * scratch needs to start at zero; every call on a GPU reuses that GPU's copy,
 * so calls that overlap on one GPU (other threads) race. The first call in a
 * process creates the library's stream, as every per-op entry does. */
int xjh_gemv_noalloc(uint32_t type, const void *dw, int64_t n_rows, int64_t k, const float *x, int T,
                     float *y, int add, char *err, size_t errlen);
/* The same product for a prefill chunk on the matrix cores: Q4_K or Q6_K
 * rows, k % 256 == 0, T in 1..64. The activations enter as two f16 planes per
 * 256-element block (v * 2^-e = hi + lo) and the weights as integers exact in
 * f16, so every product is exact and only the fp32 accumulation rounds
 * (~1e-7 of the float64 product; xjh_gemv, with 21-bit activations, agrees
 * to ~1e-6). Counterpart of the Metal batched kernel mvb
 * (src/xiaoju-pipe/metal/xj_kernels.metal:84-388) for long batches. */
int xjh_gemm(uint32_t type, const void *dw, int64_t n_rows, int64_t k, const float *x, int T,
             float *y, int add, char *err, size_t errlen);
/* Test hook, no counterpart in the reference: the GEMM of prompt pieces
 * (33 <= T <= 1024) over nseg <= 4 matrices of one type that share the input x
 * (16-byte aligned), y[i] of matrix i [T][n_rows[i]]; norm_w (may be NULL): x is
 * RMS-normalised with it first (eps 1e-6). *kind: the kernel taken, 0 the one for
 * up to 64 tokens, 1 slices of 64 tokens on it, 2 the one for more. */
int xjh_gemm_piece(uint32_t type, const void *const *dw, const int64_t *n_rows, int nseg, int64_t k, const float *x,
                   const float *norm_w, int T, float *const *y, int add, int *kind, char *err, size_t errlen);
/* Mean ms of xjh_gemm (prep launch included) over rotating copies, like xjh_gemv_time. */
double xjh_gemm_time(uint32_t type, void *const *dws, int n_copies, int64_t n_rows, int64_t k,
                     const float *x, int T, float *y, int iters, char *err, size_t errlen);
/* Time `iters` back-to-back launches of xjh_gemv over n_copies weights
 * (rotating, to defeat the caches), with HIP events on the library stream.
 * Returns the mean ms per launch, or -1. */
double xjh_gemv_time(uint32_t type, void *const *dws, int n_copies, int64_t n_rows, int64_t k,
                     const float *x, int T, float *y, int iters, char *err, size_t errlen);
/* out[t] = rmsnorm(x[t]) * w  (mode 0: x * sc * w, xj_cpu.c:56-61), x[t]/sqrt(sum x^2 + eps)
 * (mode 1, xj_cpu.c:185-193) or x * (sc * w) (mode 2, the speculative driver's norm_inplace,
 * xj_spec.c:19-25); sc = 1/sqrt(sum x^2 / n + eps) with the sum in double. */
int xjh_norm(int mode, const float *x, const float *w, int n, int rows, float eps, float *out,
             char *err, size_t errlen);
/* g[i] = silu(g[i]) * u[i] over n floats, in place.
 * Replaces: src/xiaoju-pipe/metal/xj_kernels.metal:591-600 (xj_swiglu);
 * CPU form xj_cpu.c:273. */
int xjh_swiglu(float *g, const float *u, int64_t n, char *err, size_t errlen);
/* NeoX RoPE in place: for token t < T and head h < n_heads, the pairs
 * (i, i + n_rot/2) of x + t*tok_stride + h*head_stride are rotated by
 * theta = (pos0 + t) * base^(-2i/n_rot) (cos and sin evaluated in float on the
 * host, as xj_cpu.c:68-77 does).
 * Replaces: src/xiaoju-pipe/metal/xj_kernels.metal:422-437 (xj_rope). */
int xjh_rope(float *x, int T, int n_heads, int64_t tok_stride, int64_t head_stride, int n_rot,
             int pos0, float base, char *err, size_t errlen);
/* Depthwise causal conv + SiLU in place over x [T][C] (kernel K in 2..8,
 * weights w [C][K], state [C][K-1] = the last K-1 inputs, oldest first,
 * carried across calls); ck (may be NULL when ck_n == 0) receives the state
 * after each of the first ck_n tokens, [ck_n][C][K-1]. The code is the qkv
 * GEMV's conv epilogue.
 * Replaces: src/xiaoju-pipe/metal/xj_kernels.metal:525-549 (xj_conv_silu);
 * CPU form xj_cpu.c:172-182. */
int xjh_conv_silu(float *x, float *state, const float *w, int C, int K, int T, float *ck, int ck_n,
                  char *err, size_t errlen);
/* Gated GQA attention of T new tokens at positions n_past .. n_past+T-1, after
 * the projections, through the token loop's own kernels: qg [T][H][2D]
 * (q | gate per head), k, v [T][Hkv*D] (raw projections); the new keys get
 * RMSNorm(k_norm) + RoPE and are stored with the values into the fp16 caches
 * kc, vc [n_ctx][Hkv*D] (IEEE half bits); out [T][H*D] = softmax(q'.K^T /
 * sqrt(D)) V * sigmoid(gate) with q' = RoPE(RMSNorm(q) * q_norm). D in
 * {64, 128, 256}, H/Hkv in {1, 2, 4, 8}.
 * Replaces: src/xiaoju-pipe/metal/xj_kernels.metal:439-523 (xj_kv_store,
 * xj_attn_scores, xj_softmax, xj_attn_out); CPU form xj_cpu.c:106-147. */
int xjh_attn_decode(int T, int H, int Hkv, int D, int n_rot, float rope_base, float eps, int n_past,
                    int n_ctx, const float *qg, const float *k, const float *v, const float *q_norm,
                    const float *k_norm, uint16_t *kc, uint16_t *vc, float *out,
                    char *err, size_t errlen);
/* T tokens of the DeltaNet recurrence after the conv, through the token
 * loop's own kernel: per token, q and k of each of the Hk key heads (at
 * qkv[t*qkv_stride + hk*S] and + k_off) are L2-normalised (double sum,
 * x / sqrt(sum + eps)), then value head hv (key head hv % Hk, values at
 * + v_off + hv*S) takes the gated delta rule with b = sigmoid(beta_raw[t][hv]),
 * decay exp(softplus(alpha_raw[t][hv] + dt[hv]) * A[hv]); out [T][Hv*S] =
 * (S_j . q) * qscale (before the gated norm). state [Hv][S][S] ([value j][key
 * i]) is updated; ck [ck_n][Hv][S][S] receives the state after each of the
 * first ck_n tokens (ck_n <= T). S in {64, 128}; state and ck 16-byte aligned.
 * Replaces: src/xiaoju-pipe/metal/xj_kernels.metal:552-589 (xj_delta_net,
 * with the L2 norms of xj_norm mode 1 applied inside); CPU form
 * xj_cpu.c:183-213, :218. */
int xjh_delta_step(const float *qkv, int qkv_stride, int k_off, int v_off, const float *beta_raw,
                   const float *alpha_raw, const float *dt, const float *A, int Hk, int Hv, int S, int T,
                   float eps, float qscale, float *state, float *out, float *ck, int ck_n,
                   char *err, size_t errlen);
/* One token per row of the device logits [T][n]: the app's sampler, top-k 40
 * then top-p 0.95 at `temperature` (p_i = exp((v_i - v_0) / temperature) in
 * double over the 40 largest, sorted descending), the pick made with
 * rand30[t] / 2^30 (host array, each below 2^30) in place of
 * arc4random_uniform(1 << 30); temperature <= 0: the first maximum.
 * Replaces: the app's `sample`, src/xiaoju-pipe/ios/App/XJGlue.c:251-282
 * (ties among the 40 values ordered by index). */
int xjh_sample(const float *logits, int n, int T, float temperature, const uint32_t *rand30,
               int32_t *out_host, char *err, size_t errlen);
/* UTF-8 piece streaming (host only): pieces of generated text go to cb only
 * as whole UTF-8 characters. xjh_utf8_emit appends piece (its first 256
 * bytes) to the bytes held back from earlier pieces, passes everything up to
 * an incomplete trailing character (judged from the last 4 bytes) to cb,
 * holds that character back and returns cb's result (0 when nothing is
 * passed). Replaces: the app's `emit`, src/xiaoju-pipe/ios/App/XJGlue.c:285-305,
 * with the state the app keeps in host_box (XJGlue.c:161) as its own struct;
 * xjh_piece_fn is xjg_piece_fn (XJGlue.h:12). */
typedef int (*xjh_piece_fn)(void *ctx, const char *utf8, int len);
typedef struct {
    char pending[8];
    int32_t npending;
} xjh_utf8_state;
void xjh_utf8_reset(xjh_utf8_state *st);
int xjh_utf8_emit(xjh_utf8_state *st, const char *piece, int n, xjh_piece_fn cb, void *ctx);
/* First index of the maximum of each of T rows of n floats. */
int xjh_argmax(const float *x, int n, int T, int32_t *out_host, char *err, size_t errlen);
/* Gated delta rule (standalone, decay and beta given per token and head):
 * state [H][S][S] ([head][value j][key i], as xj_cpu.c:203), q,k,v [T][H][S],
 * decay,beta [T][H], out [T][H][S]. o = S^T q * qscale after the update. */
int xjh_delta_recurrent(int H, int S, int T, const float *q, const float *k, const float *v,
                        const float *decay, const float *beta, float qscale,
                        float *state, float *out, char *err, size_t errlen);
/* The same recurrence evaluated chunk-wise (chunk tokens per chunk) with the
 * chunk-level products on MFMA; must agree with xjh_delta_recurrent. */
int xjh_delta_chunked(int H, int S, int T, int chunk, const float *q, const float *k,
                      const float *v, const float *decay, const float *beta, float qscale,
                      float *state, float *out, char *err, size_t errlen);

/* -------------------------------------------------------- long contexts -- */

/* What a context beyond the trained one needs, no counterpart in the
 * reference: rotary positions with scaled frequencies, a cache of keys and
 * values in 8 bits, and attention over it with an optional sliding window.
 *
 * Unlike the other per-op entries these enqueue on `stream` (a hipStream_t of
 * the current device, hipStreamPerThread among them; NULL and hipStreamLegacy: its
 * default stream) and return without waiting
 * (xjh_sync waits), never allocate and can be captured into a HIP graph. Device
 * buffers belong to the current device, need no alignment beyond their type's
 * (the cache and the work area: 16 bytes) and are complete when the stream
 * reaches the call. Strides are in elements. T = 0 does nothing.
 * (The other per-op entries run on the library's own stream, which does not wait
 * for any other: xjh_sync before one that reads what these wrote.) Outputs do not
 * overlap inputs unless stated.
 * Where a call takes n_past_dev (may be NULL), the tokens' position is read
 * there on the GPU instead of n_past, which then is an upper bound for it, so
 * that one captured graph serves every step; a value outside [0, n_past] counts
 * as the nearer end. The bound shapes the launch: attention far below it is right
 * but slower than a call that knows its position (one token of 16 heads on 4 of 256
 * dims at 4000 of at most 131000: 28 us, 9.4 known), so that a long context is
 * better served by a few graphs of growing bounds. */

/* Rotary positions. pairs: which elements of a head turn together, (i, i +
 * n_rot/2) or (2i, 2i + 1), i < n_rot/2; the elements past n_rot do not turn.
 * Pair i of a token at position p turns by p * f_i, f_i from base^(-2i/n_rot):
 *   XJH_ROPE_PLAIN   f_i = base^(-2i/n_rot)
 *   XJH_ROPE_LINEAR  that divided by factor
 *   XJH_ROPE_YARN    with r = n_ctx_orig * base^(-2i/n_rot) / (2 pi) turns over the
 *                    trained context and g = (r - beta_slow) / (beta_fast - beta_slow)
 *                    clamped to [0, 1]: (g + (1 - g) / factor) of it
 * and is multiplied by mscale (0: 0.1 ln(factor) + 1 for YARN, else 1).
 * YARN's g is linear in the turns r, the form in which the method was published.
 * Programs that run scaled checkpoints (and the yarn fields of GGUF files) commonly
 * take g linear in the pair's index i, between the pairs that make beta_fast and
 * beta_slow turns: other frequencies between those two (by up to 1.7 for n_rot 64,
 * base 1e7, 32768 positions, factor 4, betas 32 and 1), which this call does not form. */
enum { XJH_ROPE_HALF = 0, XJH_ROPE_INTERLEAVED = 1 };
enum { XJH_ROPE_PLAIN = 0, XJH_ROPE_LINEAR = 1, XJH_ROPE_YARN = 2 };
typedef struct {
    int32_t pairs;
    int32_t n_rot;               /* even, 2 .. min(D, 512) */
    float   base;                /* > 0 */
    int32_t scaling;
    float   factor;              /* linear, yarn: >= 1 */
    int32_t n_ctx_orig;          /* yarn: > 0 */
    float   beta_fast, beta_slow;/* yarn: beta_fast > beta_slow */
    float   mscale;
} xjh_rope_cfg;
/* out[t][h] = x[t][h] rotated, for T tokens of n_heads heads of D elements (x +
 * t*x_tok + h*x_head, out likewise), token t at position pos[t] (device, may be
 * negative) or, with pos NULL, pos0 + t. out == x with equal strides rotates
 * in place; other overlaps are not allowed. The angles are formed in double, so far positions keep
 * theirs (xjh_rope evaluates them in float, as the reference does). n_heads * D is at most 2^30. */
int xjh_rope_scaled(const float *x, int64_t x_tok, int64_t x_head, float *out, int64_t o_tok, int64_t o_head, int T,
                    int n_heads, int D, const xjh_rope_cfg *cfg, const int32_t *pos, int pos0, void *stream,
                    char *err, size_t errlen);

/* A cache of the keys and values of one layer in 8 bits, one scale (float) for
 * every `block` tokens of a kv head: a value is code * scale.
 *   XJH_KV_I8    codes -127 .. 127; scale = largest magnitude / 127 (rounded to
 *                float, at least 2^-126), code = nearest integer of x / scale
 *   XJH_KV_E4M3  OCP e4m3 codes; scale = the least power of two (at least 2^-126)
 *                with largest magnitude <= 448 scale, code = nearest e4m3 of x / scale
 * Ties go to the even code and every code is that of the exact quotient. A block
 * of zeros has scale 0. NaN is stored as 0 and an infinity as the largest code;
 * neither counts for the scale, so the cache never holds them (a code of rows within
 * a step of the largest float may stand for a value just beyond it: that loads as
 * an infinity).
 * The bytes at data, N = n_ctx rounded up to 64 positions:
 *   keys   [Hkv][N/64][4 groups of 16 positions][D/64][4 x 16 dims][16 positions][16 dims]
 *   values [Hkv][N/64][D/16 groups of 16 dims][4 q][16 dims][4 u][4 r], byte (q, u, r)
 *          holding position 16 u + 4 q + r of the tile of 64
 *   scales float [Hkv][N/block] of the keys, then of the values
 * (the order in which the matrix cores take them: a wavefront reads 1 KB runs). */
enum { XJH_KV_I8 = 0, XJH_KV_E4M3 = 1 };
typedef struct {
    int32_t  type;
    int32_t  Hkv, D;             /* D: 64, 128 or 256 */
    int32_t  n_ctx;
    int32_t  block;              /* 1, 2, 4, .. 64 */
    void    *data;               /* device, 16-byte aligned */
    uint64_t bytes;              /* at data, at least xjh_kv8_bytes */
} xjh_kv8;
/* Bytes of a cache of c's type, heads, n_ctx and block; 0 when they are not supported. */
uint64_t xjh_kv8_bytes(const xjh_kv8 *c);
/* Quantise the rows k, v [T][Hkv*D] (token strides k_tok, v_tok) into positions
 * n_past .. n_past+T-1. A block that positions before n_past began keeps the
 * larger of its scale and the new rows'; where that grew, its older codes are
 * rounded again to it; if those were never stored, clear the memory first. So after
 * going back within a block (a rejected draft) it keeps the scale that the rows
 * given up had made. Blocks written from their first position start anew. Every
 * other byte keeps its value, but tiles of 64 positions are rewritten whole: what
 * stores into a tile or reads it is ordered with this call. n_past_dev: see above. */
int xjh_kv8_store(const xjh_kv8 *c, const float *k, int64_t k_tok, const float *v, int64_t v_tok, int T, int n_past,
                  const int32_t *n_past_dev, void *stream, char *err, size_t errlen);
/* Read positions pos0 .. pos0+n-1 back: k, v [n][Hkv*D] (token strides k_tok, v_tok); either may be NULL. */
int xjh_kv8_load(const xjh_kv8 *c, int pos0, int n, float *k, int64_t k_tok, float *v, int64_t v_tok, void *stream,
                 char *err, size_t errlen);
/* Attention of T tokens at positions n_past .. n_past+T-1, whose keys and values
 * (and those of every earlier position that they see) are in the cache: query head h
 * (q + t*q_tok + h*q_head, D elements) of the token at p reads kv head h / (H/Hkv)
 * and sees the positions j <= p, with window > 0 only those with j > p - window
 * or j < n_sink (the first tokens stay visible); out[t*o_tok + h*D ..] =
 * softmax(scale q.K^T) V, times sigmoid(gate[t*g_tok + h*g_head ..]) when gate is
 * not NULL. Codes are exact operands, sums are fp32. A query's elements and the
 * weights enter with 22 bits, the elements, where a work-group has 32 rows over
 * int8 keys, to 2^-19 of their row's mean magnitude or, if the largest is more
 * than 8 times that, to 2^-30 of the largest (2^-132 at least).
 * work: xjh_attn_kv8_work_bytes bytes, for splitting the positions over the
 * GPU; a smaller area (or NULL) splits less. It holds nothing between calls, but
 * calls that may run at the same time (other streams, other graphs) need one each.
 * Positions that no token sees need not be stored: what they hold, tiles that no
 * token sees even a position of unread, counts for nothing. A query that is not
 * finite leaves its own row not finite and no other. T * H is at most 2^28. */
int xjh_attn_kv8(const xjh_kv8 *c, const float *q, int64_t q_tok, int64_t q_head, const float *gate, int64_t g_tok,
                 int64_t g_head, int T, int H, int n_past, const int32_t *n_past_dev, int window, int n_sink, float scale,
                 float *out, int64_t o_tok, void *work, size_t work_bytes, void *stream, char *err, size_t errlen);
/* The work area beyond which nothing is gained for these T, n_past (or any smaller
 * n_past), window and n_sink; 0 when they are not supported. */
size_t xjh_attn_kv8_work_bytes(const xjh_kv8 *c, int T, int H, int n_past, int window, int n_sink);

/* ------------------------------------------------------ several requests -- */

/* What a program needs that runs its own layer loop over several requests at
 * once, no counterpart in the reference: a key/value cache in pages that any
 * request may own, the tables of who owns them, and attention over batches of
 * requests of different lengths. As the long-context calls these enqueue on
 * `stream` and return without waiting, never allocate, can be captured, and read
 * every length on the GPU, so that one captured step serves them all; buffers,
 * strides and work areas follow the rules there. Row types are ggml ids (XJ_F32, XJ_F16,
 * XJ_BF16). */

/* Pages of `page` positions: which are free, and which hold a request's blocks
 * (block b of request r, its positions b*page .. b*page + page-1, lies in page
 * table[r*max_blocks + b]). */
typedef struct {
    int32_t  page;               /* 16, 32, 64, 128 or 256 */
    int32_t  n_pages;            /* n_pages * page < 2^31 */
    int32_t  max_blocks;         /* entries of a table row; max_blocks * page < 2^31 */
    int32_t *table;              /* device [n_req][max_blocks] */
    int32_t *free_list;          /* device [n_pages] */
} xjh_pages;
/* Prepare a step in which request r (row r of the table) adds n_new[r] tokens behind
 * n_past[r], while its row holds the pages of held[r] positions (held NULL: n_past):
 * pages beyond those that n_past + n_new positions need go back to the free list,
 * missing ones are taken from it. So n_past < held gives up the positions of rejected
 * drafts, and n_past = n_new = 0 a request that is over. All arrays are on the device.
 *   free_list  its first *n_free entries are the free pages. Those given back are put behind them
 *              (requests and blocks in order), then pages are taken from the end (requests and
 *              blocks in order); *n_free_out (may be n_free) is how many are left. Entries from there on keep their
 *              values, and so do table entries of blocks that are not taken.
 *   cu         [n_req+1] the requests' first rows in the step's batch, and their sum
 *   kv_len     [n_req] n_past + n_new, at most max_blocks * page
 *   pos, slot  [T] of every row its position, and page * table entry + offset for xjh_paged_store (either may be
 *              NULL); rows from the sum on get position 0 and slot -1
 *   status     [4] pages missing, positions beyond the table's rows (slot -1), rows beyond T, rows.
 *              With pages missing none is taken: the wanted blocks' table entries and their tokens' slots are
 *              -1, what was given back stays given back, and the step can be tried again with less (held as
 *              it was for requests that wanted pages, n_past for those that gave some).
 * Negative lengths count as 0, n_past and held beyond the rows as the whole row; the sum of n_new is
 * below 2^31. n_req is at most 65536, n_req * max_blocks 2^30. The lengths lie in no buffer that is written (held is not
 * kv_len's array). A page is in one row of the table only: one that rows share would be given back by each. Calls on
 * the same pages are ordered. work: xjh_page_plan_work_bytes bytes, 16-byte aligned. */
int xjh_page_plan(const xjh_pages *p, const int32_t *held, const int32_t *n_past, const int32_t *n_new, int n_req,
                  const int32_t *n_free, int32_t *n_free_out, int T, int32_t *cu, int32_t *kv_len, int32_t *pos,
                  int32_t *slot, int32_t *status, void *work, size_t work_bytes, void *stream, char *err, size_t errlen);
size_t xjh_page_plan_work_bytes(int n_req);

/* A layer's keys and values in pages, [n_pages][Hkv][page][D] each. */
typedef struct {
    int32_t  type;               /* XJ_F16 or XJ_BF16 */
    int32_t  Hkv, D;             /* D: 64, 128 or 256 */
    int32_t  page, n_pages;      /* as in xjh_pages */
    void    *k, *v;              /* device, 16-byte aligned */
    uint64_t bytes;              /* at k and at v, at least xjh_paged_bytes each */
} xjh_paged;
/* Bytes of the keys (and of the values) of these heads, page and n_pages; 0 when they are not supported. */
uint64_t xjh_paged_bytes(const xjh_paged *c);
/* Rows k, v [T][Hkv*D] (token strides k_tok, v_tok) of `type` (XJ_F32 or the cache's) into their
 * slots: row t goes to offset slot[t] % page of page slot[t] / page, rounded to nearest (beyond the type's
 * range: infinity). A slot outside [0, n_pages * page) skips its row. The slots of a call differ. T * Hkv is at most 2^26. */
int xjh_paged_store(const xjh_paged *c, int type, const void *k, int64_t k_tok, const void *v, int64_t v_tok, int T,
                    const int32_t *slot, void *stream, char *err, size_t errlen);
/* Attention of every request's new tokens over its pages: request r's are the rows cu[r] .. cu[r+1]-1
 * of q, gate and out (elements of `type`, XJ_F32 or the cache's; rows from T on do not exist), at positions
 * kv_len[r] - n .. kv_len[r]-1, n = cu[r+1] - cu[r], and their keys and values are in the cache already.
 * Query head h (q + row*q_tok + h*q_head, D elements) of the token at p reads kv head
 * h / (H/Hkv) and sees the positions j <= p, with window > 0 only those with j > p - window or j < n_sink
 * (the first tokens stay visible); out[row*o_tok + h*D ..] = softmax(scale q.K^T) V, times
 * sigmoid(gate[row*g_tok + h*g_head ..]) when gate is not NULL. A row that sees nothing (a position
 * below 0) is 0; rows that belong to no request keep their values. table [n_req][max_blocks] as in
 * xjh_pages (max_blocks * page <= 2^30; kv_len beyond that counts as it); requests may share pages.
 * A table entry outside [0, n_pages) stands for positions that are not seen. What lies at positions
 * that a row does not see, NaN too, counts for nothing in it; a value that it sees and is not finite leaves it not finite.
 * Products of 16-bit elements are exact and sums are fp32. With 16-bit rows the weights are rounded to the cache's bits
 * by the kernel for many rows and kept to twice as many by that for few. With float rows the
 * queries and the weights enter with 22 bits over f16 (queries to 2^-40 of the row's largest element,
 * weights to 2^-33 of the row's largest) and 24 over bf16. A sum over 2^n positions of bf16 values keeps its bits down to 2^(n - 93).
 * max_new: the largest n, as far as the program knows (0: it does not); it decides which kernel runs, and a
 * larger n is right too. With max_new * H/Hkv up to 32, or T * H/Hkv where it is 0, that for few rows runs for all requests, otherwise for those of
 * at most 32 rows a kv head, if there is more than one request. By that, by the other requests and by the work area the result changes with the rounding
 * of sums, and with 16-bit rows, where the kernel changes, with that of the weights: by half a step of the type (f16 2^-11, bf16 2^-8) of
 * sum_j p_j |v_j| at most, before the result is rounded.
 * Scores (scale q.K^T) are below 2^22 in magnitude: beyond, where float scores have no fractions, rows may be 0 or not finite.
 * T * H is at most 2^27, n_req 65536, min(n_req, T) * Hkv 2^22. */
int xjh_attn_paged(const xjh_paged *c, int type, const void *q, int64_t q_tok, int64_t q_head, const void *gate, int64_t g_tok,
                   int64_t g_head, const int32_t *table, int max_blocks, const int32_t *cu, const int32_t *kv_len, int n_req,
                   int T, int max_new, int H, int window, int n_sink, float scale, void *out, int64_t o_tok, void *work,
                   size_t work_bytes, void *stream, char *err, size_t errlen);
/* The work area beyond which nothing is gained for these and any smaller T and n_req; 0 when they are not supported. */
size_t xjh_attn_paged_work_bytes(const xjh_paged *c, int type, int T, int H, int n_req, int max_new, int max_blocks);
/* The same for whole sequences that lie packed in rows: sequence s is the rows cu[s] .. cu[s+1]-1 of q, k, v, gate and
 * out (all of `type`, XJ_F32, XJ_F16 or XJ_BF16), the first at position 0; kv head g of a row at k + row*k_tok +
 * g*k_head, D elements (64, 128 or 256). Float queries, keys, values and weights enter with 24 bits, and their sums keep as many as those
 * over bf16 pages; the weights of 16-bit rows are rounded as there, by the kernel that T, n_seq and the heads select (that for few rows up to some hundred rows). Rows of k and v
 * whose addresses are multiples of 16 bytes are read faster. */
int xjh_attn_packed(int type, const void *q, int64_t q_tok, int64_t q_head, const void *k, int64_t k_tok, int64_t k_head,
                    const void *v, int64_t v_tok, int64_t v_head, const void *gate, int64_t g_tok, int64_t g_head,
                    const int32_t *cu, int n_seq, int T, int H, int Hkv, int D, int window, int n_sink, float scale, void *out,
                    int64_t o_tok, void *work, size_t work_bytes, void *stream, char *err, size_t errlen);
size_t xjh_attn_packed_work_bytes(int type, int T, int H, int Hkv, int D, int n_seq);

#ifdef __cplusplus
}
#endif
#endif /* XJ_HIP_H */
