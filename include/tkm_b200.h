/*
 * tkm_b200.h -- thin C ABI of the B200 (sm_100a) hot-path kernels.
 *
 * Plain pointers and sizes only.  Every pointer argument except those marked
 * "host" is a device pointer; `stream` is a cudaStream_t (NULL = legacy
 * default stream).  All calls are asynchronous on `stream` and return a
 * tkb_status; on failure tkb_last_error() gives a one-line reason.  A kernel
 * whose bounded internal wait ran out records a code that tkb_device_error()
 * reports (the kernel returns; the context stays usable).
 *
 * Each entry point names the reference (BSODsystem32/Tokamak v4.1.0) kernel
 * and launch site it replaces.  dtype selects the storage type of the
 * activation tensors: TKB_F32, TKB_BF16 or TKB_F16.  Parameter vectors
 * (RMSNorm gain, biases) are fp32 master copies, as in the reference
 * (NodeGpuState, src/tkm_gpu.cu:829-839).
 */
#ifndef TKM_B200_H
#define TKM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { TKB_F32 = 0, TKB_BF16 = 1, TKB_F16 = 2 } tkb_dtype;

typedef enum {
    TKB_OK = 0,
    TKB_ERR_ARG = -1,         /* invalid shape, dtype, pointer or alignment */
    TKB_ERR_CUDA = -2,        /* a CUDA runtime call failed */
    TKB_ERR_UNSUPPORTED = -3, /* shape/dtype combination not implemented */
    TKB_ERR_WORKSPACE = -4    /* workspace missing or too small */
} tkb_status;

/* Library version string. */
const char *tkb_version(void);
/* Message describing the last failing call made from this host thread. */
const char *tkb_last_error(void);
/* Synchronizes `stream`, reads and clears the device error word (0 = none).
 * Bit 0: a bounded wait inside a kernel timed out; bit 1: bad launch;
 * bit 2: device data named a page, slot or row that does not exist (the
 * access was left out). */
int tkb_device_error(unsigned int *code, void *stream);
/* Number of kernels this library launched since load (all entry points). */
unsigned long long tkb_launch_count(void);
/* Self-test of the failure path (no counterpart in the reference): one
 * kernel waits, for at most limit_ns (<= 2 s), on an mbarrier that nothing
 * arrives on, gives up like a pipeline kernel whose partner stopped, and
 * records bit 0 in the device error word (read it with tkb_device_error). */
int tkb_selftest_wait_timeout(unsigned long long limit_ns, void *stream);

/* ------------------------------------------------------------ attention
 * Packed layout of the reference (src/tkm_gpu.cu:331-338, 366-368):
 *   qkv  [B][S][(Hq + 2*Hkv)*D]  Q head h at column h*D, K head g at
 *        (Hq+g)*D, V head g at (Hq+Hkv+g)*D; query head h reads kv head
 *        h / (Hq/Hkv).
 *   out  [B][S][Hq*D]
 *   lse  [B*Hq][S] fp32, natural log of the softmax denominator.
 * D must be 64 or 128; Hq % Hkv == 0.  Causal masks key > query.
 * bf16/f16 run on tcgen05 tensor cores (fp32 accumulation); f32 runs fp32 FMA. */

/* Replaces k_gqa_flash_attn_tc_fwd<HEAD_DIM> (src/tkm_gpu.cu:302-438),
 * launched at src/tkm_gpu.cu:1252-1265. */
int tkb_gqa_attn_fwd(const void *qkv, void *out, float *lse,
                     int B, int S, int Hq, int Hkv, int D, float scale, int causal,
                     int dtype, void *stream);

/* Workspace bytes tkb_gqa_attn_bwd needs (per-row Delta and LSE*log2(e), fp32). */
size_t tkb_gqa_attn_bwd_workspace(int B, int S, int Hq, int D, int dtype);

/* Workspace bytes with which tkb_gqa_attn_bwd keeps every dS tile (16-bit,
 * B * Hq * tiles * 32 KB; causal stores only the lower triangle of tiles)
 * and computes dQ as a GEMM over them instead of recomputing S, P and dP.
 * Equal to tkb_gqa_attn_bwd_workspace when that area would exceed 32 GiB.
 * Any size between the two selects the recompute path. */
size_t tkb_gqa_attn_bwd_workspace_ex(int B, int S, int Hq, int D, int causal, int dtype);

/* Replaces k_gqa_flash_attn_tc_bwd<HEAD_DIM> (src/tkm_gpu.cu:440-598),
 * launched at src/tkm_gpu.cu:1389-1403.  Writes all of dqkv (dQ, dK, dV
 * slices; the reference leaves dK/dV wrong, src/tkm_gpu.cu:588-596).
 * dK/dV are summed over the query heads that share a kv head. */
int tkb_gqa_attn_bwd(const void *qkv, const void *out, const void *dout, const float *lse,
                     void *dqkv, void *workspace, size_t workspace_bytes,
                     int B, int S, int Hq, int Hkv, int D, float scale, int causal,
                     int dtype, void *stream);

/* ------------------------------------------------------------ residual + RMSNorm
 * Replaces the residual Add plasma group and the RMSNorm plasma group
 * emitted by src/tkm_codegen.c:484-523 (specs src/tkm_registry.c:228-245,
 * 435-439).  s = x + r (r may be NULL; s may be NULL when r is NULL),
 * istd[row] = 1/sqrt(mean(s^2) + eps), y = s * istd * gamma.  C even. */
int tkb_add_rmsnorm_fwd(const void *x, const void *r, void *s, void *y,
                        const float *gamma, float *istd, int rows, int C, float eps,
                        int dtype, void *stream);

size_t tkb_add_rmsnorm_bwd_workspace(int rows, int C);

/* Backward (src/tkm_codegen.c:525-624 for an RMSNorm group; spec
 * src/tkm_registry.c:239-245): dx = istd*(g*dy - xh*mean(g*dy*xh)) + ds_skip
 * with xh = s*istd (ds_skip may be NULL); dgamma += sum_rows(dy*xh)
 * (dgamma may be NULL). */
int tkb_add_rmsnorm_bwd(const void *dy, const void *s, const float *gamma, const float *istd,
                        const void *ds_skip, void *dx, float *dgamma,
                        void *workspace, size_t workspace_bytes,
                        int rows, int C, int dtype, void *stream);

/* ------------------------------------------------------------ SwiGLU twin epilogue
 * Replaces the twin-branch plasma group (src/tkm_codegen.c:511-518 fwd,
 * 540-598 bwd; rule src/tkm_registry.c:653-686).  gu [rows][2F] holds the
 * fused gate|up GEMM output; h = silu(g + bg) * (u + bu) [rows][F].
 * bg/bu may be NULL (zero). */
int tkb_swiglu_fwd(const void *gu, const float *bg, const float *bu, void *h,
                   int rows, int F, int dtype, void *stream);

size_t tkb_swiglu_bwd_workspace(int rows, int F);

/* dgu [rows][2F] overwritten; dbg/dbu accumulated (may be NULL). */
int tkb_swiglu_bwd(const void *dh, const void *gu, const float *bg, const float *bu,
                   void *dgu, float *dbg, float *dbu, void *workspace, size_t workspace_bytes,
                   int rows, int F, int dtype, void *stream);

/* ------------------------------------------------------------ QKV prep
 * Replaces the QKV-prep plasma group (src/tkm_codegen.c:211-295, rotation
 * 43-70; rule src/tkm_registry.c:688-770).  Row layout as the packed qkv
 * above; position = row % S.  Bias add on every column; QKNorm (per-head
 * RMS over D, eps 1e-5, gain qk_gain[(Hq+Hkv)*D]) and RoPE on the Q and K
 * heads.  RoPE rotates pair i of a head by pos * f, f = theta^(-i/D), with the
 * reference's frequency adjustment when rope_scale > 1: with w = 2 pi / f, f is
 * divided by rope_scale where w > octx/low_freq_factor, and multiplied by
 * 1 - t (1 - 1/rope_scale), t = (octx/w - low) / (high - low), where
 * octx/high_freq_factor <= w <= octx/low.  This ramp runs from the whole
 * division at octx/high to none at octx/low, the other way round than
 * Llama 3's published rule, and jumps at both ends: models trained here and
 * run here agree, weights trained elsewhere with that rule do not.
 * save_istd [rows][Hq+Hkv] (needed with QKNorm). */
int tkb_qkv_prep_fwd(const void *in, const float *bias, const float *qk_gain, void *out,
                     float *save_istd, int rows, int S, int Hq, int Hkv, int D,
                     int has_qknorm, int has_rope, float theta, float rope_scale,
                     float low_freq_factor, float high_freq_factor,
                     float original_context_length, int dtype, void *stream);

size_t tkb_qkv_prep_bwd_workspace(int rows, int Hq, int Hkv, int D);

/* din accumulated (+=), dbias and dgain accumulated (may be NULL). */
int tkb_qkv_prep_bwd(const void *dout, const void *in, const float *bias, const float *qk_gain,
                     const float *save_istd, void *din, float *dbias, float *dgain,
                     void *workspace, size_t workspace_bytes,
                     int rows, int S, int Hq, int Hkv, int D,
                     int has_qknorm, int has_rope, float theta, float rope_scale,
                     float low_freq_factor, float high_freq_factor,
                     float original_context_length, int dtype, void *stream);

/* ------------------------------------------------------------ softmax, losses
 * Replaces k_softmax_fwd_h / k_softmax_bwd_h (src/tkm_gpu.cu:600-630,
 * launches 1270-1274 and 1409-1412).  dx is accumulated (+=). */
int tkb_softmax_fwd(const void *x, void *p, int rows, int C, int dtype, void *stream);
int tkb_softmax_bwd(const void *p, const void *dp, void *dx, int rows, int C, int dtype, void *stream);

size_t tkb_softmax_loss_workspace(int rows);

/* Replaces k_softmax_loss_fwd_bwd_h (src/tkm_gpu.cu:632-682, launch
 * 1275-1284).  kind 0 cross-entropy, 1 focal(gamma), 2 Brier.  labels: one
 * int32 per row (the reference reads uint8 labels[r], src/tkm_gpu.cu:646).
 * loss += mean over rows (summed in a fixed order); dlogits = dloss/dlogits
 * (may be NULL); correct += number of rows whose argmax equals the label
 * (may be NULL).  C <= 32768.  logits and dlogits 16-byte aligned when
 * C % 8 == 0 (else aligned to two elements); TKB_ERR_ARG otherwise. */
int tkb_softmax_loss(const void *logits, const int32_t *labels, void *dlogits,
                     float *loss, int *correct, void *workspace, size_t workspace_bytes,
                     int rows, int C, int kind, float gamma, int dtype, void *stream);

/* Variant of tkb_softmax_loss for callers that cannot allocate device memory
 * (no counterpart in the reference).  Code running while a CUDA graph is being
 * captured in global mode cannot call cudaMalloc, and foreign-language callers
 * may hold only raw device pointers from another framework's allocator; this
 * entry point needs no workspace.  Its per-row scratch is a fixed array inside
 * the library (1 MiB per GPU, held until exit), so rows must be at most
 * 262144; larger calls return TKB_ERR_ARG.  The first call on a device looks up
 * the array's address for that device: make it before any stream capture.
 * All calls share the array; calls that overlap on the GPU race on it.
 * Alignment as for tkb_softmax_loss. */
int tkb_softmax_loss_noalloc(const void *logits, const int32_t *labels, void *dlogits,
                             float *loss, int *correct, int rows, int C, int kind, float gamma,
                             int dtype, void *stream);

/* ------------------------------------------------------------ SGD
 * Replaces k_tkm_multi_tensor_sgd (src/tkm_gpu.cu:684-720, launch
 * 1417-1420).  `table` is device memory holding n_tensors tkb_sgd_tensor
 * records.  g += wd*p when apply_wd, v = momentum*v + g,
 * p -= lr*(momentum*v + g), lowp (if set) refreshed, *seed += 0x9E3779B9. */
typedef struct {
    float *master;
    float *vel;
    const float *grad;
    void *lowp;          /* 16-bit copy of master, or NULL */
    long long n;
    int apply_wd;
    int lowp_dtype;      /* TKB_BF16 or TKB_F16 */
} tkb_sgd_tensor;

int tkb_sgd_step(const tkb_sgd_tensor *table, int n_tensors, const float *lr,
                 float momentum, float weight_decay, uint32_t *seed, void *stream);

/* ------------------------------------------------------------ GEMM
 * Replaces the cuBLAS GEMMs of the FC layers (cublasGemmEx at
 * src/tkm_gpu.cu:1207-1236 forward, 1330-1372 input and weight gradients):
 * C[M][N] = A B (+ C when accumulate, + bias[n] when bias is not NULL),
 * bf16 operands, fp32 accumulation on the tcgen05 tensor cores.
 *   a_trans 0: A stored [M][K], lda elements per row; 1: A stored [K][M].
 *   b_trans 0: B stored [K][N], ldb elements per row; 1: B stored [N][K].
 *   c_dtype TKB_BF16 or TKB_F32 (C row-major, ldc elements per row).
 * Forward X W: (X, 0, W, 0); input gradient dY W^T: (dY, 0, W, 1); weight
 * gradient X^T dY: (X, 1, dY, 0).  lda and ldb must be multiples of 8, ldc
 * of 8 (bf16) or 4 (fp32); pointers 16-byte aligned.  bias needs a_trans 0.
 * An fp32 C whose tiles would leave the GPU's last wave mostly idle (weight
 * gradients: few output tiles, long K) splits K into partial sums kept in
 * `workspace` and added in a fixed order (deterministic); give it
 * tkb_gemm_workspace(M, N, K, c_dtype) bytes, or NULL to run unsplit. */
size_t tkb_gemm_workspace(int M, int N, int K, int c_dtype);
int tkb_gemm(const void *A, long long lda, int a_trans, const void *B, long long ldb, int b_trans,
             void *C, long long ldc, int c_dtype, int accumulate, const float *bias,
             int M, int N, int K, void *workspace, size_t workspace_bytes, void *stream);

/* The twin [gate | up] FC with its SwiGLU epilogue in one kernel (replaces
 * the cuBLAS GEMM of FC_TWIN_FUSED, src/tkm_gpu.cu:1207-1236, and the twin
 * epilogue group emitted at src/tkm_codegen.c:511-598): with [G | U] = A B,
 * A stored [M][K], B stored [K][2F] (gate columns 0..F-1, up F..2F-1),
 * GU[M][2F] receives [G | U] in bf16 (what the backward replays from) and
 * H[M][F] = SiLU(G + bias_gate) * (U + bias_up), computed from the bf16 G
 * and U.  F must be a multiple of 8; the biases may be NULL. */
int tkb_gemm_swiglu(const void *A, long long lda, const void *B, long long ldb, int F,
                    const float *bias_gate, const float *bias_up, void *GU, long long ldgu,
                    void *H, long long ldh, int M, int K, void *stream);

/* The LM head and its softmax cross-entropy without the logits in memory
 * (replaces the cuBLAS head GEMM, the Bias group and k_softmax_loss_fwd_bwd_h
 * with kind 0, src/tkm_gpu.cu:632-682 and 1275-1284): logits = X W + bias for
 * X [rows][d] (ldx per row), W [d][V] (ldw per row), bias [V] (may be NULL),
 * computed tile by tile on the tcgen05 CTA-pair GEMM.  A first pass keeps
 * per-row statistics (tile maxima, sums of exponentials, argmax, the label's
 * logit); *loss += mean over rows of -ln(max(p_label, 1e-7)); *correct (may
 * be NULL) += rows whose first argmax is the label; when dlogits is not
 * NULL a second pass recomputes each tile and writes d logits = (softmax -
 * onehot) / rows in bf16 ([rows][ldd]).  Every logit is recomputed instead of
 * stored: the [rows][V] logits buffer is never written.  Workspace:
 * tkb_lmhead_ce_workspace(rows, V) bytes, 256-byte aligned.  d and V must be
 * multiples of 8. */
size_t tkb_lmhead_ce_workspace(int rows, int V);
int tkb_lmhead_ce(const void *X, long long ldx, const void *W, long long ldw, const float *bias,
                  const int32_t *labels, void *dlogits, long long ldd, float *loss, int *correct,
                  void *workspace, size_t workspace_bytes, int rows, int d, int V, void *stream);

/* ------------------------------------------------------------ paged key-value cache
 * Generation (no counterpart in the reference, which runs whole sequences
 * only).  The cache of one attention layer: a pool of pages, each holding
 * page_size tokens of every kv head, and per sequence the list of its pages.
 *   k, v         [n_pages][Hkv][page_size][D] of `dtype`, pages page_stride
 *                elements apart (so K and V, or several layers, may share one
 *                pool); 16-byte aligned, page_stride a multiple of 16 bytes.
 *   pos          [n_pages][Hkv][page_size] position of the token a slot
 *                holds, or NULL (needed by tkb_kv_evict).
 *   weight       [n_pages][Hkv][page_size] accumulated attention weight of a
 *                slot, or NULL (needed by tkb_kv_evict).  pos and weight
 *                16-byte aligned.
 *   block_table  [B][max_pages]; slot j of sequence b lies in page
 *                block_table[b][j / page_size].  Only the entries that the
 *                lengths reach are read.
 *   seq_lens     [B] tokens each sequence holds (0 allowed).
 * page_size: a multiple of 16, at most 1024; D 64 or 128; B at most 4096.
 * The struct itself is read on the host, during the call; everything it
 * points to is device memory and is read when the kernels run, so a captured
 * CUDA graph follows the lengths and tables.  A page outside [0, n_pages)
 * or a length above max_pages * page_size sets bit 2 of the device error
 * word: such slots count as not held, such rows are not written.  Sequences
 * may share pages that only tkb_paged_attn_decode without `accumulate` and
 * tkb_paged_attn_chunk read. */
typedef struct {
    void *k, *v;
    int32_t *pos;
    float *weight;
    const int32_t *block_table;
    const int32_t *seq_lens;
    long long page_stride;
    int n_pages, page_size, max_pages;
    int B, Hkv, D, dtype;
} tkb_kv_cache;

/* Lengths on the device: seq_lens[b] = min(seq_lens[b] + n_b, limit) and
 * seen[b] += n_b (seen, the tokens a sequence has had so far, may be NULL),
 * with n_b = row_start[b + 1] - row_start[b], or `add` when row_start is
 * NULL.  Before rows are appended: limit INT32_MAX.  A sequence may then count
 * more tokens than its pages hold: the append leaves out the rows that have no
 * slot, the attention reads the full cache, each sets bit 2 of the device
 * error word, and an eviction brings the length back.  (A limit that cuts
 * the new rows off, which sets the bit here, moves them onto the last slots
 * below it, which hold tokens: tkb_kv_append counts back from seq_lens.)  After
 * an eviction: add 0 with limit `budget`. */
int tkb_kv_lens(int32_t *seq_lens, int32_t *seen, const int32_t *row_start, int add, int limit, int B, void *stream);

/* New tokens enter the cache.  Packed rows qkv [rows][(Hq + 2*Hkv)*D]
 * (qkv_stride elements apart) get tkb_qkv_prep_fwd's bias, QKNorm and RoPE
 * (same parameters, its frequency adjustment among them), except that the
 * position is the token's own:
 * row_start [B + 1] gives the rows of each sequence (NULL: row b belongs to
 * sequence b and rows == B); with n_b rows, row i of sequence b goes to slot
 * seq_lens[b] - n_b + i and stands at position seen[b] - n_b + i (seen NULL:
 * seq_lens).  seq_lens and seen therefore already count the new rows
 * (tkb_kv_lens).  K and V go to the slot, the position to pos, 0 to weight
 * (where present).  out (may be NULL) gets the prepared row: its Hq*D query
 * columns, or with out_full the whole packed row, as tkb_gqa_attn_fwd and
 * tkb_paged_attn_decode take it.  Rows that have no slot (n_b > seq_lens[b],
 * a slot past max_pages * page_size, a bad page) are not stored and set bit 2
 * of the device error word; their out is written.  A sequence with seen[b]
 * below 0 takes no part: its rows are not stored and set no bit. */
int tkb_kv_append(const tkb_kv_cache *cache, const void *qkv, long long qkv_stride, const float *bias,
                  const float *qk_gain, void *out, long long out_stride, int out_full, const int32_t *row_start,
                  const int32_t *seen, int rows, int Hq, int has_qknorm, int has_rope, float theta,
                  float rope_scale, float low_freq_factor, float high_freq_factor,
                  float original_context_length, void *stream);

/* Attention of one new token per sequence over its cached tokens: for query
 * head h (kv head h / (Hq/Hkv)) s_j = scale * q . k_j over the seq_lens[b]
 * slots, out = sum_j softmax(s)_j v_j, lse = ln sum_j exp(s_j).  q and out
 * [B] rows of Hq*D (q_stride, out_stride elements apart, 16-byte aligned),
 * lse [B][Hq] fp32 (may be NULL).  A sequence that holds nothing gets out 0
 * and lse -inf.  With `accumulate`, weight[slot] of each kv head also grows by
 * the sum over its query heads of softmax(s)_slot.  NaN in q, k or v reaches
 * the heads that use it, and so does an infinite v (NaN where its probability
 * is below the fp32 range).  The work is cut over the cached lengths and joined
 * in a fixed order: equal inputs give equal bits.
 * workspace: tkb_paged_attn_decode_workspace bytes, 256-byte aligned, zeroed
 * before its first use; every call leaves it fit for the next one, of any
 * cache and shape that it is large enough for.  Calls that may overlap need
 * workspaces of their own. */
size_t tkb_paged_attn_decode_workspace(const tkb_kv_cache *cache, int Hq, int accumulate);
int tkb_paged_attn_decode(const tkb_kv_cache *cache, const void *q, long long q_stride, void *out,
                          long long out_stride, float *lse, int Hq, float scale, int accumulate,
                          void *workspace, size_t workspace_bytes, void *stream);

/* Eviction by accumulated attention weight.  Every (sequence, kv head) that
 * holds more than `budget` tokens keeps budget of them: those within the
 * newest `recent` positions (pos >= seen[b] - recent) and the first `sinks`
 * (pos < sinks), then the others by weight, largest first, equal weights by
 * the lower slot (a NaN weight counts as the lowest).  Kept tokens in slots
 * budget and above move, with pos and weight, into the freed slots below, in
 * ascending order; slots budget and above are then free.  Slots hold no
 * order: positions do.  recent + sinks <= budget.  seq_lens is left as it is,
 * since layers share it: call tkb_kv_lens(seq_lens, NULL, NULL, 0, budget, B)
 * after the last layer.  workspace: tkb_kv_evict_workspace bytes, 16-byte
 * aligned; no state is kept in it. */
size_t tkb_kv_evict_workspace(const tkb_kv_cache *cache);
int tkb_kv_evict(const tkb_kv_cache *cache, const int32_t *seen, int budget, int recent, int sinks,
                 void *workspace, size_t workspace_bytes, void *stream);

/* ------------------------------------------------------------ many requests at once
 * Attention of a chunk of new tokens per sequence over its cached tokens:
 * pieces of prompts after earlier pieces, whole prompts, drafted tokens, or
 * single tokens, each sequence with its own number of rows.  row_start
 * [B + 1] gives the rows of each sequence (NULL: row b belongs to sequence b
 * and rows == B); they are the last n_b of its seq_lens[b] tokens and already
 * in the cache (tkb_kv_lens, tkb_kv_append): row i of sequence b attends over
 * slots 0 .. seq_lens[b] - n_b + i, in whatever order the older ones lie (after
 * an eviction).  For query head h (kv head h / (Hq/Hkv)): s_j = scale * q . k_j,
 * out = sum_j softmax(s)_j v_j, lse = ln sum_j exp(s_j).  q and out [rows] of
 * Hq*D (q_stride, out_stride elements apart, 16-byte aligned, not
 * overlapping), lse [rows][Hq] fp32 (may be NULL).  scale is positive.
 * bf16/f16 run on tcgen05 tensor cores with the probabilities rounded to the
 * type and sums in fp32; f32 runs fp32 FMA.  NaN or an infinity in q, k or v
 * reaches the rows that see it and no others.  A row that sees no slot (its
 * sequence counts fewer tokens than rows, or its pages are bad) gets out 0
 * and lse -inf.  A row_start that does not ascend inside [0, rows], a length
 * or page that does not exist sets bit 2 of the device error word; rows of no
 * sequence keep their out and lse.  Equal inputs give equal bits.
 * workspace: tkb_paged_attn_chunk_workspace bytes, 256-byte aligned; no state
 * is kept in it.  Calls that may overlap need workspaces of their own. */
size_t tkb_paged_attn_chunk_workspace(const tkb_kv_cache *cache, int rows, int Hq);
int tkb_paged_attn_chunk(const tkb_kv_cache *cache, const void *q, long long q_stride, void *out,
                         long long out_stride, float *lse, const int32_t *row_start, int rows, int Hq,
                         float scale, void *workspace, size_t workspace_bytes, void *stream);

/* Block tables from the lengths of the requests.  The pages of a pool are
 * owned by the sequences (block_table [B][max_pages], of which the first
 * held[b] entries of row b are in use) or free: free_pages [n_pages] is a
 * stack of *n_free page numbers.  Sequence b needs ceil(lens[b] / page_size)
 * pages, at most max_pages.  First the sequences that hold more give the
 * surplus back: their last entries, by sequence and then by entry, are pushed
 * in that order, and become -1.  Then those that hold fewer are served from the
 * top of the stack, in the order of the sequences and of their entries, each
 * whole or not at all: up to the first whose need, with the needs of all before
 * it, exceeds the stack; it and those after it that need pages get none.
 * Written: block_table, held, free_pages, n_free, and granted[b] (may be
 * NULL): 1 when sequence b's pages hold all its tokens.  Entries of
 * free_pages above *n_free keep what they held.
 * slots (may be NULL) gets, for each of `rows` rows, the place of its token in
 * the pool, page * page_size + slot in the page, for callers that move tokens
 * themselves: row_start as for tkb_kv_append, lens counting the new rows; -1
 * for a row without a place.  (Without slots, rows only helps to choose the
 * launch: about how many tokens have come and gone since the call before; 0
 * for a step.)  One call for a cache serves all layers that
 * share the table.  Lengths below 0, counts outside their range and more free
 * pages than n_pages set bit 2 of the device error word and are cut to the
 * range.  A number outside [0, n_pages) among the pages that move or that hold
 * a row sets it too: it moves like the others, its rows have no place, and a
 * sequence that is given one is not granted (what it held before is not
 * looked at).
 * B at most 4096, B * max_pages below 2^30, page_size 1 to 1024. */
int tkb_kv_pages(int32_t *block_table, int32_t *held, const int32_t *lens, int32_t *free_pages, int32_t *n_free,
                 int32_t *granted, int64_t *slots, const int32_t *row_start, int rows, int B, int max_pages,
                 int page_size, int n_pages, void *stream);

/* Low-rank adapters of many requests beside a shared projection: for every
 * row r of a sequence with adapter i = adapter[b] >= 0
 *   out_r = y_r + scale[i] * (x_r A_i) B_i
 * with x [rows][K], y (the shared projection's output) and out [rows][N] (out
 * may be y, at the same stride), A [n_adapters][K][R] and B [n_adapters][R][N],
 * all of one dtype, rows x_stride, y_stride, out_stride elements apart; scale
 * [n_adapters] fp32 (NULL: 1).  Products and sums are fp32 and the result is
 * rounded once; in 16-bit types x A enters the second product as two 16-bit
 * parts, off by at most 2^-16 of it in bf16 and 2^-22 in f16.  NaN and
 * infinities in x, A and y reach their rows as the formula has them; those of
 * B do too, but in 16-bit types an infinite value may give NaN.
 * adapter[b] = -1: out_r = y_r.  Rows of no sequence are left
 * as they were.  An adapter that does not exist counts as -1 and sets bit 2 of
 * the device error word.  K, N and the strides: multiples of 16 bytes, the
 * pointers 16-byte aligned; R a multiple of 8 up to 128; B at most 4096, rows at
 * most 2^21.
 * The plan sorts the rows by adapter: tkb_lora_plan writes it from adapter [B]
 * and row_start (as for tkb_kv_append), once for all projections that take
 * the same rows, and tkb_lora_add reads it.  plan: tkb_lora_plan_bytes,
 * workspace: tkb_lora_workspace bytes, both 256-byte aligned. */
size_t tkb_lora_plan_bytes(int B, int rows, int n_adapters);
int tkb_lora_plan(const int32_t *adapter, const int32_t *row_start, int B, int rows, int n_adapters, void *plan,
                  size_t plan_bytes, void *stream);
size_t tkb_lora_workspace(int rows, int R);
int tkb_lora_add(const void *plan, const void *x, long long x_stride, const void *A, const void *B_, const float *scale,
                 const void *y, long long y_stride, void *out, long long out_stride, int B, int rows, int n_adapters,
                 int K, int N, int R, int dtype, void *workspace, size_t workspace_bytes, void *stream);

/* ------------------------------------------------------------ sampling
 * One token per row of logits [rows][V] (ld elements apart) from given
 * uniform numbers u[rows] in [0, 1); temperature, top_k, top_p, min_p are per
 * row, each array may be NULL (1, off, off, off).  With x the row, m its
 * maximum: every token has the whole weight w = rint(exp(-(m - x) * (1/T)) *
 * 2^31), so that sums of weights are exact and the result does not depend on
 * their order.  In the order of falling logits, equal ones by index, the
 * tokens kept are those of weight > 0 that are among the first top_k
 * (top_k <= 0: all); whose preceding weights sum to less than top_p times
 * the weight of those (top_p >= 1: all; the first always); and whose weight
 * is at least min_p * 2^31.  The token is the first in index order at
 * which the running sum of kept weights passes u times their total.
 *   token[r]   the token, -1 when no logit is above -inf
 *   logprob[r] ln of its share of the kept weight (may be NULL)
 *   kept[r]    number of tokens kept (may be NULL)
 * temperature 0 (or anything not above 0) takes the largest logit, the lowest
 * index among equals, with logprob 0.  NaN logits count as -inf; +inf shares
 * the whole weight.  top_p and u act as multiples of 2^-32.
 * V at most 2^18. */
int tkb_sample_logits(const void *logits, long long ld, const float *u, const float *temperature,
                      const int32_t *top_k, const float *top_p, const float *min_p, int32_t *token,
                      float *logprob, int32_t *kept, int rows, int V, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif
