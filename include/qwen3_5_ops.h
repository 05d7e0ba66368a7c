/*
 * C interface of libqwen3_5_hip.so: the Qwen3.5 hybrid-decoder prefill operations for
 * AMD Instinct MI355X (gfx950), plus the few HIP runtime calls a caller needs so that
 * it loads this one library at run time and never links HIP itself.
 *
 * Drop-in boundary: every declaration in the "reference interface" sections has the
 * name, argument order, argument meaning, return convention and ABI version of the
 * reference's src/backends/cuda/qwen3_5/ops.h (ABI v6, ops.h:16-138), which its Rust
 * executor resolves by name (src/models/qwen3_5/native/src/cuda.rs:50-133). Each is
 * cited below with the ops.h line it replaces.  Declarations in the "additions"
 * section are new symbols; the reference has no counterpart and existing symbols keep
 * their semantics.
 *
 * Conventions (ops.h:1-9): tensors are row-major and bfloat16 unless a pointer is
 * float; token-major [T, heads, dim]; GQA head h reads kv head h / (H / HK).  Every
 * operation queues work on `stream` (a hipStream_t passed as void*), allocates
 * nothing, never waits on the host, and returns 0 or a hipError_t code (hipBLASLt
 * failures of the GEMMs are returned as 1000 + hipblasStatus_t).  Argument errors
 * return hipErrorInvalidValue.  Only cs1_upload / cs1_download synchronize.
 */
#pragma once

#include <stddef.h>
#include <stdint.h>

/* ops.h:16 -- the interface version the Rust loader checks (cuda.rs:12, 160-165). */
#define CS1_ABI_VERSION 6

#ifdef __cplusplus
extern "C" {
#endif

/* ---- reference interface: runtime (ops.h:22-44, runtime.cu:7-74) ---- */

uint32_t cs1_abi_version(void);                                            /* ops.h:24 */
const char* cs1_error_string(int code);                                    /* ops.h:25 */
int cs1_set_device(int device);                                            /* ops.h:26 */
int cs1_malloc(void** ptr, size_t bytes);                                  /* ops.h:27 */
int cs1_free(void* ptr);                                                   /* ops.h:28 */
int cs1_stream_create(void** stream);                                      /* ops.h:29 */
int cs1_stream_sync(void* stream);                                         /* ops.h:30 */
int cs1_stream_destroy(void* stream);                                      /* ops.h:31 */
int cs1_graph_begin(void* stream);                                         /* ops.h:32 */
int cs1_graph_end(void* stream, void** exec);                              /* ops.h:33 */
int cs1_graph_launch(void* exec, void* stream);                            /* ops.h:34 */
int cs1_graph_destroy(void* exec);                                         /* ops.h:35 */
/* Copy and wait for the copy. */
int cs1_upload(void* dst, const void* src, size_t bytes, void* stream);   /* ops.h:37 */
int cs1_download(void* dst, const void* src, size_t bytes, void* stream); /* ops.h:38 */
/* Device-to-device copy, queued only. */
int cs1_copy_dd(void* dst, const void* src, size_t bytes, void* stream);  /* ops.h:40 */
/* Pitched device-to-device copy: height rows of width bytes. */
int cs1_copy2d(void* dst, size_t dpitch, const void* src, size_t spitch, size_t width, size_t height,
               void* stream);                                              /* ops.h:43 */

/* ---- reference interface: operations (ops.h:46-126) ---- */

/* out[t] = table[ids[t]], rows of D (D % 8 == 0).                            ops.h:48 */
int cs1_embed(const int32_t* ids, const void* table, void* out, int T, int D, void* stream);

/* Zero-centred RMSNorm over rows of D: out = x * rsqrt(mean x^2 + eps) * (1 + w).  ops.h:51 */
int cs1_rms_norm(const void* x, const void* w, void* out, int rows, int D, float eps, void* stream);

/* residual = bf16(residual + delta); out = cs1_rms_norm(residual).             ops.h:54 */
int cs1_add_rms_norm(void* residual, const void* delta, const void* w, void* out, int rows, int D, float eps,
                     void* stream);

/* Gated RMSNorm of the GDN output x [T, H, 128] with z [T, H*128] in rows of ldz:
 * out = bf16(round(w * round(x * rsqrt(mean x^2 + eps))) * silu(z)).          ops.h:59 */
int cs1_gated_rms_norm(const void* x, const void* z, int ldz, const void* w, void* out, int T, int H, int D,
                       float eps, void* stream);

/* Depthwise causal conv1d (kernel 4, no bias, zero left padding) + SiLU over qkv [T, ld],
 * split into q [T, key_dim], k [T, key_dim], v [T, value_dim]; w is [2*key_dim+value_dim, 4].
 *                                                                               ops.h:64 */
int cs1_gdn_conv(const void* qkv, int ld, const void* w, void* q, void* k, void* v, int T, int key_dim,
                 int value_dim, void* stream);

/* beta = bf16(sigmoid(b)); g = -exp(A_log) * softplus(a + dt_bias) (float32); b, a are
 * [T, H] in rows of ld.                                                         ops.h:69 */
int cs1_gdn_gates(const void* b, const void* a, int ld, const void* A_log, const void* dt_bias, void* beta,
                  float* g, int T, int H, void* stream);

/* Chunked gated delta rule (chunk 64, dk = dv = 128), q and k L2-normalised inside, q
 * scaled by `scale`: q, k [T, HK, 128], v [T, H, 128], g float [T, H], beta [T, H],
 * o [T, H, 128].  The caller owns the workspace of cs1_gdn_workspace_floats(T, H) floats.
 *                                                                            ops.h:73-75 */
size_t cs1_gdn_workspace_floats(int T, int H);
int cs1_gdn_prefill(const void* q, const void* k, const void* v, const float* g, const void* beta, void* o,
                    float* workspace, int T, int H, int HK, float scale, void* stream);

/* Same scan with an explicit float32 state: s_in [H, 128, 128] (K-major) before the
 * window, or null for zero; s_out receives the state after it, or null.  T == 0 copies
 * s_in to s_out (zeroes s_out when s_in is null).  A continuation that starts at a
 * multiple of 64 repeats the one-pass arithmetic bit for bit.                ops.h:82-84 */
int cs1_gdn_prefill_x(const void* q, const void* k, const void* v, const float* g, const void* beta, void* o,
                      float* workspace, int T, int H, int HK, float scale, const void* s_in, void* s_out,
                      void* stream);

/* Attention inputs: q and gate from qg [T, Hq, 2*Dh], k from kr [T, Hk, Dh], both in
 * rows of ld; per-head zero-centred RMSNorm, then rotate_half RoPE on the first 2*half
 * dims with cos/sin [T, half] (bf16).  Writes q [T, Hq, Dh], gate [T, Hq*Dh], k [T, Hk, Dh].
 * The reference accepts Dh = 256 only; this build also accepts Dh = 128.      ops.h:89 */
int cs1_attn_prep(const void* qg, const void* kr, int ld, const void* qw, const void* kw, const void* cos,
                  const void* sin, void* q, void* gate, void* k, int T, int Hq, int Hk, int Dh, int half, float eps,
                  void* stream);

/* Causal GQA attention, Dh = 256: q [T, Hq, Dh], k [T, Hk, Dh], v [T, Hk, Dh] in rows of
 * ldv; out [T, Hq, Dh].                                                        ops.h:95 */
int cs1_attention(const void* q, const void* k, const void* v, int ldv, void* out, int T, int Hq, int Hk, int Dh,
                  float scale, void* stream);

/* Same, with the sigmoid gate [T, Hq, Dh] fused into the epilogue: out =
 * bf16(round(attn) * round(sigmoid(gate))), bit-identical to cs1_attention followed by
 * cs1_sigmoid_gate.  gate must be non-null when T > 0.                        ops.h:101 */
int cs1_attention_gated(const void* q, const void* k, const void* v, int ldv, const void* gate, void* out, int T,
                        int Hq, int Hk, int Dh, float scale, void* stream);

/* Windowed variant: k and v cover rows [0, T); q, gate and out rows [q_base, T) of
 * buffers indexed from row 0.  q_base % 64 == 0.                               ops.h:108 */
int cs1_attention_gated_prefix(const void* q, const void* k, const void* v, int ldv, const void* gate, void* out,
                               int T, int Hq, int Hk, int Dh, float scale, int q_base, void* stream);

/* x = bf16(x * round(sigmoid(gate))), n elements.                              ops.h:113 */
int cs1_sigmoid_gate(void* x, const void* gate, size_t n, void* stream);

/* out [T, I] = bf16(round(silu(gate)) * up) from gate_up [T, 2I] (gate first), rows of ld.
 *                                                                              ops.h:116 */
int cs1_silu_mul(const void* gate_up, int ld, void* out, int T, int I, void* stream);

/* y [M, N] (rows of ldy) = x [M, K] * w [N, K]^T, bf16 in and out, float32 accumulation,
 * with one fixed plan per shape and workspace size: this library's kernel, or hipBLASLt's first
 * heuristic choice without atomic split-K accumulation.  Never waits on the host.  A handle serves
 * one thread and one stream at a time: its workspace holds the partial sums of split products, so
 * calls in flight on two streams need a handle each.                       ops.h:120-124 */
void* cs1_gemm_create(size_t workspace_bytes);
void cs1_gemm_destroy(void* gemm);
int cs1_gemm(void* gemm, const void* x, const void* w, void* y, int M, int N, int K, int ldy, void* stream);

/* Additive (no counterpart in ops.h): cs1_gemm with the shape's plan re-chosen by timing up
 * to 16 of hipBLASLt's heuristic candidates and this library's kernel on these operands, fastest
 * kept (y holds the kept kernel's result on return). Unlike cs1_gemm it synchronises the stream, so it must
 * not be called under stream capture (returns hipErrorStreamCaptureUnsupported). The
 * choice follows measured times, so two processes may keep different kernels for a shape;
 * without this call every plan is the deterministic default. */
int cs1_gemm_tune(void* gemm, const void* x, const void* w, void* y, int M, int N, int K, int ldy, void* stream);

/* ---- reference interface: vision tower (ops.h:127-138) ----
 * Out of scope for this build (the vision tower is not on the text prefill path).  The
 * symbols exist so that the reference loader, which resolves every name, can load the
 * library (cuda.rs:33-46); each returns hipErrorNotSupported. */
int cs1_vision_linear(void* gemm, const void* x, const void* w, const void* bias, void* y, int M, int N, int K,
                      void* stream);
int cs1_gemm_f32(void* gemm, const float* x, const float* w, float* y, int M, int N, int K, void* stream);
int cs1_vision_norm(const void* x, const void* w, const void* b, void* y, int rows, int d, void* stream);
int cs1_vision_position(void* x, const void* table, const int* indices, const float* weights, int n, void* stream);
int cs1_vision_rope(const void* qkv, const float* co, const float* si, void* q, void* k, int n, void* stream);
int cs1_vision_attention(const void* q, const void* k, const void* v, void* out, int n, void* stream);
int cs1_vision_bias(void* x, const void* bias, size_t n, int d, void* stream);
int cs1_vision_gelu(void* x, size_t n, int exact, void* stream);
int cs1_vision_add(void* x, const void* delta, size_t n, void* stream);
int cs1_vision_to_float(const void* x, float* out, size_t n, void* stream);
int cs1_vision_lora_add(void* x, const float* delta, size_t n, float scale, void* stream);

/* ---- additions (no counterpart in the reference) ---- */

/* Causal GQA attention for Dh = 128 or 256 with everything optional: gate (null = no
 * gate), lse [Hq, T] float32 natural-log log-sum-exp of each query row's scaled scores
 * (null = not written), q_base as in cs1_attention_gated_prefix.  With Dh = 256 and a
 * gate it is cs1_attention_gated_prefix bit for bit. */
int cs1_attention_ex(const void* q, const void* k, const void* v, int ldv, const void* gate, void* out, float* lse,
                     int T, int Hq, int Hk, int Dh, float scale, int q_base, void* stream);

/* Varlen form of cs1_attention_ex for packed sequences (replaces the per-sequence launch
 * loop of the reference executor, model.rs:1242-1282): cu_seqlens is a HOST array of
 * nseq + 1 nondecreasing row offsets with cu_seqlens[0] = 0; sequence s is rows
 * [cu_seqlens[s], cu_seqlens[s + 1]) of q, k, v (rows of ldv), gate and out, causal within
 * itself; lse is [Hq, cu_seqlens[nseq]].  Each sequence's result equals a cs1_attention_ex
 * call on its rows bit for bit.  One launch per 64 sequences. */
int cs1_attention_varlen(const void* q, const void* k, const void* v, int ldv, const void* gate, void* out,
                         float* lse, const int32_t* cu_seqlens, int nseq, int Hq, int Hk, int Dh, float scale,
                         void* stream);

/* Varlen form of cs1_gdn_conv for packed sequences that all continue one history (the
 * per-candidate conv of the reference's scoring path, model.rs:1427-1434 and 1421-1470):
 * cu_seqlens is a HOST array of nseq + 1 (at most 64) nondecreasing row offsets with
 * cu_seqlens[0] = 0; sequence s is rows [cu_seqlens[s], cu_seqlens[s + 1]) of qkv (rows of
 * ld) and of q, k, v.  Each sequence's first outputs see the three rows of hist (rows of ld:
 * the three pre-conv rows before position 0; null: zeros) as their history, so each result
 * equals cs1_gdn_conv on [hist | its rows] bit for bit.  Requires 8 | key_dim, value_dim and
 * ld and 16-byte aligned buffers.  One launch. */
int cs1_gdn_conv_varlen(const void* qkv, int ld, const void* w, void* q, void* k, void* v, const int32_t* cu_seqlens,
                        int nseq, const void* hist, int key_dim, int value_dim, void* stream);

/* cs1_attention_varlen for packed sequences that all continue one shared prefix (the
 * candidate scoring of the reference executor, model.rs:1495-1554, which attends each
 * candidate to the cached prefix K/V): pre (a multiple of 64) prefix rows whose post-prep K
 * is kp (rows of Hk * Dh) and V is vp (rows of ldvp).  Sequence s is rows [cu_seqlens[s],
 * cu_seqlens[s + 1]) of q, k, v, gate and out at positions pre, pre + 1, ...: its queries
 * attend to the prefix keys and, causally, its own; lse is [Hq, cu_seqlens[nseq]].  Each
 * sequence's result equals cs1_attention_ex on [prefix K/V | its K/V] with q_base = pre bit
 * for bit.  No K/V copies; one launch per 64 sequences. */
int cs1_attention_prefix_varlen(const void* q, const void* k, const void* v, int ldv, const void* kp, const void* vp,
                                int ldvp, int pre, const void* gate, void* out, float* lse, const int32_t* cu_seqlens,
                                int nseq, int Hq, int Hk, int Dh, float scale, void* stream);

/* No counterpart in the reference: cs1_gdn_prefill_x without the workspace argument, for
 * callers that cannot allocate device memory (code under graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  The workspace is a 64 MiB array inside the library, one
 * per GPU, kept until the process ends; the call itself allocates nothing.  Limit: the
 * workspace of (T, H) must fit, i.e. ceil(T / 64) * H <= 910 (e.g. T <= 1792 at H = 32,
 * T <= 58,240 at H = 1); larger shapes return hipErrorInvalidValue.  Every call on a GPU
 * shares that GPU's array, so calls that overlap in time on one GPU race: serialise them.
 * Results are bit for bit those of cs1_gdn_prefill_x. */
int cs1_gdn_prefill_x_static(const void* q, const void* k, const void* v, const float* g, const void* beta, void* o,
                             int T, int H, int HK, float scale, const void* s_in, void* s_out, void* stream);

/* Varlen form of cs1_gdn_prefill_x for packed sequences (the candidate-packed prefill of the
 * reference's scoring path, model.rs:1421-1470, which runs the delta rule per candidate):
 * cu_seqlens is a HOST array of nseq + 1 (at most 64) nondecreasing row offsets with
 * cu_seqlens[0] = 0; sequence s is rows [cu_seqlens[s], cu_seqlens[s + 1]) of q, k (rows of
 * HK * 128), v and o (rows of H * 128), g and beta (rows of H).  Sequence s starts from the
 * float32 state s_in + s * s_in_stride ([H, 128, 128]; stride 0: one state shared by all,
 * s_in null: zeros) and, when s_out is non-null, leaves its final state at
 * s_out + s * s_out_stride.  Chunks restart at each sequence (each result equals a
 * cs1_gdn_prefill_x call on the sequence's rows bit for bit).  The workspace must hold
 * cs1_gdn_workspace_floats(64 * sum_s ceil(len_s / 64), H) floats.  One launch pair. */
int cs1_gdn_prefill_varlen(const void* q, const void* k, const void* v, const float* g, const void* beta, void* o,
                           float* workspace, const int32_t* cu_seqlens, int nseq, int H, int HK, float scale,
                           const void* s_in, size_t s_in_stride, void* s_out, size_t s_out_stride, void* stream);

/* Gated forms of cs1_gdn_prefill_x and cs1_gdn_prefill_varlen (no reference counterpart:
 * they fold the reference's separate gates launch, cs1_gdn_gates / gdn_gates_kernel at
 * elementwise.cu:42-55 and 115-124, into the GDN prep).  Instead of g and beta they take the
 * raw projections b and a (bf16; token t, head h at b[t * ld + h], a[t * ld + h], ld >= H)
 * and the per-head A_log and dt_bias (bf16 [H]); beta = bf16(sigmoid(b)) and
 * g = -exp(A_log) * softplus(a + dt_bias) are computed in the prep with cs1_gdn_gates'
 * arithmetic, so each result equals cs1_gdn_gates followed by cs1_gdn_prefill_x (or _varlen)
 * bit for bit, without the g / beta buffers or the extra launch.  Everything else (workspace,
 * states, varlen rules, T = 0 pass-through) is that of the ungated form. */
int cs1_gdn_prefill_gated_x(const void* q, const void* k, const void* v, const void* b, const void* a, int ld,
                            const void* A_log, const void* dt_bias, void* o, float* workspace, int T, int H, int HK,
                            float scale, const void* s_in, void* s_out, void* stream);
int cs1_gdn_prefill_gated_varlen(const void* q, const void* k, const void* v, const void* b, const void* a, int ld,
                                 const void* A_log, const void* dt_bias, void* o, float* workspace,
                                 const int32_t* cu_seqlens, int nseq, int H, int HK, float scale, const void* s_in,
                                 size_t s_in_stride, void* s_out, size_t s_out_stride, void* stream);

/* ---- additions: decoding one token at a time (no counterpart in the reference) ----
 *
 * A serving program keeps, for up to nseq sequences, the keys and values of every attention
 * layer in pages and the state of every Gated DeltaNet layer in one slot a sequence.  Each call
 * below works on a list of sequences: seqs is a DEVICE array of sequence numbers (null: row i is
 * sequence i), so a captured graph serves whatever sequences the array names when it is
 * replayed.  A number outside [0, nseq) is a padding row.  Where a call changes a sequence, the
 * first row that names it has it and later rows that name it again are padding rows.  Calls on one
 * table run one after another, on one stream or ordered by events.  All take device pointers of the
 * device that is current, allocate nothing and may be captured. */

/* The page table, on the device; the struct itself is read during the call.  Sequence s holds
 * lens[s] tokens, token j in slot j % page of page table[s * max_pages + j / page]; refs[p] counts
 * the sequences that hold page p (0: free).  A program starts with table filled with -1 and
 * lens and refs with 0.  Limits: nseq <= 8192, npages <= 2^30, page a multiple of 16, max_pages *
 * page < 2^31.  One layer's K pages and V pages are two buffers ("pools") of [npages, page, Hk, Dh], all
 * layers under the one table, on 16 bytes.  Only the calls below change the three arrays.  A page
 * number outside [0, npages) in a row of the table is never followed: its tokens are neither read nor
 * written. */
typedef struct Cs1PageTable {
    int32_t* table; /* [nseq, max_pages] */
    int32_t* lens;  /* [nseq] */
    int32_t* refs;  /* [npages] */
    int nseq, max_pages, npages, page;
} Cs1PageTable;

/* Make room for new tokens: lens[s] grows by one for each of the n listed sequences (cu_seqlens
 * null), or by cu_seqlens[i + 1] - cu_seqlens[i] (a HOST array as in cs1_attention_varlen, n <= 64),
 * and the pages that this needs are the lowest-numbered free ones, in the order of the list.
 * All or nothing: *status (device) receives 0, or the number of pages that are missing, or -1
 * where a sequence would need more than max_pages; if it is not 0 nothing else has changed, and
 * the step that the room was for must not run (it would write over the sequences' last tokens): a
 * program that cannot tell beforehand keeps this call out of the step's graph.  n <= 8192. */
int cs1_kv_reserve(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, int32_t* status,
                   void* stream);

/* Store the last tokens' keys and values of one layer: row r of k (rows of ldk) and of v (rows of
 * ldv), Hk * Dh values each, goes to the pages kp and vp.  cu_seqlens null: row i is the last
 * token (lens[s] - 1) of listed sequence i; else (HOST, cu_seqlens[n] <= 2^23) rows [cu_seqlens[i],
 * cu_seqlens[i + 1]) are its last tokens in order.  Rows of padding or before position 0 are left out.
 * A row goes to its page whether or not forks hold that page too (cs1_kv_fork shares whole pages), and is then
 * theirs as well: after a cs1_kv_reserve that found no room, a token's row would replace the last shared one.
 * Hk * Dh and both row lengths are multiples of 8, k and v on 16 bytes, n <= 8192; Hk * Dh <= 2^24. */
int cs1_kv_write(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, const void* k,
                 int ldk, const void* v, int ldv, void* kp, void* vp, int Hk, int Dh, void* stream);

/* Continue sequences src[i] (device, n <= 8192) as the empty sequences dst[i] (device): dst[i]
 * shares the whole pages and gets a page of its own, the lowest free ones in list order, for what
 * the last page holds if it is not full; those tokens' rows (row_bytes a token) are copied in all
 * npools pools (a HOST array of device pointers to [npages, page * row_bytes bytes]).  Left out are
 * pairs with a number out of range, whose dst holds tokens or an earlier pair names as dst, or whose src
 * is empty or any pair names as dst.  status as in cs1_kv_reserve (0, or the missing pages, and then
 * nothing has changed).  row_bytes: a multiple of 16, up to 2^32; page * row_bytes <= 2^34.  workspace:
 * cs1_kv_workspace_bytes(npages, n) bytes on 16, this call's own until it is done on the device. */
size_t cs1_kv_workspace_bytes(int npages, int n);
int cs1_kv_fork(const Cs1PageTable* pages, const int32_t* src, const int32_t* dst, int n, void* const* pools,
                int npools, size_t row_bytes, void* workspace, int32_t* status, void* stream);

/* End the listed sequences: each page's count falls by one, the rows of the table become -1 and the
 * lengths 0.  n <= 8192. */
int cs1_kv_free(const Cs1PageTable* pages, const int32_t* seqs, int n, void* stream);

/* Move the pages that are held to the start of every pool: with L of them, the i-th held page
 * from L on moves to the i-th free page before L; table and refs follow.  *status receives L.
 * row_bytes as in cs1_kv_fork; (npages / 2 + 1) * (page * row_bytes / 4096 + 1) < 2^25 (256 GiB a
 * pool).  workspace: cs1_kv_workspace_bytes(npages, 0) bytes, as there. */
int cs1_kv_compact(const Cs1PageTable* pages, void* const* pools, int npools, size_t row_bytes, void* workspace,
                   int32_t* status, void* stream);

/* Copy entry src[i] to entry dst[i] (device, n <= 8192) in each of npools buffers of `entries`
 * entries of entry_bytes (a multiple of 16, up to 2^34): pages, or with a sequence's GDN state or conv
 * ring as the entry, what cs1_kv_fork does for the Gated DeltaNet layers (lengths are not looked at
 * here).  Left out are pairs with a number out of range, whose dst an earlier pair names as dst, or
 * whose src any pair names as dst. */
int cs1_kv_copy(void* const* pools, int npools, size_t entry_bytes, int entries, const int32_t* src, const int32_t* dst,
                int n, void* stream);

/* Attention of one new token per row over the pages (after cs1_kv_write); of several of a sequence at once:
 * cs1_attention_paged_varlen.  q, gate (null: none) and
 * out [B, Hq, Dh], Dh 128 or 256; row r's q head h sees the lens[s] keys of sequence s = seqs[r] through kv
 * head h / (Hq / Hk).  lse [Hq, B] float32 (null: not written) as in cs1_attention_ex.  Unlike there the
 * output is rounded once, after the gate.  A padding row, or one of an empty sequence, gets zeros and an
 * lse of -inf.  q, kp, vp, gate and out on 16 bytes; Hk * Dh <= 2^24, B * Hq <= 2^22, npages * page < 2^31 and
 * B * Hk * ceil(Hq / Hk / 16) * (max_pages * page / 32 + 1) < 2^31.  The handle holds the partial
 * results of sequences that are split over the chip (80 MiB): it belongs to the device that is current
 * when it is created (not during a capture; null if that fails) and, as a GEMM handle, serves one
 * thread and one stream at a time (graphs captured with one handle must not run at the same time). */
void* cs1_attention_paged_create(void);
void cs1_attention_paged_destroy(void* paged);
int cs1_attention_paged(void* paged, const void* q, const void* kp, const void* vp, const Cs1PageTable* pages,
                        const int32_t* seqs, const void* gate, void* out, float* lse, int B, int Hq, int Hk, int Dh,
                        float scale, void* stream);

/* One token per row through a Gated DeltaNet layer, from the projections to the normed output: conv1d + SiLU
 * (as cs1_gdn_conv), gates, one step of the delta rule (as cs1_gdn_prefill_gated_x) and, unless z and
 * norm_w are null, the gated RMSNorm.  Row r of qkv, z, b and a (all in rows of ld) is the token at
 * position p = lens[s] - 1 of sequence s = seqs[r]; state is float32 [nseq, H, 128, 128] (K-major, as s_out) and
 * ring bf16 [nseq, 4, (2 HK + H) * 128], the pre-conv row of position i in ring row i % 4; both are
 * updated in place.  At p = 0 the state and at p < 3 the rows before position 0 count as zero, whatever
 * is stored.  All in float32, rounded once in out [B, H, 128].  Padding rows (also lens[s] < 1) get
 * zeros.  lens is a page table's, or any device array of nseq lengths; B <= 8192, B * H <= 2^22, state on 16
 * bytes.  After a prefill of n tokens, ring row i % 4 holds the projection's q | k | v of position i for
 * n - 3 <= i < n: two cs1_copy2d at most. */
int cs1_gdn_decode(const void* qkv, int ld, const void* w, const void* z, const void* b, const void* a,
                   const void* A_log, const void* dt_bias, const void* norm_w, float eps, void* ring, float* state,
                   const int32_t* seqs, const int32_t* lens, int nseq, void* out, int B, int H, int HK, float scale,
                   void* stream);

/* ---- additions: several new tokens of a sequence at once (no counterpart in the reference) ----
 *
 * The second turn of a chat, drafted tokens that are verified, a long prompt in parts, candidates behind a
 * prompt of any length, and any mixture of them with single tokens.  The new tokens of listed
 * sequence i are rows [cu_seqlens[i], cu_seqlens[i + 1]) of a packed batch, and the last tokens that the sequence
 * holds; cu_seqlens is here a DEVICE array of n + 1 offsets that do not fall, from 0 on (n <= 8192), so that one
 * captured graph serves other batches.  `rows` is the number of rows of the batch's buffers: those behind
 * cu_seqlens[n] are no one's.  A step is cs1_kv_extend and cs1_kv_rows once, then per attention layer
 * cs1_attn_prep_paged and cs1_attention_paged_varlen; cs1_token_logprobs reads its logits, and cs1_kv_trim
 * takes tokens back that were not accepted.  A step without room must not run: its rows would be the
 * sequences' last tokens, whose keys and values prep would write over, also in pages that forks share, and cs1_kv_trim would
 * take tokens of earlier steps.  So cs1_kv_extend's status is read before the rest is queued, or the rest goes by it
 * on the device: cs1_kv_rows_if_room in place of cs1_kv_rows, and a drop of 0 for cs1_kv_trim. */

/* cs1_kv_reserve for such a batch: sequence i grows by cu_seqlens[i + 1] - cu_seqlens[i] tokens (a negative number
 * counts as 0).  Pages, status and what follows from it are as there.  max_pages times the lesser of n and nseq < 2^31. */
int cs1_kv_extend(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, int32_t* status,
                  void* stream);

/* Where each row is: pos[r] is its token's position in its sequence and slot[r] its place in the pools, page * pages->page
 * + position % pages->page (int32 [rows] each).  Both are -1 for rows of padding entries (also those of a sequence that
 * an earlier entry names), before position 0 or behind cu_seqlens[n]; slot also where the page's number is out of range.
 * npages * page < 2^31. */
int cs1_kv_rows(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, int rows, int32_t* pos,
                int32_t* slot, void* stream);

/* cs1_kv_rows behind a cs1_kv_extend in one graph: where *status (device, that call's answer) is not 0, all of pos and slot
 * are -1, so that cs1_attn_prep_paged leaves q, gate and the pages as they are.  (What attention then makes of such
 * a step has no meaning.) */
int cs1_kv_rows_if_room(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* cu_seqlens, int n, int rows,
                        const int32_t* status, int32_t* pos, int32_t* slot, void* stream);

/* Take the last drop[i] tokens (device, n <= 8192; less than 0 counts as 0, more than there are as all) off the listed
 * sequences; whole pages behind the new end are released.  A sequence that would end inside a page which others hold
 * too stays as it is (its next token would be written over theirs); *status receives the number of these. */
int cs1_kv_trim(const Cs1PageTable* pages, const int32_t* seqs, const int32_t* drop, int n, int32_t* status,
                void* stream);

/* Rotary positions.  The first `dims` dims of a head (a multiple of 16, 0: none) turn in pairs: (i, i + dims / 2), or
 * with `interleaved` (2i, 2i + 1).  Pair i turns by freqs[i] (DEVICE float64 [dims / 2], on 8 bytes) radians a
 * position, and grows by `magnitude`; angles are formed in float64, so that far positions lose nothing. */
typedef struct Cs1Rotary {
    const double* freqs;
    int dims, interleaved;
    float magnitude;
} Cs1Rotary;

/* freqs (HOST, dims / 2 values; dims even, > 0) for a rotary base, f_i = base^(-2i / dims), and a context `factor` (>= 1)
 * times the `original` one: with r_i = original f_i / (2 pi) turns over it, f_i / factor up to r_i = slow,
 * f_i from r_i = fast on, and in between ((1 - y) / factor + y) f_i with y = (r_i - slow) / (fast - slow) (Peng et al.,
 * "YaRN", arXiv 2309.00071, section 3.2; slow = 1 and fast = 32 there, with magnitude 0.1 ln(factor) + 1).  fast =
 * INFINITY slows all pairs alike (positions divided by the factor).  0 <= slow <= fast.  Needs no device. */
int cs1_rotary_freqs(double* freqs, int dims, double base, double factor, double original, double slow, double fast);

/* Attention inputs of T rows, straight into the pages: row t of qg is Hq heads of Dh (q) or with `gate` of 2 Dh (q | gate),
 * row t of kr and v Hk heads of Dh, all in rows of ld.  q and k are normed (x rsqrt(mean x^2 + eps) (1 + w); qw, kw [Dh],
 * null: not) and turned for position pos[t]; q and gate are written as [T, Hq, Dh], k and v to slot[t] of the pools
 * kp and vp (pos and slot: cs1_kv_rows; of `pages` only npages and page are read).  In float32, each value rounded
 * once.  Rows with pos[t] < 0 are left out, and k and v of rows whose slot is not in [0, npages * page).  Slots differ
 * from row to row.  Dh 128 or 256; ld a multiple of 8, all tensors on 16 bytes; Hk * Dh <= 2^24, T < 2^24. */
int cs1_attn_prep_paged(const void* qg, const void* kr, const void* v, int ld, const void* qw, const void* kw, float eps,
                        const Cs1Rotary* rotary, const Cs1PageTable* pages, const int32_t* pos, const int32_t* slot,
                        void* q, void* gate, void* kp, void* vp, int T, int Hq, int Hk, int Dh, void* stream);

/* Attention of such a batch's rows over the pages, which hold their keys and values already: q, gate (null: none) and
 * out [rows, Hq, Dh]; the row at position p of its sequence sees keys 0 .. p.  max_new is the most rows that an entry has
 * (those behind it are left out).  out and lse [Hq, rows] (float32, null: not written) as in cs1_attention_paged, but
 * for the probabilities, which go to the second product as bfloat16 (entries of up to 16 / (Hq / Hk) rows: as there, if
 * max_new is no more or n > 1).  Rows of padding entries and rows before position
 * 0 get zeros and an lse of -inf; rows behind cu_seqlens[n] are left as they are.  A sequence may be named twice.  Keys of a page
 * whose number is out of range are left out.  scale > 0 (1e-30 to 1e30), Hq / Hk <= 128, rows * Hq <= 2^24,
 * Hk * Dh <= 2^24, npages * page < 2^31; q, kp, vp, gate and out on 16 bytes.  The handle is cs1_attention_paged's, with
 * the same rules. */
int cs1_attention_paged_varlen(void* paged, const void* q, const void* kp, const void* vp, const Cs1PageTable* pages,
                               const int32_t* seqs, const int32_t* cu_seqlens, int n, int max_new, const void* gate,
                               void* out, float* lse, int rows, int Hq, int Hk, int Dh, float scale, void* stream);

/* Log-probabilities of given tokens, entropy and the best alternatives of `rows` rows of V logits (bfloat16, or
 * float32 with is_float; rows of ld, on their own size): logprob[r] = log softmax(row)[targets[r]] (targets and logprob both or
 * neither; 0 where the target is not in [0, V)), entropy[r] = -sum p log p in nats (null: not written), and the k <= 32 largest
 * logits, the lowest index first among equals: top_ids and top_logprobs [rows, k], -1 and NaN behind the last of
 * fewer.  In float32 throughout.  Logits of -inf have no weight; a row with a NaN or +inf, or of -inf only, has NaN for each
 * value and -1 for each index.  V <= 2^28, rows < 2^23.  workspace: cs1_token_logprobs_workspace_bytes(rows, V, k) bytes on 16 (0:
 * null will do), this call's own until it is done on the device.  What it says for rows, V and k is enough for fewer of
 * each as well (under 560 KB), but for 1024 rows and more, which need none: a program whose batches may be
 * smaller than its largest asks for the smaller of that and 1023 rows. */
size_t cs1_token_logprobs_workspace_bytes(int rows, int V, int k);
int cs1_token_logprobs(const void* logits, int is_float, size_t ld, const int32_t* targets, int rows, int V, int k,
                       float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs, void* workspace,
                       void* stream);

#ifdef __cplusplus
}
#endif
