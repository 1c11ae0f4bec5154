/* sheaf_b200 kernel-library entry points (C ABI).
 *
 * Each entry point runs one fused op of Sheaf's compiled fwd+VJP graphs on
 * caller-owned device memory, asynchronously on the caller's CUDA stream
 * (`stream` is a cudaStream_t; NULL = the legacy default stream). They are
 * the building blocks the module executor (sheaf_b200.h) schedules, exported
 * so the primitive-op sweep and the parity tests can drive one kernel at a
 * time. All return 0 on success and a non-zero SB_OPERR_* code otherwise.
 *
 * Element types use the IREE HAL element-type codes that Sheaf's runtime
 * passes today (sheaf/src/runtime/iree_ffi.rs:32-36).
 */
#ifndef SHEAF_B200_OPS_H_
#define SHEAF_B200_OPS_H_

#include <stddef.h>
#include <stdint.h>

#ifndef SB_API
#define SB_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define SB_ELEM_F16 0x21000010u
#define SB_ELEM_F32 0x21000020u
#define SB_ELEM_BF16 0x22000010u
#define SB_ELEM_I32 0x10000020u

#define SB_OPERR_ARGS 1        /* bad shape, null pointer or unsupported dtype */
#define SB_OPERR_TMA 2         /* operand not 16-byte aligned for TMA */
#define SB_OPERR_LAUNCH 4      /* kernel launch failed */
#define SB_OPERR_WORKSPACE 5   /* workspace missing or too small */
#define SB_OPERR_SCRATCH 6     /* size beyond a fixed built-in scratch array */

/* C[M,N] = op(A) @ op(B), fp32 accumulation.
 * Replaces `stablehlo.dot_general` with contracting_dims = [1] x [0]
 * (sheaf/src/lowering/stablehlo/dot_ops.rs:32-79) and, through trans_a /
 * trans_b, the swapaxes operands of the `@` VJP
 * (sheaf/src/autodiff/reverse.rs:585-689).
 *   elem    : SB_ELEM_BF16 (tcgen05 tensor cores) or SB_ELEM_F32 (CUDA cores)
 *   trans_a : 0 -> A stored [M,K] row-major (row stride lda);
 *             1 -> A stored [K,M] (op(A) = A^T)
 *   trans_b : 0 -> B stored [K,N]; 1 -> B stored [N,K] (op(B) = B^T)
 *   c_elem  : SB_ELEM_F32 or SB_ELEM_BF16 output (ldc = row stride)
 *   workspace: fp32 scratch for split-K partials, at least
 *             sb_op_matmul_workspace_size(...) bytes (may be NULL when 0). */
SB_API int sb_op_matmul(uint32_t elem, const void* a, int64_t lda, int trans_a, const void* b, int64_t ldb, int trans_b,
                 int32_t m, int32_t n, int32_t k, void* c, int64_t ldc, uint32_t c_elem, void* workspace,
                 size_t workspace_bytes, void* stream);
SB_API size_t sb_op_matmul_workspace_size(uint32_t elem, int trans_a, int trans_b, int32_t m, int32_t n, int32_t k);
/* The matmul fused with the MLP activation, as the nanoGPT plan runs the fc
 * layer: u = A @ B^T (B stored [N,K]) rounded to the element type, then
 * y = gelu(u) and dy = gelu'(u) in the epilogue (lib/nn.shf:10-11 and its
 * derivative through the tanh, reverse.rs:969-975), both [M,N] with row
 * stride ldc in the element type. No workspace. */
SB_API int sb_op_matmul_gelu(uint32_t elem, const void* a, int64_t lda, const void* b, int64_t ldb, int32_t m,
                             int32_t n, int32_t k, void* y, void* dy, int64_t ldc, void* stream);
/* The matmul with a multiplicative epilogue, as the nanoGPT plan runs the
 * fc2 VJP through the GELU: C = (op(A) @ op(B)) * aux elementwise (the `*`
 * VJP rule fused into the dot_general, reverse.rs:551-583), aux [M,N] with
 * row stride ldaux in the element type; trans_a / trans_b as sb_op_matmul. */
SB_API int sb_op_matmul_mul(uint32_t elem, const void* a, int64_t lda, int trans_a, const void* b, int64_t ldb,
                            int trans_b, int32_t m, int32_t n, int32_t k, const void* aux, int64_t ldaux, void* c,
                            int64_t ldc, void* stream);

/* Layer norm without beta over the last dim (examples/nanogpt/model.shf:11-14:
 * (x - mean) / sqrt(var + 1e-5) * gamma, two-pass population variance as in
 * sheaf/src/lowering/codegen/reduction_builtins.rs:287-358).
 *   x f32 [rows, d]; gamma, y of type `elem` (SB_ELEM_BF16 / SB_ELEM_F32);
 *   mean, rstd f32 [rows] saved for the VJP. d must be a multiple of 4. */
SB_API int sb_op_layernorm_fwd(uint32_t elem, const void* x, const void* gamma, void* y, void* mean, void* rstd,
                               int32_t rows, int32_t d, void* stream);
/* VJP (the `/`, `-`, `sqrt`, `var`, `mean` rules of
 * sheaf/src/autodiff/reverse.rs:551-583,847-914,961-967, composed):
 *   dres (f32 [rows, d]) += dx; dgamma (`elem`, [d]) = sum_rows dy * xhat.
 *   dy is f32. */
SB_API size_t sb_op_layernorm_bwd_workspace_size(int32_t rows, int32_t d);
SB_API int sb_op_layernorm_bwd(uint32_t elem, const void* dy, const void* x, const void* mean, const void* rstd,
                               const void* gamma, void* dres, void* dgamma, void* workspace, size_t workspace_bytes,
                               int32_t rows, int32_t d, void* stream);

/* The same layer-norm VJP for callers that cannot allocate device memory
 * while they run (a host runtime that owns the device heap through its own
 * allocator and passes only finished buffers and a stream, or a
 * latency-critical loop that cannot afford cudaMalloc's device-wide
 * synchronisation). No counterpart in the reference: it exists for such
 * callers of this library. It takes no workspace: the dgamma partial sums go
 * to a fixed 128 KB array compiled into the library (held on every GPU that
 * uses it until the library is unloaded). d must be a multiple of 4 and at
 * most 4096; a larger d returns SB_OPERR_SCRATCH before any GPU work.
 * The first call on a device looks up the array's device address (with that
 * device current); make that first call before any stream capture. All calls
 * share the array, so calls that overlap on the GPU race: serialise them.
 * Allocates nothing (no cudaMalloc / cudaFree). */
SB_API int sb_op_layernorm_bwd_noalloc(uint32_t elem, const void* dy, const void* x, const void* mean,
                                       const void* rstd, const void* gamma, void* dres, void* dgamma, int32_t rows,
                                       int32_t d, void* stream);

/* cross-entropy-loss fused with its VJP (sheaf/lib/nn.shf:28-30,44-50):
 *   loss_f32[0] = -mean_r log_softmax(logits[r])[targets[r]];
 *   dlogits = (softmax(logits) - one_hot(targets)) / rows.
 * logits / dlogits of type `elem` with row strides ld / ldd; targets are f32
 * class ids. As in the reference's one_hot (an f32 compare against an iota,
 * sheaf/src/lowering/stablehlo/tensor_ops.rs:163-217), a target that is not
 * exactly an integer in [0, v) selects no class: its row adds nothing to the
 * loss (which still divides by every row) and its dlogits row is zero. */
SB_API size_t sb_op_cross_entropy_workspace_size(int32_t rows);
SB_API int sb_op_cross_entropy(uint32_t elem, const void* logits, int64_t ld, int32_t rows, int32_t v,
                               const void* targets, void* dlogits, int64_t ldd, void* workspace,
                               size_t workspace_bytes, void* loss_f32, void* stream);

/* GELU, tanh form (sheaf/lib/nn.shf:10-11), elementwise over n values of
 * type `elem`: y = gelu(x). The VJP (chain rule through the inlined tanh /
 * multiply / add ops, sheaf/src/autodiff/reverse.rs:969-975) is
 * dx = g * gelu'(x). Inside the fused plans GELU lives in GEMM epilogues;
 * these standalone forms serve the primitive sweep and other graphs. */
SB_API int sb_op_gelu_fwd(uint32_t elem, const void* x, void* y, int64_t n, void* stream);
SB_API int sb_op_gelu_bwd(uint32_t elem, const void* x, const void* g, void* dx, int64_t n, void* stream);

/* Token + position embedding: x[n] = wte[clamp(ids[n])] + wpe[n % t] (f32 out)
 * (`stablehlo.convert` + `stablehlo.gather`,
 * sheaf/src/lowering/stablehlo/indexing_ops.rs:416-484; wpe `slice`). */
SB_API int sb_op_embedding_fwd(uint32_t elem, const void* ids, const void* wte, const void* wpe, void* x,
                               int32_t ntok, int32_t t, int32_t v, int32_t d, void* stream);
/* Embedding VJP as a scatter-add (the reference's one-hot matmul,
 * sheaf/src/autodiff/reverse.rs:1077-1122) and the wpe slice VJP (pad,
 * sheaf/src/lowering/codegen/builtins.rs:208-271): dx f32 [b*t, d] ->
 * dwte [v, d], dwpe [p, d] (rows >= t zero), both of type `elem`. The
 * one-hot compares the f32 id with an f32 iota, so an id that is not exactly
 * an integer in [0, v) adds nothing (the forward gather instead truncates
 * and clamps it). */
SB_API size_t sb_op_embedding_bwd_workspace_size(int32_t v, int32_t d);
SB_API int sb_op_embedding_bwd(uint32_t elem, const void* ids, const void* dx, int32_t b, int32_t t, int32_t p,
                               int32_t v, int32_t d, void* dwte, void* dwpe, void* workspace, size_t workspace_bytes,
                               void* stream);

/* Fused causal self-attention over the packed projection qkv [b*t, 3*h*hd]
 * (q | k | v, head j at columns j*hd), as examples/nanogpt/model.shf:55-70
 * computes it: softmax(where(tril, q k^T / sqrt(hd), -1e10)) v, heads merged
 * to o [b*t, h*hd]; lse f32 [b*h*t] (log-sum-exp of the scaled scores) is
 * saved for the VJP. hd is 32 or 64. */
SB_API int sb_op_attention_fwd(uint32_t elem, const void* qkv, void* o, void* lse, int32_t b, int32_t t, int32_t h,
                               int32_t hd, void* stream);
/* VJP: dqkv [b*t, 3*h*hd] (dq | dk | dv) from qkv, o, do and lse. */
SB_API size_t sb_op_attention_bwd_workspace_size(uint32_t elem, int32_t b, int32_t t, int32_t h, int32_t hd);
SB_API int sb_op_attention_bwd(uint32_t elem, const void* qkv, const void* o, const void* dout, const void* lse,
                               void* dqkv, void* workspace, size_t workspace_bytes, int32_t b, int32_t t, int32_t h,
                               int32_t hd, void* stream);

/* Optimizer step of nanoGPT's train-step (examples/nanogpt/train.shf:29-32):
 * clip-by-global-norm(g, max_norm) then adamw-step(params, g, m, v, t, lr, b1,
 * b2, eps, wd) as sheaf/lib/optim.shf:19-32,42-51 define them, over n_leaves
 * tensors of element type `elem` (f32 or bf16) at once. The pointer arrays
 * are host arrays of device pointers; counts[i] is leaf i's element count.
 * t and lr are device f32 scalars; t_out receives t + 1. params_out / m_out /
 * v_out may alias params / m / v. max_norm <= 0 disables clipping; norm_out
 * (device f32, optional) receives the global norm of the unclipped gradients.
 * Replaces the optimizer part of the compiled train-step module (IREE
 * dispatches behind iree_runtime_session_call_by_name,
 * sheaf/src/runtime/iree_session.rs:576-583). */
SB_API size_t sb_op_adamw_workspace_size(const int64_t* counts, int32_t n_leaves);
SB_API int sb_op_adamw_step(uint32_t elem, int32_t n_leaves, const int64_t* counts, const void* const* grads,
                            const void* const* params, const void* const* m, const void* const* v,
                            void* const* params_out, void* const* m_out, void* const* v_out, const void* t,
                            void* t_out, const void* lr, float b1, float b2, float eps, float wd, float max_norm,
                            void* norm_out, void* workspace, size_t workspace_bytes, void* stream);
/* Global norm sqrt(sum_i sum(g_i^2)) of n_leaves gradient tensors
 * (sheaf/lib/optim.shf:42-45), f32 accumulation, written to norm_out. */
SB_API int sb_op_global_norm(uint32_t elem, int32_t n_leaves, const int64_t* counts, const void* const* grads,
                             void* norm_out, void* workspace, size_t workspace_bytes, void* stream);

/* get-batch of examples/nanogpt/train.shf:15-21 on the device: x, y
 * [batch, block] f32 token ids, rows starting at random-randint(key, [batch],
 * 0, n - block - 1) (sheaf/src/core/prng.rs:124-134) in `data` (n f32 ids);
 * y is x shifted by one. `key` is four f32 limbs (prng.rs:29-40); all
 * pointers are device memory. Requires 0 < n - block - 1 <= 2^24. */
SB_API int sb_op_get_batch(const void* data, int64_t n, const void* key, int32_t block, int32_t batch, void* x,
                           void* y, void* stream);
/* random-split of `key` into n child keys written as [n, 4] f32 limbs
 * (child i = threefry(key, [i, 1]), prng.rs:81-84, random_ops.rs:146-162). */
SB_API int sb_op_random_split(const void* key, int32_t n, void* out, void* stream);

/* ---- cached generation and scoring -------------------------------------
 * The reference has no cache: its sampler runs the whole window for every
 * token (examples/nanogpt/sample.shf:28-45), and its loss gives the mean over
 * the rows alone (sheaf/lib/nn.shf:44-50). These serve callers that draw
 * several answers to one prompt inside the context and learn from the answers'
 * log probabilities. Index arguments (sequences, positions, page tables,
 * lengths) are int32 device arrays; strides are in elements. A pointer that is
 * not on whole values of its type returns SB_OPERR_ARGS. */

/* One layer's paged key / value cache: row r of head h of page p starts at
 * element p * page_stride + r * row_stride + h * head_stride of `k` and `v`.
 * `k`, `v` and the strides (in bytes) are multiples of 16 bytes; a head's
 * head_dim values are contiguous. */
typedef struct sb_kv_cache {
  void* k;
  void* v;
  int64_t page_stride, row_stride, head_stride;
  int32_t n_pages, page_rows, n_heads, head_dim;
  uint32_t elem; /* SB_ELEM_BF16 or SB_ELEM_F32 */
} sb_kv_cache;

#define SB_ROTARY_NONE 0
#define SB_ROTARY_HALVES 1 /* value i turns with value i + rot_dim / 2 */
#define SB_ROTARY_PAIRS 2  /* value 2 i turns with value 2 i + 1 */

/* Appends n tokens' keys and values. qkv [n, (h_q + 2 * n_heads) * head_dim]
 * (q | k | v, row stride ld) in the cache's element type; token i belongs to
 * sequence seq[i] at position pos[i], whose own page table (row seq[i] of
 * pages [n_seqs, max_pages]) starts at position `base`: it is written to page
 * pages[seq][(pos - base) / page_rows], row (pos - base) % page_rows. The
 * first rot_dim values of each query and key head are rotated by row pos of
 * cos_table / sin_table (f32 [n_pos, rot_dim / 2]); the queries go to q_out
 * [n, h_q * head_dim] (row stride ldq), which may be qkv itself with ldq = ld.
 * seq[i] < 0 marks padding: nothing is appended, its q_out row is zero. A
 * token whose sequence, position or page lies outside its table is treated
 * likewise (a page outside the cache: its q_out row is still computed) and
 * sb_op_device_error reports 2. With h_q = 0, qkv is k | v and q_out NULL.
 * head_dim: 32, 64 or 128. */
SB_API int sb_op_kv_append(const sb_kv_cache* cache, const void* qkv, int64_t ld, int32_t n, int32_t h_q, void* q_out,
                           int64_t ldq, const void* seq, const void* pos, int32_t base, const void* pages,
                           int32_t n_seqs, int32_t max_pages, int32_t rotary, int32_t rot_dim, const void* cos_table,
                           const void* sin_table, int32_t n_pos, void* stream);

/* Attention of b sequences that share their first prefix_len keys: sequence s
 * has those (in pages prefix_pages[0 .. ceil(prefix_len / page_rows))), then
 * lens[s] keys of its own (pages[s], row stride max_pages), the last tq of
 * which belong to its tq query tokens. Query t of sequence s sees the keys up
 * to its own, number prefix_len + lens[s] - tq + t:
 *   out = softmax(scale * q k^T) v,  lse = log sum exp(scale * q k^T)
 * q, out [b * tq, h_q * head_dim] (row strides ldq, ldo; query head h reads
 * key head h / (h_q / n_heads)) in the cache's element type; lse f32
 * [b * tq, h_q], or NULL. A query that sees no key (lens[s] < 0 marks an idle
 * slot) gets a zero row and lse = -inf; so does one all of whose scores are
 * -inf. An infinite value makes its column inf or NaN for the queries that see
 * its key, and for no others. Sums are f32. With a bf16 cache and 17 query rows
 * a key head or more (tq * h_q / n_heads to a sequence's own keys, b times that
 * to the prefix) probabilities may be rounded to bf16 for the product with v
 * (errors of 2.3e-3 of the outputs); with fewer they keep 16 bits (1.7e-3, the
 * outputs' own rounding). prefix_len = 0 is plain attention
 * over a paged cache, max_pages = 0 attention to the prefix alone. lens[s]
 * beyond its table counts as the table's capacity and a page outside the
 * cache as page 0; sb_op_device_error then reports 2. scale > 0. q, out and
 * their row strides are multiples of 16 bytes. head_dim: 32, 64 or 128. */
SB_API size_t sb_op_prefix_attention_workspace_size(const sb_kv_cache* cache, int32_t b, int32_t tq, int32_t h_q,
                                                    int32_t prefix_len, int32_t max_pages);
SB_API int sb_op_prefix_attention(const sb_kv_cache* cache, const void* q, int64_t ldq, void* out, int64_t ldo,
                                  void* lse, int32_t b, int32_t tq, int32_t h_q, float scale, const void* prefix_pages,
                                  int32_t prefix_len, const void* pages, int32_t max_pages, const void* lens,
                                  void* workspace, size_t workspace_bytes, void* stream);

/* Scores rows of logits [rows, v] (row stride ld, any alignment) at a
 * temperature in [1e-6, 1e6], with z = logits / temperature:
 *   logp [rows]    = z[t] - lse for the row's given token t (f32 class id as
 *                    in sb_op_cross_entropy: one that is not exactly an
 *                    integer in [0, v) gives 0)
 *   entropy [rows] = -sum_j p_j log p_j, p = softmax(z)
 *   lse [rows]     = log sum_j exp z_j
 *   top_ids, top_logp [rows, k] = the k likeliest tokens (i32), the larger
 *                    logit first, equal ones by the lower index, and their
 *                    log probabilities; 0 <= k <= min(v, 32)
 * f32 outputs, each NULL when not wanted (targets are needed for logp alone).
 * A logit of -inf has probability 0; a row of nothing else has lse = -inf and
 * entropy 0. A row with a NaN or +inf has NaN statistics, and a NaN orders
 * before every number. */
#define SB_LOGPROBS_MAX_TOP 32
SB_API int sb_op_token_logprobs(uint32_t elem, const void* logits, int64_t ld, int32_t rows, int32_t v,
                                const void* targets, float temperature, void* logp, void* entropy, void* lse,
                                int32_t k, void* top_ids, void* top_logp, void* stream);
/* Its VJP in logp and entropy, from the lse and entropy it gave:
 *   dlogits_j = (dlogp (1[j = t] - p_j) - dentropy p_j (log p_j + entropy)) / temperature
 * dlogits [rows, v] (row stride ldd) in the logits' type; it may be the
 * logits' own memory with ldd = ld. dlogp, dentropy f32 [rows], either NULL
 * for none (targets are needed with dlogp, entropy with dentropy). A row whose
 * lse is -inf has a zero gradient. p_j = exp(z_j - lse), so the rounding of lse
 * to f32, |lse| 2^-24, is an error of log p_j: far from zero (|lse| > 10^5)
 * take the row's maximum off the logits first. */
SB_API int sb_op_token_logprobs_bwd(uint32_t elem, const void* logits, int64_t ld, int32_t rows, int32_t v,
                                    const void* targets, float temperature, const void* lse, const void* entropy,
                                    const void* dlogp, const void* dentropy, void* dlogits, int64_t ldd,
                                    void* stream);

/* Reads and clears the device error word that kernels set (0 = no error,
 * 1 = a barrier wait timed out, 2 = an index outside its table or cache).
 * Synchronizes the device. */
SB_API int sb_op_device_error(void);

#ifdef __cplusplus
}
#endif

#endif /* SHEAF_B200_OPS_H_ */
