/* libcfattn.so -- the layer ops around the attention in a cpuforge training
 * step, on HBM-resident buffers (AMD MI355X, gfx950).
 *
 * Each entry point replaces one reference function of the CPU trainer with
 * the same argument meaning, the same overwrite / accumulate (+=) contract
 * and the same checks, on device pointers and a HIP stream instead of host
 * slices, so a layer's activations stay in HBM between the projections, the
 * norms and the attention (include/cfattn.h).  `stream` NULL is the device's
 * null stream.  A context (cfattn_create) provides the device and the
 * scratch pool.  Its calls are queued one at a time and share the scratch: on
 * different streams they must not overlap, and neither may a graph's replays
 * that such calls were recorded into (their scratch stays allocated until
 * cfattn_destroy).  Status codes and cfattn_last_error() are those of cfattn.h.
 *
 * Reference sources (Sm0r3s-source/cpuforge, crates/...):
 *   core/src/matmul.rs:127-147   matmul_nn / matmul_nt / matmul_tn
 *   core/src/ops/rmsnorm.rs      rmsnorm_forward / rmsnorm_backward
 *   core/src/ops/swiglu.rs       silu_mul_forward / silu_mul_backward
 *   core/src/ops/loss.rs         cross_entropy_fwd_bwd, IGNORE_INDEX
 *   model/src/linear.rs:56-91    Linear::forward / Linear::backward (LoRA)
 *   model/src/model.rs:436-457   LM head + loss in Model::forward_backward
 *   train/src/optim.rs:9-30      adamw_update
 */
#ifndef CFOPS_H
#define CFOPS_H

#include <stddef.h>
#include <stdint.h>

#include "cfattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* crates/core/src/ops/loss.rs:4: targets equal to this are not scored. */
#define CFOPS_IGNORE_INDEX (-100)

/* matmul kinds (core/src/matmul.rs:127-147), row-major, C[m,n] (+)= ...:
 *   CFOPS_NN  A[m,k]  . B[k,n]
 *   CFOPS_NT  A[m,k]  . B[n,k]^T
 *   CFOPS_TN  A[k,m]^T . B[k,n]
 * acc != 0 accumulates into C, acc == 0 overwrites it (k == 0 then zeroes C). */
enum { CFOPS_NN = 0, CFOPS_NT = 1, CFOPS_TN = 2 };
int cfops_matmul(cfattn_ctx* ctx, int kind, const float* a, const float* b, float* c, size_t m, size_t k, size_t n,
                 int acc, void* stream);

/* rmsnorm_forward (rmsnorm.rs:4-28): y = x * rsqrt(mean(x^2) + eps) * w per
 * row of `dim`; y and rstd (1/rms per row) are overwritten.  The sum of
 * squares runs in element order, so y and rstd equal the reference's f32
 * results bit for bit. */
int cfops_rmsnorm_forward(cfattn_ctx* ctx, const float* x, const float* w, float* y, float* rstd, size_t rows,
                          size_t dim, float eps, void* stream);
/* rmsnorm_backward (rmsnorm.rs:33-67): accumulates into dx and, when dw is
 * non-null, into dw (NULL: a frozen gain, no gradient work). */
int cfops_rmsnorm_backward(cfattn_ctx* ctx, const float* dy, const float* x, const float* w, const float* rstd,
                           float* dx, float* dw, size_t rows, size_t dim, void* stream);

/* No reference counterpart: the same with acc == 0 overwriting dx and dw
 * (for callers whose buffers hold nothing yet), acc != 0 adding to them. */
int cfops_rmsnorm_grad(cfattn_ctx* ctx, const float* dy, const float* x, const float* w, const float* rstd, float* dx,
                       float* dw, size_t rows, size_t dim, int acc, void* stream);

/* ---- other decoders' layers ------------------------------------------------
 * No reference counterpart (its layers are RMSNorm and half-layout RoPE). */

/* Layer norm over rows of `dim`: mean = sum x / dim, rstd = 1 / sqrt(sum (x - mean)^2 /
 * dim + eps), y = (x - mean) rstd w + b (b NULL: no bias).  x and y [rows, dim] are
 * of `dtype` (CFATTN_F32 or CFATTN_BF16); w, b [dim], mean and rstd [rows] are f32;
 * y, mean and rstd are overwritten.  Sums and statistics are f32; y is rounded
 * once.  What is not finite in a row stays with that row.  (A buffer that either call
 * writes shares memory with no other.) */
int cfops_layernorm_forward(cfattn_ctx* ctx, int dtype, const void* x, const float* w, const float* b, void* y,
                            float* mean, float* rstd, size_t rows, size_t dim, float eps, void* stream);
/* From dy: dx (of `dtype`, as dy and x) and, where non-null, dw = sum dy (x - mean)
 * rstd and db = sum dy over the rows (f32), each added to what is there (acc
 * == 0: overwritten).  Rows are summed in an order that their number alone decides. */
int cfops_layernorm_backward(cfattn_ctx* ctx, int dtype, const void* dy, const void* x, const float* w,
                             const float* mean, const float* rstd, void* dx, float* dw, float* db, size_t rows,
                             size_t dim, int acc, void* stream);

/* Rotary positions of tensors of heads [batch, seq, heads, head_dim], with any strides
 * (in values; a head's values lie side by side): of a head's first 2 `half` values pair
 * i is turned by the angle of position p, (a, b) -> (a c - b s, b c + a s) with c =
 * cos[p][i] and s = sin[p][i] ([max_pos][half], f32; inverse != 0: s negated, the
 * gradient's way).  The pairs are (i, i + half), as cfattn_prologue_fwd's, or
 * (interleaved != 0) (2 i, 2 i + 1); the values behind them are copied.  A token's
 * position is positions[batch][seq] (int64), or, with positions NULL, pos0 plus its
 * place in its sequence; one outside [0, max_pos) turns the values to NaN.  All x are of
 * x_dtype and all y of y_dtype (rounded once).  A y may be its own x (same pointer,
 * strides and type); it shares no memory with any x otherwise, nor with another y. */
typedef struct cfops_rotary_tensor {
    const void* x;
    void* y;
    size_t heads;
    int64_t x_stride[3]; /* of sequences, tokens and heads */
    int64_t y_stride[3];
} cfops_rotary_tensor;
enum { CFOPS_ROTARY_MAX = 4 };
int cfops_rotary(cfattn_ctx* ctx, const cfops_rotary_tensor* tensors, size_t n, int x_dtype, int y_dtype, size_t batch,
                 size_t seq, size_t head_dim, size_t half, const float* cos, const float* sin, size_t max_pos,
                 const int64_t* positions, size_t pos0, int interleaved, int inverse, void* stream);

/* silu_mul_forward / _backward (swiglu.rs:10-30): h = silu(g) * u
 * (overwritten); the backward accumulates into dg and du. */
int cfops_silu_mul_forward(cfattn_ctx* ctx, const float* g, const float* u, float* h, size_t n, void* stream);
int cfops_silu_mul_backward(cfattn_ctx* ctx, const float* dh, const float* g, const float* u, float* dg, float* du,
                            size_t n, void* stream);

/* The same with acc == 0 overwriting dg and du, acc != 0 adding to them. */
int cfops_silu_mul_grad(cfattn_ctx* ctx, const float* dh, const float* g, const float* u, float* dg, float* du,
                        size_t n, int acc, void* stream);

/* cross_entropy_fwd_bwd (loss.rs:9-55): mean cross-entropy over the rows
 * whose target is not CFOPS_IGNORE_INDEX; dlogits [rows, vocab] is
 * overwritten (ignored rows get zeros; dlogits may equal logits).  Like the
 * reference it returns the loss, so it waits for the stream and writes the
 * loss to host *loss.  A target outside [0, vocab) is CFATTN_ERR_ARG (the
 * reference panics). */
int cfops_cross_entropy_fwd_bwd(cfattn_ctx* ctx, const float* logits, const int64_t* targets, float* dlogits,
                                size_t rows, size_t vocab, float* loss, void* stream);

/* The LM head and its loss, as Model::forward_backward and backward_from run
 * them (model.rs:436-457): logits = hn . head^T, the loss and dlogits of
 * cross_entropy_fwd_bwd, dhn = dlogits . head (overwritten) and, when dhead
 * is non-null, dhead += dlogits^T . hn.  hn [t, d], head [vocab, d].  Rows
 * go through in chunks whose logits fit the context's head chunk limit
 * (cfops_set_head_chunk_limit, default 512 MiB), so the [t, vocab] logits
 * are never held whole.  Waits for the stream; the loss goes to host *loss. */
int cfops_lm_head_ce(cfattn_ctx* ctx, const float* hn, const float* head, const int64_t* targets, size_t t, size_t d,
                     size_t vocab, float* dhn, float* dhead, float* loss, void* stream);
int cfops_set_head_chunk_limit(cfattn_ctx* ctx, size_t bytes);

/* The loss block cfops_lm_head_ce_dev writes, in device memory. */
typedef struct cfops_ce_result {
    int32_t n_valid; /* rows scored (target != CFOPS_IGNORE_INDEX) */
    int32_t bad_row; /* first row whose target is outside [0, vocab), or INT32_MAX */
    float loss;      /* the mean cross-entropy over the scored rows */
} cfops_ce_result;

/* No reference counterpart: cfops_lm_head_ce for callers that capture the
 * training step in a HIP graph or keep host waits out of it.  The same
 * launches on `stream`, with the loss block written to `result` (device
 * memory) and no wait for the stream: once the stream has drained,
 * result->loss is the loss, and result->bad_row != INT32_MAX names a row
 * whose target is out of range, which the caller reports (cfops_lm_head_ce
 * fails with "target T out of range for vocab V" there).  t must be
 * positive; dhn and dhead as in cfops_lm_head_ce. */
int cfops_lm_head_ce_dev(cfattn_ctx* ctx, const float* hn, const float* head, const int64_t* targets, size_t t,
                         size_t d, size_t vocab, float* dhn, float* dhead, cfops_ce_result* result, void* stream);

/* Linear::forward (linear.rs:56-71): y [t,out] = x [t,in] . W^T (overwritten),
 * W [out,in].  With an adapter (lora_a non-null; A [rank,in], B [out,rank]):
 * xs [t,rank] = scale * x . A^T (overwritten) and y += xs . B^T, as more terms
 * of the same sums (rounded once where the reference rounds twice). */
int cfops_linear_forward(cfattn_ctx* ctx, const float* x, const float* w, const float* lora_a, const float* lora_b,
                         float lora_scale, size_t t, size_t in, size_t out, size_t rank, float* y, float* xs,
                         void* stream);
/* Linear::backward (linear.rs:73-91): dx += dy . W; gw += dy^T . x when gw is
 * non-null; with an adapter gb += dy^T . xs (gb non-null), and with
 * dxa = scale * dy . B: ga += dxa^T . x (ga non-null) and dx += dxa . A.
 * NULL gradients are frozen tensors (the reference's empty LinGrad vectors). */
int cfops_linear_backward(cfattn_ctx* ctx, const float* x, const float* xs, const float* dy, const float* w,
                          const float* lora_a, const float* lora_b, float lora_scale, size_t t, size_t in, size_t out,
                          size_t rank, float* dx, float* gw, float* ga, float* gb, void* stream);

/* No reference counterpart: the linears of one input (a layer's q, k and v
 * projections, its gate and up projections; layer.rs:98-102, 133-134) in the
 * launches of one.  Fields of a linear the direction does not name are not
 * read.  Forward: w, out, y and, with an adapter, lora_a, lora_b, lora_scale,
 * rank, xs.  Backward: w, out, dy, gw and, with an adapter, lora_a, lora_b,
 * lora_scale, rank, xs, ga, gb; dx NULL: x needs no gradient.  acc != 0 adds to
 * dx and the gradients, as cfops_linear_backward does linear by linear; acc
 * == 0 overwrites them. */
typedef struct cfops_linear {
    const float* w;
    const float* lora_a;
    const float* lora_b;
    float lora_scale;
    size_t out;
    size_t rank;
    float* y;
    float* xs;
    const float* dy;
    float* gw;
    float* ga;
    float* gb;
} cfops_linear;
int cfops_linears_forward(cfattn_ctx* ctx, const float* x, size_t t, size_t in, const cfops_linear* lin, size_t n,
                          void* stream);
int cfops_linears_backward(cfattn_ctx* ctx, const float* x, size_t t, size_t in, float* dx, const cfops_linear* lin,
                           size_t n, int acc, void* stream);

/* adamw_update (optim.rs:9-30): one AdamW step of one tensor of n values,
 * t the 1-based step count; p, m, v updated in place.  Every product and sum
 * is rounded in the reference's order, so results equal its f32 arithmetic
 * bit for bit. */
int cfops_adamw_update(cfattn_ctx* ctx, float* p, const float* g, float* m, float* v, size_t n, uint64_t t, float lr,
                       float beta1, float beta2, float eps, float weight_decay, void* stream);

/* AdamW::step's loop over the parameters (optim.rs:48-61) in few launches:
 * adamw_update of `count` tensors, tensor i of n[i] values with its own weight
 * decay.  Where tensors share memory the result is that of updating one after
 * the other. */
int cfops_adamw_update_multi(cfattn_ctx* ctx, size_t count, float* const* p, const float* const* g, float* const* m,
                             float* const* v, const size_t* n, const float* weight_decay, uint64_t t, float lr,
                             float beta1, float beta2, float eps, void* stream);

/* ---- preference and policy training ---------------------------------------
 * No reference counterpart (the reference trains on cross-entropy alone):
 * log-probabilities of the targets through the LM head, the losses that start
 * from them, and AdamW with its moments in 8 bits.  Queued on `stream` with no
 * host wait; results are blocks in device memory. */

/* logits = hn . head^T; lse[r] = log sum_v exp(logits[r][v]); logp[r] =
 * logits[r][targets[r]] - lse[r], both 0 where the target is
 * CFOPS_IGNORE_INDEX.  hn [t, d], head [vocab, d]; logp, lse [t] and the block
 * `result` (device memory) are overwritten: result->loss is the mean of -logp
 * over the scored rows, result->bad_row names the first row whose target is
 * outside [0, vocab) (such a row's logp and lse are NaN), as
 * cfops_lm_head_ce_dev's does.  The logits are never held whole.  d and vocab
 * must be positive, t below 2^24 and vocab below 2^26.  What is not finite in a row
 * of hn stays with that row; in the head it is in every row's sum.
 * `keep` (device memory of keep_bytes, 16-byte aligned, or NULL) takes what a
 * backward reads, so that it need not form the logits again: a buffer of
 * cfops_lm_head_logprobs_keep_bytes(t, d, vocab), about 4 t vocab + 4 d vocab
 * bytes; where that is 0 (few rows) it is not used. */
size_t cfops_lm_head_logprobs_keep_bytes(size_t t, size_t d, size_t vocab);
int cfops_lm_head_logprobs(cfattn_ctx* ctx, const float* hn, const float* head, const int64_t* targets, size_t t,
                           size_t d, size_t vocab, float* logp, float* lse, cfops_ce_result* result, void* keep,
                           size_t keep_bytes, void* stream);
/* From the gradient dlogp [t] of logp: dhn [t, d] (overwritten; NULL: not wanted)
 * and, when dhead is non-null, dhead [vocab, d] += dlogits^T . hn (acc == 0: =).
 * hn, head, targets and lse are the forward's, and so is keep (NULL: the logits
 * are formed again, a chunk of rows that fit cfops_set_head_chunk_limit at a
 * time; what a forward of other sizes kept gives NaN gradients).  Rows that are
 * not scored, or have a target out of range, have no gradient, and
 * their hn, lse and dlogp do not matter.  Each row of dhead is exact to f32 of its
 * own size, however small its probabilities (to e^-60) or its row of the head. */
int cfops_lm_head_logprobs_backward(cfattn_ctx* ctx, const float* hn, const float* head, const int64_t* targets,
                                    const float* lse, const float* dlogp, size_t t, size_t d, size_t vocab,
                                    float* dhn, float* dhead, int acc, const void* keep, size_t keep_bytes,
                                    void* stream);

/* Distillation from a teacher's top logits.  Row r of hn has k entries: tokens ids[r]
 * (int64, [t, k], in any order) and the teacher's logits teacher[r] of them; one whose
 * id is CFOPS_IGNORE_INDEX or whose logit is -inf is not there.  With the logits
 * x = hn . head^T / temperature, never held whole, q = softmax(x) and the teacher's
 * p_k = exp(teacher_k / temperature - L):
 *   loss[r] = sum_k p_k (log p_k - log q_k) + p_rest (log p_rest - log q_rest),
 * with L = teacher_lse[r], log sum_v exp(teacher_v / temperature) over its whole
 * vocabulary, and the tokens that are no entry (the rest) as one more class, of
 * probability 1 - sum p; or, with teacher_lse NULL, L the entries' own and p_rest = 0.  (A
 * teacher_lse below the entries' own, -inf among them, counts as that, and where every
 * token is an entry it is not read.)  A row without entries is not
 * scored: loss 0, no gradient.  A bad row has a token outside [0, vocab) or twice, or a
 * teacher's value that is NaN or +inf: its loss is NaN, it has no gradient, and
 * result->bad_row names the first one.
 * result->loss is the mean over the rows with entries.  k is 1 to 1024; d, vocab and t as
 * cfops_lm_head_logprobs's, as is keep, of cfops_lm_head_distill_keep_bytes (few rows:
 * 4 t vocab, the logits' gradients). */
size_t cfops_lm_head_distill_keep_bytes(size_t t, size_t d, size_t vocab, size_t k);
int cfops_lm_head_distill(cfattn_ctx* ctx, const float* hn, const float* head, const int64_t* ids,
                          const float* teacher, const float* teacher_lse, size_t t, size_t d, size_t vocab, size_t k,
                          double temperature, float* loss, cfops_ce_result* result, void* keep, size_t keep_bytes,
                          void* stream);
/* From the gradient dloss [t] of loss: dhn [t, d] (overwritten; NULL: not wanted) and,
 * when dhead is non-null, dhead [vocab, d] += (acc == 0: =), as
 * cfops_lm_head_logprobs_backward; the other arguments are the forward's.  dloss of rows
 * that are not scored, or bad, is not read. */
int cfops_lm_head_distill_backward(cfattn_ctx* ctx, const float* hn, const float* head, const int64_t* ids,
                                   const float* teacher, const float* teacher_lse, const float* dloss, size_t t,
                                   size_t d, size_t vocab, size_t k, double temperature, float* dhn, float* dhead,
                                   int acc, const void* keep, size_t keep_bytes, void* stream);

/* Rows of packed sequences: sequence i is rows [offsets[i], offsets[i + 1]) of
 * logp (int64 in device memory, rising within [0, rows]).  A row whose target
 * is CFOPS_IGNORE_INDEX is not scored (targets NULL: every row is): its inputs
 * are not read, its gradient is 0.  Rows of no sequence keep their dlogp.
 * Where offsets do not rise within [0, rows] they are not followed: the
 * sequence counts as empty, the loss is NaN and the block's bad_seq names the
 * first one (INT32_MAX: none). */
typedef struct cfops_preference_result {
    int32_t bad_seq;
    float loss;     /* the mean over the pairs */
    float accuracy; /* share of pairs whose chosen sequence has the larger reward */
    float margin;   /* mean difference of their rewards */
} cfops_preference_result;
enum { CFOPS_PREFERENCE_SIGMOID = 0, CFOPS_PREFERENCE_HINGE = 1, CFOPS_PREFERENCE_SQUARED = 2 };
/* Sequence 2j is the chosen and 2j + 1 the rejected one of pair j; offsets has
 * 2 * pairs + 1 entries.  A sequence's reward is beta times the sum over its
 * scored rows (length_mean != 0: the mean; 0 with none) of logp - ref_logp
 * (ref_logp NULL: of logp); z = reward(chosen) - reward(rejected) - margin:
 *   SIGMOID  -(1 - s) log sigmoid(z) - s log sigmoid(-z), s = label_smoothing
 *   HINGE    max(0, 1 - z)
 *   SQUARED  (z - 1/2)^2
 * rewards [2 * pairs] and dlogp, the gradient of the mean loss, are
 * overwritten.  label_smoothing is in [0, 1) and 0 for the other forms. */
int cfops_preference_loss(cfattn_ctx* ctx, const float* logp, const float* ref_logp, const int64_t* targets,
                          size_t rows, const int64_t* offsets, size_t pairs, int form, double beta, double margin,
                          double label_smoothing, int length_mean, float* dlogp, float* rewards,
                          cfops_preference_result* result, void* stream);

typedef struct cfops_policy_result {
    int32_t n_scored;
    int32_t bad_seq;
    float loss;
    float kl;      /* the KL estimate under the loss's weights (0 without ref_logp) */
    float clipped; /* share of scored rows whose ratio is cut */
} cfops_policy_result;
enum { CFOPS_POLICY_TOKEN_MEAN = 0, CFOPS_POLICY_SEQUENCE_MEAN = 1 };
/* With r = exp(logp - old_logp) (old_logp NULL: r = 1, for one step on fresh
 * samples) and A the row's advantage, a scored row's loss is
 *   -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef k,
 *   k = exp(x) - x - 1, x = ref_logp - logp (ref_logp NULL: no KL term),
 * weighted 1 / N over all N scored rows (TOKEN_MEAN) or 1 / (M n_i) for the
 * n_i scored rows of one of the M sequences that have any (SEQUENCE_MEAN).
 * advantages: one a row (per_token != 0) or one a sequence.  offsets has seqs +
 * 1 entries.  dlogp is overwritten. */
int cfops_policy_loss(cfattn_ctx* ctx, const float* logp, const float* old_logp, const float* ref_logp,
                      const float* advantages, const int64_t* targets, size_t rows, const int64_t* offsets,
                      size_t seqs, int per_token, double clip_low, double clip_high, double kl_coef, int reduction,
                      float* dlogp, cfops_policy_result* result, void* stream);

/* AdamW over many tensors, each with its moments in 32 bits (m and v, updated as
 * cfops_adamw_update does, bit for bit) or, where state8 is non-null, in 8: a
 * buffer of cfops_adamw8_state_bytes(n) bytes, 16-byte aligned; zeroed, it
 * holds zeros.  It holds blocks of 256 values, each with a power of two of its own
 * for either moment: m as sign, 4 exponent and 3 mantissa bits, v as 5 and 3.
 * A moment is rounded up or down by its fraction of a step against a threshold
 * that is a function of its index and t, so that the mean of its roundings is its
 * value; a positive v is never held as zero; what f32 does not hold is held as
 * NaN (m) and infinity (v).  The update itself is f32, from the new moments
 * before they are rounded.  Tensors that share memory are updated in order. */
typedef struct cfops_adamw_tensor {
    float* p;
    const float* g;
    float* m;       /* update: not read where state8 is non-null */
    float* v;
    uint8_t* state8;
    size_t n;
    float weight_decay;
} cfops_adamw_tensor;
size_t cfops_adamw8_state_bytes(size_t n);
int cfops_adamw8_update_multi(cfattn_ctx* ctx, size_t count, const cfops_adamw_tensor* tensors, uint64_t t, float lr,
                              float beta1, float beta2, float eps, void* stream);
/* f32 moments m and v of the tensors that have a state8 into it, each to the
 * nearest of its steps, and back.  An unpacked state packs to the same values.
 * (p, g and weight_decay are not read.) */
int cfops_adamw8_pack_multi(cfattn_ctx* ctx, size_t count, const cfops_adamw_tensor* tensors, void* stream);
int cfops_adamw8_unpack_multi(cfattn_ctx* ctx, size_t count, const cfops_adamw_tensor* tensors, void* stream);

#ifdef __cplusplus
}
#endif
#endif
