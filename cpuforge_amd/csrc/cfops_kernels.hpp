// Internal launch interface of the layer-op kernels (layer_ops.hip) used by
// the C ABI in cfops_capi.cpp.  All pointers are device memory, f32 unless
// stated, row-major and contiguous.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace cfattn {

// RMSNorm (crates/core/src/ops/rmsnorm.rs:4-67).  Forward overwrites y and
// rstd.  Backward adds to (acc) or overwrites dx and, when non-null, dw; it
// needs `partial` scratch of rmsnorm_bwd_partial_floats(rows, dim) floats.
hipError_t launch_rmsnorm_fwd(const float* x, const float* w, float* y, float* rstd, size_t rows, size_t dim, float eps,
                              hipStream_t st);
size_t rmsnorm_bwd_partial_floats(size_t rows, size_t dim);
hipError_t launch_rmsnorm_bwd(const float* dy, const float* x, const float* w, const float* rstd, float* dx, float* dw,
                              float* partial, size_t rows, size_t dim, int acc, hipStream_t st);

// Layer norm (layer_norm.hip); x, y, dy and dx are f32 or bf16, b may be null.  Forward
// overwrites y, mean and rstd.  Backward adds to (acc) or overwrites dx and, where
// non-null, dw and db, with `partial` scratch of layernorm_partial_floats(rows, dim)
// floats for those.  rows and dim are positive, dim below 2^31.
hipError_t launch_layernorm_fwd(bool bf16, const void* x, const float* w, const float* b, void* y, float* mean,
                                float* rstd, size_t rows, size_t dim, float eps, hipStream_t st);
size_t layernorm_partial_floats(size_t rows, size_t dim);
hipError_t launch_layernorm_bwd(bool bf16, const void* dy, const void* x, const float* w, const float* mean,
                                const float* rstd, void* dx, float* dw, float* db, float* partial, size_t rows,
                                size_t dim, int acc, hipStream_t st);

// Rotary positions of up to kRotaryTensors tensors (rotary.hip).  Strides are in values, of
// sequences, tokens and heads; rotary_fits says whether a launch takes the sizes.
constexpr int kRotaryTensors = 4;
struct RotaryTensor {
    const void* x;
    void* y;
    long xs[3], ys[3];
    int heads;  // not 0
    int copy;   // whether the values behind the turned ones are written
    // set by launch_rotary: pieces of a head and of a token, tokens to a workgroup or
    // workgroups to a token and its pieces of each, the first workgroup
    int pieces;
    unsigned per_token, per_token_rcp, pieces_rcp, tokens_wg, parts, part, block0;
};
struct RotaryArgs {
    RotaryTensor t[kRotaryTensors];
    const float *cos, *sin;    // [max_pos][half]
    const int64_t* positions;  // of every token, or null: pos0 + its place in its sequence
    long max_pos, pos0;
    unsigned tokens, seq, token0;  // a launch has tokens [token0, tokens); set by launch_rotary, as
    int turned;                    // pieces of a head that are turned
    int count, head_dim, half, interleaved, inverse;
};
bool rotary_fits(size_t tokens, size_t heads, size_t head_dim);
hipError_t launch_rotary(const RotaryArgs& g, bool x_bf16, bool y_bf16, hipStream_t st);

// SwiGLU gate (crates/core/src/ops/swiglu.rs:10-30): forward overwrites h,
// backward adds to (acc) or overwrites dg and du.
hipError_t launch_silu_mul_fwd(const float* g, const float* u, float* h, size_t n, hipStream_t st);
hipError_t launch_silu_mul_bwd(const float* dh, const float* g, const float* u, float* dg, float* du, size_t n, int acc,
                               hipStream_t st);

// Cross-entropy with its gradient (crates/core/src/ops/loss.rs:9-55), in three
// launches over a `misc` block of kCeMiscBytes (valid-row count, first bad
// row, loss) and `row_loss` scratch of `rows` floats:
//   ce_begin:  count the rows to score, reset the bad-row marker;
//   ce_rows:   rows [row0, row0 + nrows): `logits` and `dlogits` point at
//              row row0 (dlogits may alias logits: each row is read before it
//              is written), targets and row_loss are indexed from row 0; a
//              target outside [0, vocab) marks its row as bad;
//   ce_finish: the mean loss, summed in f64 in row order.
constexpr size_t kCeMiscBytes = 256;
struct CeMisc {
    int n_valid;
    int bad_row;  // first row with a target out of range, or INT_MAX
    float loss;
};
hipError_t launch_ce_begin(const int64_t* targets, size_t rows, void* misc, hipStream_t st);
hipError_t launch_ce_rows(const float* logits, const int64_t* targets, float* dlogits, float* row_loss, size_t row0,
                          size_t nrows, size_t vocab, void* misc, hipStream_t st);
hipError_t launch_ce_finish(const int64_t* targets, const float* row_loss, size_t rows, void* misc, hipStream_t st);

// One AdamW update (crates/train/src/optim.rs:9-30) of `count` tensors, none
// empty; bc1, bc2 are the bias corrections 1 - beta^t, computed by the caller.
constexpr int kAdamwBatch = 64;
struct AdamwTensor {
    float* p;
    const float* g;
    float *m, *v;
    long n;
    float weight_decay;
    int vec;      // set by launch_adamw, as block0
    long block0;
};
struct AdamwArgs {
    AdamwTensor t[kAdamwBatch];
    int count;
    float lr, beta1, beta2, eps, bc1, bc2;
};
hipError_t launch_adamw(AdamwArgs a, hipStream_t st);

// f32 GEMMs over a common row count m (gemm_f32.hip).  Problem i is
//   C_i[m, n_i] (+)= sum over its segments s of A_s B_s,
// the segments being runs of one long contraction (a base product and an
// adapter's, or the products of several linears into one gradient).  A
// element (row, k) is at a[row * lda + k], or a[k * lda + row] with
// a_strided; B element (k, col) at b[col * ldb + k], or b[k * ldb + col] with
// b_strided.  No operand needs more than its natural alignment.
constexpr int kGemmSegs = 8, kGemmProblems = 4;
struct GemmSeg {
    const float *a, *b;
    long lda, ldb;
    int k;
};
struct GemmProblem {
    GemmSeg seg[kGemmSegs];
    int nseg = 0;
    float* c = nullptr;
    int n = 0;
    float scale = 1.0f;  // of the sum (launch_gemm_rows only)
};
struct GemmF32 {
    GemmProblem pr[kGemmProblems];
    int npr = 0, m = 0;
    int acc = 0;  // 1: add to C, 0: overwrite it
    bool a_strided = false, b_strided = false;
};
// `ws` is scratch for the partial sums of a split contraction.
hipError_t launch_gemm_f32(const GemmF32& g, float* ws, size_t ws_floats, hipStream_t st);
// The same products on the f32 MFMA, a workgroup to 16 rows and 16 columns, for
// a_strided = false: an adapter's products with its rank as n, and those of few
// rows, which launch_gemm_f32 passes on.
hipError_t launch_gemm_rows(const GemmF32& g, hipStream_t st);

// The gradients of LoRA adapters in Linear::backward (linear.rs:75-90), for up
// to kGemmProblems linears over the same t tokens in one launch (lora.hip):
//   out (+)= big^T small, [ncol x r] (gb from dy and xs), or its transpose
//   [r x ncol] (ga from x and dxa).
struct LoraGradJob {
    const float *big, *small;
    float* out;
    int ncol, r, transposed;
    long off;  // of its partial sums (set by lora_grad_plan)
};
struct LoraGrad {
    LoraGradJob job[2 * kGemmProblems];
    int njobs = 0, t = 0, acc = 1;
    int chunks, tokens;     // set by lora_grad_plan
    float* part = nullptr;  // scratch of as many floats as lora_grad_plan returns
};
size_t lora_grad_plan(LoraGrad& g);
hipError_t launch_lora_grad(const LoraGrad& g, hipStream_t st);

// AdamW over tensors whose moments are held in 8 bits (state8) or 32 (m, v)
// (adamw8.hip); none empty.  Update reads and writes p and the state; pack and
// unpack convert between m, v and state8.
// A launch takes up to kAdamw8Batch tensors as arguments (28 KiB of them; SmolLM-135M's
// 420 adapters in batches of 60, 240 and 448: 89, 45 and 39 us), or up to
// kAdamw8Few, which are a microsecond less to pass.
constexpr int kAdamw8Batch = 448, kAdamw8Few = 16;
struct Adamw8Tensor {
    float* p;
    const float* g;
    float *m, *v;
    uint8_t* state8;
    long n;
    float weight_decay;
    int vec;      // set by launch_adamw8, as block0
    long block0;
};
struct Adamw8Step {
    int count;
    float lr, beta1, beta2, eps, bc1, bc2;  // 32-bit states, as AdamwArgs
    float c1, c2;                           // 1 / bc1, 1 / sqrt(bc2)
    uint32_t key;                           // adamw8_key(t)
};
enum class Adamw8Op { kUpdate, kPack, kUnpack };
size_t adamw8_state_bytes(size_t n);
uint32_t adamw8_key(uint64_t t);
hipError_t launch_adamw8(Adamw8Tensor* t, const Adamw8Step& step, Adamw8Op op, hipStream_t st);

// Losses over packed sequences (seq_loss.hip); at least one pair or sequence.
struct PreferenceResult {
    int bad_seq;  // first sequence whose offsets do not rise within the rows, or INT_MAX
    float loss, accuracy, margin;
};
struct PreferenceArgs {
    const float *logp, *ref_logp;  // ref_logp may be null
    const int64_t *targets, *offsets;  // targets may be null: every row is scored
    long rows, pairs;
    int form, length_mean;
    double beta, margin, label_smoothing;
    float *dlogp, *rewards;
    PreferenceResult* result;
    // set by launch_preference: each part's sum and scored rows, parts to a sequence
    double2* terms;
    int parts;
};
size_t preference_scratch_bytes(size_t rows, size_t pairs);
hipError_t launch_preference(PreferenceArgs a, void* scratch, hipStream_t st);

struct PolicyResult {
    int n_scored, bad_seq;
    float loss, kl, clipped;
};
struct PolicyArgs {
    const float *logp, *old_logp, *ref_logp, *advantages;  // old_logp, ref_logp may be null
    const int64_t *targets, *offsets;
    long rows, seqs;
    int per_token, sequence_mean;
    double low, high, log_low, log_high, kl_coef;  // the ratio's borders and their logarithms
    float* dlogp;
    PolicyResult* result;
    // set by launch_policy: each part's terms and scored rows, parts to a sequence; with
    // many of them the scored rows and the sequences that have any, else null
    double *terms, *totals;
    int *counts, parts;
};
size_t policy_scratch_bytes(size_t rows, size_t seqs);
hipError_t launch_policy(PolicyArgs a, void* scratch, hipStream_t st);

// Log-probabilities of the targets (head_logp.hip).  Rows whose target is within
// the vocabulary are scored; `idx` and `count` (device memory) name them in
// order, and the kernels below work on scored rows [j0, j0 + nrows), of which
// `logits` holds the logits; those at or past *count are zeros in what they
// write, or not written.  The other arrays are indexed by row.
//   select:    idx and, from idx + rows on, their targets; count[0], tag in count[1]; the
//              result block (CeMisc; or null), and logp
//              and lse (or null) of the rows that are not scored;
//   gather:    the scored rows of hn side by side;   scatter: back, other rows 0;
//   grad_rows: the logits become their gradients;
//   finish:    the mean of sign logp, summed in f64 in a fixed order.
hipError_t launch_logp_select(const int64_t* targets, size_t rows, size_t vocab, int* idx, int* count, int tag,
                              float* logp, float* lse, void* misc, hipStream_t st);
hipError_t launch_logp_gather(const float* hn, const int* idx, const int* count, float* out, size_t rows, size_t d,
                              hipStream_t st);
hipError_t launch_logp_scatter(const float* in, const int* idx, const int* count, float* dhn, size_t rows, size_t d,
                               hipStream_t st);
hipError_t launch_logp_grad_rows(float* logits, const int64_t* targets, const int* idx, const int* count,
                                 const float* lse, const float* dlogp, size_t j0, size_t nrows, size_t vocab,
                                 hipStream_t st);
hipError_t launch_logp_finish(const int64_t* targets, const float* logp, double sign, size_t rows, void* misc,
                              hipStream_t st);
// All of the forward for at most kLogpFew rows in two launches, in scratch of
// logp_few_bytes(t, vocab).
constexpr size_t kLogpFew = 32;
// Up to as many rows a forward keeps nothing, and the gradients are f32 products over
// logits formed again.  Forward and dhn so, and over packed operands with what the forward
// keeps for them, us: 64 rows 576 x 49152 177 and 182, 2048 x 49152 390 and 469, 2048 x
// 128256 913 and 1109, 500 x 50001 179 and 173; 96 rows 225 and 183, 511 and 475, 1191 and
// 1121, 219 and 175.  With the head's gradient 64 rows 232 and 269, 590 and 689, 1488 and
// 1664, 231 and 265.
constexpr size_t kLogpUnkept = 64;
// Which form takes the forward, us of a call by either (rows, d x vocab):
//   few or mid: 16 rows 576 x 49152 37 and 43, 2048 x 128256 267 and 249; 17 rows 46 and
//   44, 319 and 252; where mid's workgroups of 128 rows of the head do not fill half of the
//   card it has the latency of d for itself: 32 rows 2048 x 1000 55 and 90;
//   mid or packed: 256 rows 576 x 49152 77 and 96, 512 rows 133 and 128, 1024 rows 210 and
//   209; 512 rows 2048 x 128256 860 and 1118, 2048 x 32000 250 and 299, 1024 rows 1669 and
//   1818, 443 and 474, 1536 rows (2048 x 49152) 987 and 969; with rows of the head that are
//   read value by value 256 rows 129 x 49152 44 and 45, 384 rows 59 and 52.
inline bool logp_takes_few(size_t t, size_t vocab) { return t <= 16 || (t <= kLogpFew && vocab <= 16384); }
inline bool logp_takes_mid(size_t t, size_t d, const float* head) {
    return t <= (d % 4 || (uintptr_t)head % 16 ? 256 : d < 1024 ? 512 : 1024);
}
size_t logp_few_bytes(size_t t, size_t vocab);
hipError_t launch_logp_few(const float* hn, const float* head, const int64_t* targets, size_t t, size_t d, size_t vocab,
                           float* logp, float* lse, void* misc, void* scratch, hipStream_t st);

// The same for many rows, on packed f16 operands (head_gemm.hip), the logits only
// in registers.  A plan holds the sizes of the buffers, of which rows are in
// chunks: those of stats, xt, keep and factor begin at the chunk's first scored row.
//   pack:      rows, scale, packed and exponents, and with back non-null also that, with
//              rows_back non-null that too; with head null only what is of rows (rows may be null then);
//   stats:     logp and lse (or null) of scored rows [j0, j0 + chunk), j0 a
//              multiple of chunk; with keep non-null (and back packed) also that and
//              factor, from which
//   dhn:       `rows` of dhn, at most a pass, from `local` (a multiple of 128) on, and
//   dhead:     what so many rows add to dhead
//              (acc 0: give as dhead), in scratch of up(rows, 32) v_pad 4 bytes and vocab words;
//   zero_rows: dhn of the rows that are not scored.
// What a forward of other sizes kept (count[1] is not the plan's tag) counts as no
// scored row, and gives NaN gradients.
struct HeadPlan {
    int k16, splits_max, back_mb, tag;  // 16-k steps of a row
    size_t t_pad, v_pad, d_pad, chunk, pass;  // pass: rows of a dhn
    size_t rows_bytes, head_bytes, back_bytes, stats_bytes, keep_bytes, factor_bytes, rows_back_bytes, part_bytes;
};
struct HeadBuffers {
    int *idx, *count, *exponents;        // [2 t], [4], [v_pad / 32]
    char *rows, *packed, *back, *keep, *rows_back;  // operands
    float *scale, *xt, *factor, *part;   // scale [t_pad], xt [chunk]
    void* stats;
    float mul = 1.0f;                    // of hn
};
// In a target's place what distill_kept leaves of a row: dlogits are dloss (a f e_v + dl of the listed
// entry that v is), f the factor of v's part and e_v its kept value, which is an exponential, or of
// an entry that is not listed its gradient over a f, of a listed one 0; dhn is times mul.
struct HeadEntries {
    const int *ids, *count;  // [t][k], and how many are listed
    const float *dl, *a;     // [t][k], [t]
    int k;
};
HeadPlan head_plan(size_t t, size_t d, size_t vocab, size_t chunk_bytes);
hipError_t launch_head_pack(const HeadPlan& p, const HeadBuffers& b, const float* hn, const float* head, size_t d,
                            size_t vocab, hipStream_t st);
hipError_t launch_head_mid(const HeadPlan& p, const HeadBuffers& b, const float* head, size_t t, size_t d, size_t vocab,
                           float* logp, float* lse, hipStream_t st);
hipError_t launch_head_stats(const HeadPlan& p, const HeadBuffers& b, size_t t, size_t j0, size_t vocab,
                             float* logp, float* lse, hipStream_t st);
hipError_t launch_head_dhn(const HeadPlan& p, const HeadBuffers& b, size_t t, const float* head,
                           const float* dlogp, const HeadEntries* entries, size_t j0, size_t local, size_t rows,
                           size_t d, float* dhn, hipStream_t st);
hipError_t launch_head_dhead(const HeadPlan& p, const HeadBuffers& b, size_t t, const float* dlogp,
                             const HeadEntries* entries, size_t j0, size_t local, size_t rows, size_t d, size_t vocab,
                             char* packed_dlogits, unsigned* col_top, float* dhead, int acc, hipStream_t st);
hipError_t launch_head_zero_rows(const HeadPlan& p, const HeadBuffers& b, size_t t, float* dhn, size_t d,
                                 hipStream_t st);

// Distillation from a teacher's top logits (distill.hip).  entries: the rows' entries by
// rising token, what the teacher's distribution is, and a `target` by which launch_logp_select
// takes rows (kept, of which the head's products kept statistics and exponentials) or puts
// them aside (negative: not scored); logits: few rows [j0, j0 + nrows), whose products are in memory.
constexpr size_t kDistillMost = 1024;  // entries of a row
struct TeacherRow {
    double l, p_rest, scale;  // the log-sum-exp that it takes, p_rest (negative: no rest), p / e
};
struct DistillEntries {
    const int64_t* raw_ids;
    const float *teacher, *teacher_lse;  // teacher_lse may be null
    long t, vocab;
    int k;
    double inv_t;
    int *ids, *count;  // [t][k], [t]
    float *z, *e;      // [t][k]: logits, exp((z - the row's largest) inv_t)
    TeacherRow* row;   // [t]
    int64_t* target;   // [t]
    int* tag_at;       // takes the tag (null: none)
    int tag;
};
hipError_t launch_distill_entries(const DistillEntries& g, hipStream_t st);
struct DistillKept {
    int *ids, *count;  // all entries of a row; with dl and a, left as those of HeadEntries
    const float *z, *e;
    const TeacherRow* row;
    int k;
    double inv_t;
    const int *idx, *scored;  // scored rows, how many and the plan's tag
    int tag, j0, chunk, parts, vocab, v16, d;
    long ld;
    const float2* stats;
    char* keep;
    float* factor;
    const float *hn, *head;
    float mul;
    float *loss, *dl, *a;  // loss may be null; dl and a may be, together
};
hipError_t launch_distill_kept(const DistillKept& g, hipStream_t st);
struct DistillRows {
    const int *ids, *count;
    const float *z, *e;
    const TeacherRow* row;
    int k;
    double inv_t;
    const int64_t* target;
    long t, vocab;   // rows from t on: zeros
    int j0;
    float mul;       // of the products
    float* loss;     // may be null
    float2* slices;  // scratch: [rows][distill_slices(vocab)], and
    float* xs;       // [rows][k]
};
size_t distill_slices(size_t vocab);
hipError_t launch_distill_logits(float* logits, size_t nrows, bool grad, const DistillRows& g, hipStream_t st);
// grads [n][vocab] . head into `part` of distill_dhn_floats(n, d, vocab) floats, in parts for up to
// kDistillRowsHead rows, else (by launch_gemm_f32) whole: us of either, with the sum, 24 and 40 rows of
// 49152 x 576 41 and 57, 62 and 56, of 49152 x 2048 112 and 134, 148 and 133.  sum: rows [j0, j0 + n) of
// dhn.  scaled: `padded` rows of hn times mul and dloss.  finish: the result's counts and mean.
struct DistillScored {
    const int64_t* target;  // [t]
    const int* tag_at;      // where the forward left its tag (null: the targets are this call's)
    int tag, t;
};
constexpr size_t kDistillRowsHead = 32;
size_t distill_dhn_floats(size_t n, size_t d, size_t vocab);
hipError_t launch_distill_rows_head(const float* grads, size_t n, size_t d, size_t vocab, const float* head,
                                    float* part, hipStream_t st);
hipError_t launch_distill_rows_sum(const float* part, size_t j0, size_t n, size_t d, size_t vocab, float mul,
                                   const float* dloss, const DistillScored& g, float* dhn, hipStream_t st);
hipError_t launch_distill_scaled(const float* hn, float mul, const float* dloss, const DistillScored& g, size_t padded,
                                 size_t d, float* out, hipStream_t st);
hipError_t launch_distill_finish(const int64_t* target, const float* loss, size_t t, void* misc, hipStream_t st);

}  // namespace cfattn
