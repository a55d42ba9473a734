// C ABI of the layer ops (declared in include/cfops.h).
//
// Host-side plumbing only: argument checks, scratch from the context's pool
// and dispatch to the gfx950 kernels of gemm_f32.hip, lora.hip, layer_ops.hip,
// head_logp.hip, seq_loss.hip and adamw8.hip.  There is no CPU compute path.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstring>

#include "cfattn_ctx.hpp"
#include "cfops.h"
#include "cfops_kernels.hpp"

namespace {

using namespace cfcapi;

hipStream_t to_stream(void* st) { return static_cast<hipStream_t>(st); }

// Scratch of a GEMM that splits its contraction (partial products).
constexpr size_t kGemmWorkspace = (size_t)32 << 20;

bool fits_int(size_t x) { return x <= (size_t)INT_MAX; }

// A slot's buffer as T*.
template <typename T>
int take(cfattn_ctx* c, int s, size_t bytes, T*& p) {
    int rc = CFATTN_OK;
    p = static_cast<T*>(slot(c, s, bytes, &rc));
    return p ? CFATTN_OK : rc;
}

int launch_gemm(cfattn_ctx* c, const cfattn::GemmF32& g, hipStream_t st) {
    int rc = CFATTN_OK;
    float* ws = static_cast<float*>(slot(c, cfattn_ctx::OPS_WS, kGemmWorkspace, &rc));
    if (!ws) return rc;
    CF_HIP(c, cfattn::launch_gemm_f32(g, ws, kGemmWorkspace / sizeof(float), st), "GEMM launch");
    return CFATTN_OK;
}

// An overwritten gradient of a call without rows: the empty sum.
int zero_grad(cfattn_ctx* c, float* g, size_t n, hipStream_t st) {
    if (g && n) CF_HIP(c, cfattn::launch_fill_zero(g, n, st), "zero-fill launch");
    return CFATTN_OK;
}

// Row-major C[m,n] = op(A) op(B) (+ C when acc), as matmul.rs's
// matmul_nn / matmul_nt / matmul_tn (core/src/matmul.rs:127-147).
int gemm(cfattn_ctx* c, int kind, const float* a, const float* b, float* out, size_t m, size_t k, size_t n, bool acc,
         hipStream_t st) {
    if (m == 0 || n == 0) return CFATTN_OK;
    if (!fits_int(m) || !fits_int(n) || !fits_int(k))
        return fail(c, CFATTN_ERR_UNSUPPORTED, "GEMM dimension above 2^31 (m=%zu, k=%zu, n=%zu)", m, k, n);
    if (k == 0) {  // matmul.rs:58-67: zero C unless accumulating
        if (!acc) CF_HIP(c, cfattn::launch_fill_zero(out, m * n, st), "zero-fill launch");
        return CFATTN_OK;
    }
    if (kind != CFOPS_NN && kind != CFOPS_NT && kind != CFOPS_TN)
        return fail(c, CFATTN_ERR_ARG, "unknown matmul kind %d", kind);
    cfattn::GemmF32 g;
    g.npr = 1, g.m = (int)m, g.acc = acc;
    g.a_strided = kind == CFOPS_TN, g.b_strided = kind != CFOPS_NT;
    g.pr[0].nseg = 1, g.pr[0].c = out, g.pr[0].n = (int)n;
    g.pr[0].seg[0] = {a, b, (long)(kind == CFOPS_TN ? m : k), (long)(kind == CFOPS_NT ? k : n), (int)k};
    return launch_gemm(c, g, st);
}

// Memory that one tensor's update reads or writes.
struct Range {
    uintptr_t lo, hi;
    bool written;
};
Range range(const void* p, size_t bytes, bool written) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return {lo, lo + bytes, written};
}

// Whether one of the ranges that is written shares memory with any other (a
// parameter under two names, or beside a view of itself).  Sorts them.
bool overlaps(Range* r, int n) {
    std::sort(r, r + n, [](const Range& x, const Range& y) { return x.lo < y.lo; });
    uintptr_t end = 0, end_written = 0;
    for (int i = 0; i < n; i++) {
        if (r[i].lo < (r[i].written ? end : end_written)) return true;
        end = std::max(end, r[i].hi);
        if (r[i].written) end_written = std::max(end_written, r[i].hi);
    }
    return false;
}

bool adamw_overlaps(const cfattn::AdamwArgs& a) {
    Range r[4 * cfattn::kAdamwBatch];
    int n = 0;
    for (int i = 0; i < a.count; i++) {
        const cfattn::AdamwTensor& t = a.t[i];
        const float* const ptr[4] = {t.p, t.m, t.v, t.g};
        for (int j = 0; j < 4; j++) r[n++] = range(ptr[j], (size_t)t.n * sizeof(float), j < 3);
    }
    return overlaps(r, n);
}

bool adamw8_overlaps(const cfattn::Adamw8Tensor* ts, int count, cfattn::Adamw8Op op) {
    using cfattn::Adamw8Op;
    Range r[4 * cfattn::kAdamw8Batch];
    int n = 0;
    for (int i = 0; i < count; i++) {
        const cfattn::Adamw8Tensor& t = ts[i];
        const size_t bytes = (size_t)t.n * sizeof(float);
        if (t.state8) r[n++] = range(t.state8, cfattn::adamw8_state_bytes((size_t)t.n), op != Adamw8Op::kUnpack);
        if (op == Adamw8Op::kUpdate) {
            r[n++] = range(t.p, bytes, true);
            r[n++] = range(t.g, bytes, false);
        }
        if (op != Adamw8Op::kUpdate || !t.state8) {
            r[n++] = range(t.m, bytes, op != Adamw8Op::kPack);
            r[n++] = range(t.v, bytes, op != Adamw8Op::kPack);
        }
    }
    return overlaps(r, n);
}

int check_linears(cfattn_ctx* c, size_t t, size_t in, const cfops_linear* lin, size_t n) {
    if (!fits_int(t) || !fits_int(in)) return fail(c, CFATTN_ERR_UNSUPPORTED, "t=%zu, in=%zu above 2^31", t, in);
    for (size_t i = 0; i < n; i++)
        if (!fits_int(lin[i].out) || (lin[i].lora_a && !fits_int(lin[i].rank)))
            return fail(c, CFATTN_ERR_UNSUPPORTED, "out=%zu, rank=%zu above 2^31", lin[i].out, lin[i].rank);
    return CFATTN_OK;
}

// Linear::forward (linear.rs:58-69) of up to kGemmProblems linears of one
// input: xs_i = scale_i x A_i^T in one launch, then y_i = [x xs_i] [W_i B_i]^T in one.
int linears_forward(cfattn_ctx* c, const float* x, size_t t, size_t in, const cfops_linear* lin, size_t n,
                    hipStream_t st) {
    cfattn::GemmF32 g, down;
    down.m = g.m = (int)t;
    for (size_t i = 0; i < n; i++) {
        const cfops_linear& l = lin[i];
        if (l.lora_a) {
            cfattn::GemmProblem& p = down.pr[down.npr++];
            p.seg[p.nseg++] = {x, l.lora_a, (long)in, (long)in, (int)in};
            p.c = l.xs, p.n = (int)l.rank, p.scale = l.lora_scale;
        }
        if (l.out == 0) continue;
        cfattn::GemmProblem& p = g.pr[g.npr++];
        p.c = l.y, p.n = (int)l.out;
        p.seg[p.nseg++] = {x, l.w, (long)in, (long)in, (int)in};
        if (l.lora_a) p.seg[p.nseg++] = {l.xs, l.lora_b, (long)l.rank, (long)l.rank, (int)l.rank};
    }
    CF_HIP(c, cfattn::launch_gemm_rows(down, st), "GEMM launch");
    return g.npr ? launch_gemm(c, g, st) : CFATTN_OK;
}

// Linear::backward (linear.rs:75-90) of up to kGemmProblems linears of one
// input: dxa_i = scale_i dy_i B_i in one launch; dx (+)= [dy_1 dxa_1 dy_2 ..]
// [W_1; A_1; W_2; ..] in one; the adapters' gradients in two.
int linears_backward(cfattn_ctx* c, const float* x, size_t t, size_t in, float* dx, const cfops_linear* lin, size_t n,
                     bool acc_dx, bool acc, hipStream_t st) {
    cfattn::GemmF32 g, down;
    cfattn::LoraGrad lg;
    int rc = CFATTN_OK;
    size_t dxa_floats = 0;
    for (size_t i = 0; i < n; i++) dxa_floats += lin[i].lora_a ? t * lin[i].rank : 0;
    float* dxa = nullptr;
    if (dxa_floats) {
        dxa = static_cast<float*>(slot(c, cfattn_ctx::OPS_DXA, dxa_floats * sizeof(float), &rc));
        if (!dxa) return rc;
    }
    down.m = g.m = lg.t = (int)t;
    down.b_strided = g.b_strided = true, g.acc = acc_dx, lg.acc = acc;
    g.npr = 1, g.pr[0].c = dx, g.pr[0].n = (int)in;
    for (size_t i = 0; i < n; i++) {
        const cfops_linear& l = lin[i];
        cfattn::GemmSeg* seg = g.pr[0].seg;
        seg[g.pr[0].nseg++] = {l.dy, l.w, (long)l.out, (long)in, (int)l.out};
        if (!l.lora_a) continue;
        if (dx || l.ga) {
            cfattn::GemmProblem& p = down.pr[down.npr++];
            p.seg[p.nseg++] = {l.dy, l.lora_b, (long)l.out, (long)l.rank, (int)l.out};
            p.c = dxa, p.n = (int)l.rank, p.scale = l.lora_scale;
            seg[g.pr[0].nseg++] = {dxa, l.lora_a, (long)l.rank, (long)in, (int)l.rank};
        }
        if (l.gb && l.out) lg.job[lg.njobs++] = {l.dy, l.xs, l.gb, (int)l.out, (int)l.rank, 0, 0};
        if (l.ga && in) lg.job[lg.njobs++] = {x, dxa, l.ga, (int)in, (int)l.rank, 1, 0};
        dxa += t * l.rank;
    }
    CF_HIP(c, cfattn::launch_gemm_rows(down, st), "GEMM launch");
    if (dx && in) CF_TRY(launch_gemm(c, g, st));
    for (size_t i = 0; i < n; i++)
        if (lin[i].gw) CF_TRY(gemm(c, CFOPS_TN, lin[i].dy, x, lin[i].gw, lin[i].out, t, in, acc, st));
    if (lg.njobs == 0) return CFATTN_OK;
    lg.part = static_cast<float*>(
        slot(c, cfattn_ctx::OPS_LORA, cfattn::lora_grad_plan(lg) * sizeof(float), &rc));
    if (!lg.part) return rc;
    CF_HIP(c, cfattn::launch_lora_grad(lg, st), "lora launch");
    return CFATTN_OK;
}

// Rust's f32::powi at run time (compiler-rt __powisf2): square-and-multiply
// from the low bit of the exponent, reciprocal for a negative one.
float powi_f32(float a, int b) {
    const bool recip = b < 0;
    unsigned int e = recip ? (unsigned int)(-(long)b) : (unsigned int)b;
    float r = 1.0f;
    for (;;) {
        if (e & 1u) r *= a;
        e >>= 1;
        if (e == 0) break;
        a *= a;
    }
    return recip ? 1.0f / r : r;
}

// Reads the loss block after the stream has drained; reports a target out
// of range as the reference's panic message.
int ce_result(cfattn_ctx* c, const void* misc, const int64_t* targets, size_t vocab, float* loss, hipStream_t st) {
    cfattn::CeMisc m{};
    CF_HIP(c, hipMemcpyAsync(&m, misc, sizeof m, hipMemcpyDeviceToHost, st), "hipMemcpyAsync D2H loss");
    CF_HIP(c, hipStreamSynchronize(st), "cross-entropy");
    if (m.bad_row != INT_MAX) {
        int64_t t = 0;
        CF_HIP(c, hipMemcpy(&t, targets + m.bad_row, sizeof t, hipMemcpyDeviceToHost), "hipMemcpy D2H target");
        return fail(c, CFATTN_ERR_ARG, "target %lld out of range for vocab %zu", (long long)t, vocab);
    }
    *loss = m.loss;
    return CFATTN_OK;
}

#define CF_LOCK(c, stream)                                                                  \
    if (!(c)) return CFATTN_ERR_ARG;                                                      \
    std::lock_guard<std::mutex> lk((c)->mu);                                              \
    (c)->err.clear();                                                                     \
    DeviceGuard dev_guard_((c)->device);                                                  \
    if (!dev_guard_.ok) return fail((c), CFATTN_ERR_HIP, "hipSetDevice(%d) failed", (c)->device); \
    note_capture((c), to_stream(stream))

}  // namespace

extern "C" {

int cfops_matmul(cfattn_ctx* c, int kind, const float* a, const float* b, float* out, size_t m, size_t k, size_t n,
                 int acc, void* stream) {
    CF_LOCK(c, stream);
    if ((m && n && !out) || (m && n && k && (!a || !b))) return fail(c, CFATTN_ERR_ARG, "null buffer");
    return gemm(c, kind, a, b, out, m, k, n, acc != 0, to_stream(stream));
}

int cfops_rmsnorm_forward(cfattn_ctx* c, const float* x, const float* w, float* y, float* rstd, size_t rows,
                          size_t dim, float eps, void* stream) {
    CF_LOCK(c, stream);
    if (rows == 0 || dim == 0) return CFATTN_OK;
    if (!x || !w || !y || !rstd) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (!fits_int(dim)) return fail(c, CFATTN_ERR_UNSUPPORTED, "dim=%zu above 2^31", dim);
    CF_HIP(c, cfattn::launch_rmsnorm_fwd(x, w, y, rstd, rows, dim, eps, to_stream(stream)), "rmsnorm forward launch");
    return CFATTN_OK;
}

int cfops_rmsnorm_backward(cfattn_ctx* c, const float* dy, const float* x, const float* w, const float* rstd,
                           float* dx, float* dw, size_t rows, size_t dim, void* stream) {
    return cfops_rmsnorm_grad(c, dy, x, w, rstd, dx, dw, rows, dim, 1, stream);
}

int cfops_rmsnorm_grad(cfattn_ctx* c, const float* dy, const float* x, const float* w, const float* rstd, float* dx,
                       float* dw, size_t rows, size_t dim, int acc, void* stream) {
    CF_LOCK(c, stream);
    if (rows == 0 && !acc) return zero_grad(c, dw, dim, to_stream(stream));
    if (rows == 0 || dim == 0) return CFATTN_OK;
    if (!dy || !x || !w || !rstd || !dx) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (!fits_int(dim)) return fail(c, CFATTN_ERR_UNSUPPORTED, "dim=%zu above 2^31", dim);
    float* partial = nullptr;
    if (dw) {
        int rc = CFATTN_OK;
        partial = static_cast<float*>(
            slot(c, cfattn_ctx::OPS_PARTIAL, cfattn::rmsnorm_bwd_partial_floats(rows, dim) * sizeof(float), &rc));
        if (!partial) return rc;
    }
    CF_HIP(c, cfattn::launch_rmsnorm_bwd(dy, x, w, rstd, dx, dw, partial, rows, dim, acc != 0, to_stream(stream)),
           "rmsnorm backward launch");
    return CFATTN_OK;
}

int cfops_silu_mul_forward(cfattn_ctx* c, const float* g, const float* u, float* h, size_t n, void* stream) {
    CF_LOCK(c, stream);
    if (n == 0) return CFATTN_OK;
    if (!g || !u || !h) return fail(c, CFATTN_ERR_ARG, "null buffer");
    CF_HIP(c, cfattn::launch_silu_mul_fwd(g, u, h, n, to_stream(stream)), "silu_mul forward launch");
    return CFATTN_OK;
}

int cfops_silu_mul_backward(cfattn_ctx* c, const float* dh, const float* g, const float* u, float* dg, float* du,
                            size_t n, void* stream) {
    return cfops_silu_mul_grad(c, dh, g, u, dg, du, n, 1, stream);
}

int cfops_silu_mul_grad(cfattn_ctx* c, const float* dh, const float* g, const float* u, float* dg, float* du, size_t n,
                        int acc, void* stream) {
    CF_LOCK(c, stream);
    if (n == 0) return CFATTN_OK;
    if (!dh || !g || !u || !dg || !du) return fail(c, CFATTN_ERR_ARG, "null buffer");
    CF_HIP(c, cfattn::launch_silu_mul_bwd(dh, g, u, dg, du, n, acc != 0, to_stream(stream)), "silu_mul backward launch");
    return CFATTN_OK;
}

int cfops_cross_entropy_fwd_bwd(cfattn_ctx* c, const float* logits, const int64_t* targets, float* dlogits,
                                size_t rows, size_t vocab, float* loss, void* stream) {
    CF_LOCK(c, stream);
    if (!loss) return fail(c, CFATTN_ERR_ARG, "null loss");
    *loss = 0.0f;
    if (rows == 0) return CFATTN_OK;
    if (!logits || !targets || !dlogits) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (rows > (size_t)INT_MAX) return fail(c, CFATTN_ERR_UNSUPPORTED, "rows=%zu above 2^31", rows);
    const hipStream_t st = to_stream(stream);
    int rc = CFATTN_OK;
    void* misc = slot(c, cfattn_ctx::OPS_MISC, cfattn::kCeMiscBytes, &rc);
    if (!misc) return rc;
    float* row_loss = static_cast<float*>(slot(c, cfattn_ctx::OPS_ROWLOSS, rows * sizeof(float), &rc));
    if (!row_loss) return rc;
    CF_HIP(c, cfattn::launch_ce_begin(targets, rows, misc, st), "cross-entropy launch");
    CF_HIP(c, cfattn::launch_ce_rows(logits, targets, dlogits, row_loss, 0, rows, vocab, misc, st),
           "cross-entropy launch");
    CF_HIP(c, cfattn::launch_ce_finish(targets, row_loss, rows, misc, st), "cross-entropy launch");
    return ce_result(c, misc, targets, vocab, loss, st);
}

int cfops_set_head_chunk_limit(cfattn_ctx* c, size_t bytes) {
    if (!c) return CFATTN_ERR_ARG;
    std::lock_guard<std::mutex> lk(c->mu);
    c->head_chunk_bytes = bytes;
    return CFATTN_OK;
}

// The LM head and loss queued on `st` with the loss block at `misc` (device
// memory: n_valid, bad_row, loss); the caller holds the context lock and
// has checked the arguments.
static int lm_head_ce_queue(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets, size_t t, size_t d,
                     size_t vocab, float* dhn, float* dhead, void* misc, hipStream_t st) {
    size_t chunk = c->head_chunk_bytes / (vocab * sizeof(float));
    if (chunk < 1) chunk = 1;
    if (chunk > t) chunk = t;
    int rc = CFATTN_OK;
    float* row_loss = static_cast<float*>(slot(c, cfattn_ctx::OPS_ROWLOSS, t * sizeof(float), &rc));
    if (!row_loss) return rc;
    float* logits = static_cast<float*>(slot(c, cfattn_ctx::OPS_LOGITS, chunk * vocab * sizeof(float), &rc));
    if (!logits) return rc;
    CF_HIP(c, cfattn::launch_ce_begin(targets, t, misc, st), "cross-entropy launch");
    for (size_t r0 = 0; r0 < t; r0 += chunk) {
        const size_t nr = t - r0 < chunk ? t - r0 : chunk;
        // logits = hn . head^T (model.rs:438), then dlogits in place.
        CF_TRY(gemm(c, CFOPS_NT, hn + r0 * d, head, logits, nr, d, vocab, false, st));
        CF_HIP(c, cfattn::launch_ce_rows(logits, targets, logits, row_loss, r0, nr, vocab, misc, st),
               "cross-entropy launch");
        // dhn = dlogits . head (model.rs:454, overwritten); dhead += dlogits^T . hn (:457).
        CF_TRY(gemm(c, CFOPS_NN, logits, head, dhn + r0 * d, nr, vocab, d, false, st));
        if (dhead) CF_TRY(gemm(c, CFOPS_TN, logits, hn + r0 * d, dhead, vocab, nr, d, true, st));
    }
    CF_HIP(c, cfattn::launch_ce_finish(targets, row_loss, t, misc, st), "cross-entropy launch");
    return CFATTN_OK;
}

int cfops_lm_head_ce(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets, size_t t, size_t d,
                     size_t vocab, float* dhn, float* dhead, float* loss, void* stream) {
    CF_LOCK(c, stream);
    if (!loss) return fail(c, CFATTN_ERR_ARG, "null loss");
    *loss = 0.0f;
    if (t == 0) return CFATTN_OK;
    if (!hn || !head || !targets || !dhn) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (vocab == 0) return fail(c, CFATTN_ERR_ARG, "vocab must be positive");
    if (t > (size_t)INT_MAX) return fail(c, CFATTN_ERR_UNSUPPORTED, "t=%zu above 2^31", t);
    const hipStream_t st = to_stream(stream);
    int rc = CFATTN_OK;
    void* misc = slot(c, cfattn_ctx::OPS_MISC, cfattn::kCeMiscBytes, &rc);
    if (!misc) return rc;
    CF_TRY(lm_head_ce_queue(c, hn, head, targets, t, d, vocab, dhn, dhead, misc, st));
    return ce_result(c, misc, targets, vocab, loss, st);
}

static_assert(sizeof(cfops_ce_result) == sizeof(cfattn::CeMisc) &&
                  offsetof(cfops_ce_result, bad_row) == offsetof(cfattn::CeMisc, bad_row) &&
                  offsetof(cfops_ce_result, loss) == offsetof(cfattn::CeMisc, loss),
              "cfops_ce_result is the kernels' loss block");

int cfops_lm_head_ce_dev(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets, size_t t,
                         size_t d, size_t vocab, float* dhn, float* dhead, cfops_ce_result* result, void* stream) {
    CF_LOCK(c, stream);
    if (!result) return fail(c, CFATTN_ERR_ARG, "null result");
    if (t == 0) return fail(c, CFATTN_ERR_ARG, "t must be positive");
    if (!hn || !head || !targets || !dhn) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (vocab == 0) return fail(c, CFATTN_ERR_ARG, "vocab must be positive");
    if (t > (size_t)INT_MAX) return fail(c, CFATTN_ERR_UNSUPPORTED, "t=%zu above 2^31", t);
    return lm_head_ce_queue(c, hn, head, targets, t, d, vocab, dhn, dhead, result, to_stream(stream));
}

int cfops_linear_forward(cfattn_ctx* c, const float* x, const float* w, const float* lora_a, const float* lora_b,
                         float lora_scale, size_t t, size_t in, size_t out, size_t rank, float* y, float* xs,
                         void* stream) {
    CF_LOCK(c, stream);
    if (t == 0 || out == 0) return CFATTN_OK;
    if (!x || !w || !y) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (lora_a && (!lora_b || !xs || rank == 0)) return fail(c, CFATTN_ERR_ARG, "adapter needs A, B, xs and rank > 0");
    cfops_linear l{};
    l.w = w, l.lora_a = lora_a, l.lora_b = lora_b, l.lora_scale = lora_scale, l.out = out, l.rank = rank;
    l.y = y, l.xs = xs;
    CF_TRY(check_linears(c, t, in, &l, 1));
    return linears_forward(c, x, t, in, &l, 1, to_stream(stream));
}

int cfops_linear_backward(cfattn_ctx* c, const float* x, const float* xs, const float* dy, const float* w,
                          const float* lora_a, const float* lora_b, float lora_scale, size_t t, size_t in, size_t out,
                          size_t rank, float* dx, float* gw, float* ga, float* gb, void* stream) {
    CF_LOCK(c, stream);
    if (t == 0) return CFATTN_OK;
    if (!x || !dy || !w || !dx) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (lora_a && (!lora_b || !xs || rank == 0)) return fail(c, CFATTN_ERR_ARG, "adapter needs A, B, xs and rank > 0");
    cfops_linear l{};
    l.w = w, l.lora_a = lora_a, l.lora_b = lora_b, l.lora_scale = lora_scale, l.out = out, l.rank = rank;
    l.xs = const_cast<float*>(xs), l.dy = dy, l.gw = gw, l.ga = lora_a ? ga : nullptr, l.gb = lora_a ? gb : nullptr;
    CF_TRY(check_linears(c, t, in, &l, 1));
    return linears_backward(c, x, t, in, dx, &l, 1, true, true, to_stream(stream));
}

int cfops_linears_forward(cfattn_ctx* c, const float* x, size_t t, size_t in, const cfops_linear* lin, size_t n,
                          void* stream) {
    CF_LOCK(c, stream);
    if (t == 0 || n == 0) return CFATTN_OK;
    if (!x || !lin) return fail(c, CFATTN_ERR_ARG, "null buffer");
    for (size_t i = 0; i < n; i++) {
        const cfops_linear& l = lin[i];
        if (l.out && (!l.w || !l.y)) return fail(c, CFATTN_ERR_ARG, "null buffer");
        if (l.lora_a && (!l.lora_b || !l.xs || l.rank == 0))
            return fail(c, CFATTN_ERR_ARG, "adapter needs A, B, xs and rank > 0");
    }
    CF_TRY(check_linears(c, t, in, lin, n));
    for (size_t i = 0; i < n; i += cfattn::kGemmProblems) {
        const size_t m = n - i < (size_t)cfattn::kGemmProblems ? n - i : (size_t)cfattn::kGemmProblems;
        CF_TRY(linears_forward(c, x, t, in, lin + i, m, to_stream(stream)));
    }
    return CFATTN_OK;
}

int cfops_linears_backward(cfattn_ctx* c, const float* x, size_t t, size_t in, float* dx, const cfops_linear* lin,
                           size_t n, int acc, void* stream) {
    CF_LOCK(c, stream);
    if (t == 0 && !acc)
        for (size_t i = 0; lin && i < n; i++) {
            const cfops_linear& l = lin[i];
            CF_TRY(zero_grad(c, l.gw, l.out * in, to_stream(stream)));
            CF_TRY(zero_grad(c, l.ga, l.rank * in, to_stream(stream)));
            CF_TRY(zero_grad(c, l.gb, l.out * l.rank, to_stream(stream)));
        }
    if (n == 0 && !acc) return zero_grad(c, dx, t * in, to_stream(stream));
    if (t == 0 || n == 0) return CFATTN_OK;
    if (!x || !lin) return fail(c, CFATTN_ERR_ARG, "null buffer");
    for (size_t i = 0; i < n; i++) {
        const cfops_linear& l = lin[i];
        if (!l.dy || !l.w) return fail(c, CFATTN_ERR_ARG, "null buffer");
        if (l.lora_a && (!l.lora_b || !l.xs || l.rank == 0))
            return fail(c, CFATTN_ERR_ARG, "adapter needs A, B, xs and rank > 0");
    }
    CF_TRY(check_linears(c, t, in, lin, n));
    for (size_t i = 0; i < n; i += cfattn::kGemmProblems) {
        const size_t m = n - i < (size_t)cfattn::kGemmProblems ? n - i : (size_t)cfattn::kGemmProblems;
        CF_TRY(linears_backward(c, x, t, in, dx, lin + i, m, acc || i > 0, acc != 0, to_stream(stream)));
    }
    return CFATTN_OK;
}

int cfops_adamw_update(cfattn_ctx* c, float* p, const float* g, float* m, float* v, size_t n, uint64_t t, float lr,
                       float beta1, float beta2, float eps, float weight_decay, void* stream) {
    return cfops_adamw_update_multi(c, 1, &p, &g, &m, &v, &n, &weight_decay, t, lr, beta1, beta2, eps, stream);
}

int cfops_adamw_update_multi(cfattn_ctx* c, size_t count, float* const* p, const float* const* g, float* const* m,
                             float* const* v, const size_t* n, const float* weight_decay, uint64_t t, float lr,
                             float beta1, float beta2, float eps, void* stream) {
    CF_LOCK(c, stream);
    if (count && (!p || !g || !m || !v || !n || !weight_decay)) return fail(c, CFATTN_ERR_ARG, "null array");
    for (size_t i = 0; i < count; i++)
        if (n[i] && (!p[i] || !g[i] || !m[i] || !v[i])) return fail(c, CFATTN_ERR_ARG, "null buffer");
    cfattn::AdamwArgs a;
    a.count = 0, a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.eps = eps;
    // optim.rs:21-22: the bias corrections, `t as i32` as in the reference.
    a.bc1 = 1.0f - powi_f32(beta1, (int)(int32_t)t);
    a.bc2 = 1.0f - powi_f32(beta2, (int)(int32_t)t);
    for (size_t i = 0; i < count; i++) {
        if (n[i]) a.t[a.count++] = {p[i], g[i], m[i], v[i], (long)n[i], weight_decay[i], 0, 0};
        if (a.count == cfattn::kAdamwBatch || (i + 1 == count && a.count)) {
            // Tensors of one launch are updated side by side.
            const int step = adamw_overlaps(a) ? 1 : a.count;
            for (int k = 0; k < a.count; k += step) {
                cfattn::AdamwArgs b = a;
                std::copy(a.t + k, a.t + k + step, b.t);
                b.count = step;
                CF_HIP(c, cfattn::launch_adamw(b, to_stream(stream)), "adamw launch");
            }
            a.count = 0;
        }
    }
    return CFATTN_OK;
}

// ---------------------------------------- preference and policy training

namespace {

int check_logprobs(cfattn_ctx* c, size_t t, size_t d, size_t vocab) {
    if (d == 0 || vocab == 0) return fail(c, CFATTN_ERR_ARG, "d and vocab must be positive");
    // (A launch with a workgroup of 256 threads to each row, or 1024 to 32 of the head, has
    // fewer than 2^32.)
    if (t >= (size_t)1 << 24 || !fits_int(d) || vocab >= (size_t)1 << 26)
        return fail(c, CFATTN_ERR_UNSUPPORTED, "t=%zu not below 2^24, d=%zu above 2^31, or vocab=%zu not below 2^26", t,
                    d, vocab);
    return CFATTN_OK;
}

// Scratch of the log-probabilities of few rows: the scored rows, their hidden
// states (in the backward over them their gradients), and the logits of a chunk.
struct LogpRows {
    int *idx, *count;
    float *hn, *logits;
    size_t chunk;
};
int logp_rows(cfattn_ctx* c, size_t t, size_t d, size_t vocab, LogpRows& r) {
    // A chunk's logits fit the head's limit, its rows a launch of workgroups.
    r.chunk = std::min<size_t>(c->head_chunk_bytes / (vocab * sizeof(float)), (size_t)1 << 22);
    r.chunk = std::min(std::max<size_t>(r.chunk, 1), t);
    CF_TRY(take(c, cfattn_ctx::OPS_IDX, (4 + 2 * t) * sizeof(int), r.count));
    r.idx = r.count + 4;
    CF_TRY(take(c, cfattn_ctx::OPS_ROWS, t * d * sizeof(float), r.hn));
    return take(c, cfattn_ctx::OPS_LOGITS, r.chunk * vocab * sizeof(float), r.logits);
}

// Buffers of those of many rows: what a backward reads lies in `keep` where the
// caller holds it, else in scratch.
size_t align_up(size_t x) { return (x + 1023) / 1024 * 1024; }
struct KeepLayout {
    size_t keep, back, factor, bytes;  // offsets; count, idx and exponents come first
};
KeepLayout keep_layout(const cfattn::HeadPlan& p, size_t t) {
    KeepLayout l{};
    l.keep = align_up((4 + 2 * t + p.v_pad / 32) * sizeof(int));
    l.back = l.keep + align_up(p.keep_bytes);
    l.factor = l.back + align_up(p.back_bytes);
    l.bytes = l.factor + align_up(p.factor_bytes);
    return l;
}
void keep_at(const cfattn::HeadPlan& p, size_t t, char* base, cfattn::HeadBuffers& b) {
    const KeepLayout l = keep_layout(p, t);
    b.count = reinterpret_cast<int*>(base);
    b.idx = b.count + 4;
    b.exponents = b.idx + 2 * t;
    b.keep = base + l.keep;
    b.back = base + l.back;
    b.factor = reinterpret_cast<float*>(base + l.factor);
}

// The forward's scratch; with no keep, the small parts of it are scratch too.
int head_scratch(cfattn_ctx* c, const cfattn::HeadPlan& p, size_t t, cfattn::HeadBuffers& b, bool mid = false) {
    char *rows = nullptr, *stats = nullptr;
    CF_TRY(take(c, cfattn_ctx::OPS_ROWS, p.rows_bytes + p.t_pad * sizeof(float), rows));
    b.rows = rows;
    b.scale = reinterpret_cast<float*>(rows + p.rows_bytes);
    CF_TRY(take(c, cfattn_ctx::OPS_STATS, p.stats_bytes + p.chunk * sizeof(float), stats));
    b.stats = stats;
    b.xt = reinterpret_cast<float*>(stats + p.stats_bytes);
    if (!mid) CF_TRY(take(c, cfattn_ctx::OPS_HEAD, p.head_bytes, b.packed));
    if (b.count) return CFATTN_OK;
    CF_TRY(take(c, cfattn_ctx::OPS_IDX, (4 + 2 * t + p.v_pad / 32) * sizeof(int), b.count));
    b.idx = b.count + 4;
    b.exponents = b.idx + 2 * t;
    return CFATTN_OK;
}

int check_keep(cfattn_ctx* c, const void* keep, size_t have, size_t need) {
    if (reinterpret_cast<uintptr_t>(keep) % 16) return fail(c, CFATTN_ERR_ARG, "keep must be 16-byte aligned");
    if (have < need) return fail(c, CFATTN_ERR_ARG, "keep holds %zu bytes, %zu are needed", have, need);
    return CFATTN_OK;
}

int logprobs_many(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets, size_t t, size_t d,
                  size_t vocab, float* logp, float* lse, void* result, void* keep, size_t keep_bytes,
                  hipStream_t st) {
    const cfattn::HeadPlan p = cfattn::head_plan(t, d, vocab, SIZE_MAX);
    cfattn::HeadBuffers b{};
    if (keep) {
        CF_TRY(check_keep(c, keep, keep_bytes, keep_layout(p, t).bytes));
        keep_at(p, t, static_cast<char*>(keep), b);
    }
    const bool mid = !keep && cfattn::logp_takes_mid(t, d, head);
    CF_TRY(head_scratch(c, p, t, b, mid));
    CF_HIP(c, cfattn::launch_logp_select(targets, t, vocab, b.idx, b.count, p.tag, logp, lse, result, st),
           "log-probability launch");
    CF_HIP(c, cfattn::launch_head_pack(p, b, hn, mid ? nullptr : head, d, vocab, st), "log-probability launch");
    if (mid) {
        CF_HIP(c, cfattn::launch_head_mid(p, b, head, t, d, vocab, logp, lse, st), "log-probability launch");
        return CFATTN_OK;
    }
    CF_HIP(c, cfattn::launch_head_stats(p, b, t, 0, vocab, logp, lse, st), "log-probability launch");
    return CFATTN_OK;
}

int logprobs_backward_many(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets,
                           const float* dlogp, size_t t, size_t d, size_t vocab, float* dhn, float* dhead,
                           bool acc, const void* keep, size_t keep_bytes, hipStream_t st) {
    const cfattn::HeadPlan p = cfattn::head_plan(t, d, vocab, keep ? SIZE_MAX : c->head_chunk_bytes);
    cfattn::HeadBuffers b{};
    if (keep) {
        CF_TRY(check_keep(c, keep, keep_bytes, keep_layout(p, t).bytes));
        keep_at(p, t, static_cast<char*>(const_cast<void*>(keep)), b);
    } else {
        CF_TRY(head_scratch(c, p, t, b));
        CF_TRY(take(c, cfattn_ctx::OPS_LOGITS, p.keep_bytes, b.keep));
        CF_TRY(take(c, cfattn_ctx::OPS_BACK, p.back_bytes + p.factor_bytes, b.back));
        b.factor = reinterpret_cast<float*>(b.back + p.back_bytes);
        CF_HIP(c, cfattn::launch_logp_select(targets, t, vocab, b.idx, b.count, p.tag, nullptr, nullptr, nullptr, st),
               "log-probability launch");
    }
    // The head's gradient goes through dlogits that fit the head's limit (and a launch
    // with a row of workgroups to 32 rows).
    const size_t pass = std::min({p.chunk, (size_t)1 << 20,
                                  std::max<size_t>(c->head_chunk_bytes / (p.v_pad * sizeof(float)) / 128 * 128, 128)});
    char* dlogits = nullptr;
    unsigned* col_top = nullptr;
    if (dhead) {
        CF_TRY(take(c, cfattn_ctx::OPS_DLOGITS, pass * p.v_pad * sizeof(float) + vocab * sizeof(unsigned), dlogits));
        col_top = reinterpret_cast<unsigned*>(dlogits + pass * p.v_pad * sizeof(float));
        char* rows = nullptr;
        CF_TRY(take(c, cfattn_ctx::OPS_ROWS_BACK, p.rows_back_bytes + p.t_pad * sizeof(float), rows));
        b.rows_back = rows;
        if (keep) {
            // (A pack of the rows alone; their exponents come out the same.)
            b.scale = reinterpret_cast<float*>(rows + p.rows_back_bytes);
            cfattn::HeadBuffers only = b;
            only.back = nullptr;
            CF_HIP(c, cfattn::launch_head_pack(p, only, hn, nullptr, d, vocab, st), "log-probability launch");
        }
    }
    if (!keep) CF_HIP(c, cfattn::launch_head_pack(p, b, hn, head, d, vocab, st), "log-probability launch");
    if (dhn) {
        CF_TRY(take(c, cfattn_ctx::OPS_PART, p.part_bytes, b.part));
        CF_HIP(c, cfattn::launch_head_zero_rows(p, b, t, dhn, d, st), "log-probability launch");
    }
    for (size_t j0 = 0; j0 < t; j0 += p.chunk) {
        if (!keep)
            CF_HIP(c, cfattn::launch_head_stats(p, b, t, j0, vocab, nullptr, nullptr, st),
                   "log-probability launch");
        for (size_t i = 0; dhn && i < p.chunk && j0 + i < t; i += p.pass)
            CF_HIP(c, cfattn::launch_head_dhn(p, b, t, head, dlogp, j0, i, std::min(p.chunk - i, p.pass), d, dhn, st),
                   "log-probability launch");
        for (size_t i = 0; dhead && i < p.chunk && j0 + i < t; i += pass)
            CF_HIP(c, cfattn::launch_head_dhead(p, b, t, dlogp, j0, i, std::min({t - j0 - i, p.chunk - i, pass}),
                                                d, vocab, dlogits, col_top, dhead, acc || j0 + i, st),
                   "log-probability launch");
    }
    return CFATTN_OK;
}

int check_sequences(cfattn_ctx* c, size_t rows, size_t seqs) {
    // (A launch has fewer than 2^32 threads, a workgroup to each sequence or pair.)
    if (!fits_int(rows) || seqs > (size_t)1 << 22)
        return fail(c, CFATTN_ERR_UNSUPPORTED, "rows=%zu above 2^31 or sequences=%zu above 2^22", rows, seqs);
    return CFATTN_OK;
}

int adamw8_multi(cfattn_ctx* c, size_t count, const cfops_adamw_tensor* tensors, cfattn::Adamw8Op op,
                 cfattn::Adamw8Step step, hipStream_t st) {
    using cfattn::Adamw8Op;
    if (count && !tensors) return fail(c, CFATTN_ERR_ARG, "null array");
    for (size_t i = 0; i < count; i++) {
        const cfops_adamw_tensor& x = tensors[i];
        if (x.n == 0 || (op != Adamw8Op::kUpdate && !x.state8)) continue;
        if ((op == Adamw8Op::kUpdate && (!x.p || !x.g)) ||
            ((op != Adamw8Op::kUpdate || !x.state8) && (!x.m || !x.v)))
            return fail(c, CFATTN_ERR_ARG, "null buffer");
        if (reinterpret_cast<uintptr_t>(x.state8) % 16)
            return fail(c, CFATTN_ERR_ARG, "state8 must be 16-byte aligned");
    }
    cfattn::Adamw8Tensor batch[cfattn::kAdamw8Batch];
    int n = 0;
    for (size_t i = 0; i < count; i++) {
        const cfops_adamw_tensor& x = tensors[i];
        if (x.n && (op == Adamw8Op::kUpdate || x.state8))
            batch[n++] = {x.p, x.g, x.m, x.v, x.state8, (long)x.n, x.weight_decay, 0, 0};
        if (n == cfattn::kAdamw8Batch || (i + 1 == count && n)) {
            // Tensors of one launch are updated side by side.
            step.count = n > 1 && adamw8_overlaps(batch, n, op) ? 1 : n;
            for (int k = 0; k < n; k += step.count)
                CF_HIP(c, cfattn::launch_adamw8(batch + k, step, op, st), "adamw launch");
            n = 0;
        }
    }
    return CFATTN_OK;
}

}  // namespace

size_t cfops_lm_head_logprobs_keep_bytes(size_t t, size_t d, size_t vocab) {
    if (t <= cfattn::kLogpUnkept || t >= (size_t)1 << 24 || d == 0 || vocab == 0 || !fits_int(d) ||
        vocab >= (size_t)1 << 26)
        return 0;
    return keep_layout(cfattn::head_plan(t, d, vocab, SIZE_MAX), t).bytes;
}

int cfops_lm_head_logprobs(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets, size_t t,
                           size_t d, size_t vocab, float* logp, float* lse, cfops_ce_result* result, void* keep,
                           size_t keep_bytes, void* stream) {
    CF_LOCK(c, stream);
    if (!result) return fail(c, CFATTN_ERR_ARG, "null result");
    CF_TRY(check_logprobs(c, t, d, vocab));
    if (!head || (t && (!hn || !targets || !logp || !lse))) return fail(c, CFATTN_ERR_ARG, "null buffer");
    const hipStream_t st = to_stream(stream);
    if (t == 0) {
        CF_HIP(c, cfattn::launch_ce_begin(targets, 0, result, st), "log-probability launch");
        return CFATTN_OK;
    }
    if (cfattn::logp_takes_few(t, vocab)) {
        char* scratch = nullptr;
        CF_TRY(take(c, cfattn_ctx::OPS_STATS, cfattn::logp_few_bytes(t, vocab), scratch));
        CF_HIP(c, cfattn::launch_logp_few(hn, head, targets, t, d, vocab, logp, lse, result, scratch, st),
               "log-probability launch");
        return CFATTN_OK;
    }
    if (t <= cfattn::kLogpUnkept) keep = nullptr;
    CF_TRY(logprobs_many(c, hn, head, targets, t, d, vocab, logp, lse, result, keep, keep_bytes, st));
    CF_HIP(c, cfattn::launch_logp_finish(targets, logp, t, result, st), "log-probability launch");
    return CFATTN_OK;
}

int cfops_lm_head_logprobs_backward(cfattn_ctx* c, const float* hn, const float* head, const int64_t* targets,
                                    const float* lse, const float* dlogp, size_t t, size_t d, size_t vocab,
                                    float* dhn, float* dhead, int acc, const void* keep, size_t keep_bytes,
                                    void* stream) {
    CF_LOCK(c, stream);
    CF_TRY(check_logprobs(c, t, d, vocab));
    if (t == 0 && !acc) return zero_grad(c, dhead, vocab * d, to_stream(stream));
    if (t == 0 || (!dhn && !dhead)) return CFATTN_OK;
    if (!hn || !head || !targets || !lse || !dlogp) return fail(c, CFATTN_ERR_ARG, "null buffer");
    const hipStream_t st = to_stream(stream);
    if (t > cfattn::kLogpUnkept)
        return logprobs_backward_many(c, hn, head, targets, dlogp, t, d, vocab, dhn, dhead, acc != 0, keep, keep_bytes,
                                      st);
    // With zeros in the rows behind the last one the head's gradient sums over whole steps of
    // 32 (us with 2048 x 128256, as they are and so: 24 rows 1586 and 1352, 49 rows 1805 and
    // 1516; 8 rows 1538 and 1504, but 1 row 1253 and 1463).
    const size_t padded = dhead && t > 16 ? (t + 31) / 32 * 32 : t;
    LogpRows rows{};
    CF_TRY(logp_rows(c, padded, d, vocab, rows));
    CF_HIP(c, cfattn::launch_logp_select(targets, t, vocab, rows.idx, rows.count, 0, nullptr, nullptr, nullptr,
                                              st),
           "log-probability launch");
    CF_HIP(c, cfattn::launch_logp_gather(hn, rows.idx, rows.count, rows.hn, padded, d, st), "log-probability launch");
    for (size_t j0 = 0; j0 < padded; j0 += rows.chunk) {
        const size_t nr = std::min(padded - j0, rows.chunk);
        float* h = rows.hn + j0 * d;
        CF_TRY(gemm(c, CFOPS_NT, h, head, rows.logits, nr, d, vocab, false, st));
        CF_HIP(c, cfattn::launch_logp_grad_rows(rows.logits, targets, rows.idx, rows.count, lse, dlogp, j0, nr, vocab,
                                                st),
               "log-probability launch");
        if (dhead) CF_TRY(gemm(c, CFOPS_TN, rows.logits, h, dhead, vocab, nr, d, acc || j0, st));
        if (dhn) CF_TRY(gemm(c, CFOPS_NN, rows.logits, head, h, nr, vocab, d, false, st));
    }
    if (dhn)
        CF_HIP(c, cfattn::launch_logp_scatter(rows.hn, rows.idx, rows.count, dhn, t, d, st), "log-probability launch");
    return CFATTN_OK;
}

static_assert(sizeof(cfops_preference_result) == sizeof(cfattn::PreferenceResult) &&
                  sizeof(cfops_policy_result) == sizeof(cfattn::PolicyResult) &&
                  offsetof(cfops_policy_result, clipped) == offsetof(cfattn::PolicyResult, clipped),
              "the results are the kernels' blocks");

int cfops_preference_loss(cfattn_ctx* c, const float* logp, const float* ref_logp, const int64_t* targets,
                          size_t rows, const int64_t* offsets, size_t pairs, int form, double beta, double margin,
                          double label_smoothing, int length_mean, float* dlogp, float* rewards,
                          cfops_preference_result* result, void* stream) {
    CF_LOCK(c, stream);
    if (pairs == 0) return fail(c, CFATTN_ERR_ARG, "pairs must be positive");
    if (!offsets || !result || (rows && (!logp || !dlogp)) || !rewards) return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (form != CFOPS_PREFERENCE_SIGMOID && form != CFOPS_PREFERENCE_HINGE && form != CFOPS_PREFERENCE_SQUARED)
        return fail(c, CFATTN_ERR_ARG, "unknown preference form %d", form);
    if (!(label_smoothing >= 0.0 && label_smoothing < 1.0) ||
        (form != CFOPS_PREFERENCE_SIGMOID && label_smoothing != 0.0))
        return fail(c, CFATTN_ERR_ARG, "label_smoothing must be in [0, 1), and 0 for the hinge and squared forms");
    CF_TRY(check_sequences(c, rows, pairs));
    int rc = CFATTN_OK;
    void* scratch = slot(c, cfattn_ctx::OPS_SEQ, cfattn::preference_scratch_bytes(rows, pairs), &rc);
    if (!scratch) return rc;
    cfattn::PreferenceArgs a{};
    a.logp = logp, a.ref_logp = ref_logp, a.targets = targets, a.offsets = offsets, a.rows = (long)rows;
    a.pairs = (long)pairs, a.form = form, a.length_mean = length_mean != 0, a.beta = beta, a.margin = margin;
    a.label_smoothing = label_smoothing, a.dlogp = dlogp, a.rewards = rewards;
    a.result = reinterpret_cast<cfattn::PreferenceResult*>(result);
    CF_HIP(c, cfattn::launch_preference(a, scratch, to_stream(stream)), "preference loss launch");
    return CFATTN_OK;
}

int cfops_policy_loss(cfattn_ctx* c, const float* logp, const float* old_logp, const float* ref_logp,
                      const float* advantages, const int64_t* targets, size_t rows, const int64_t* offsets,
                      size_t seqs, int per_token, double clip_low, double clip_high, double kl_coef, int reduction,
                      float* dlogp, cfops_policy_result* result, void* stream) {
    CF_LOCK(c, stream);
    if (seqs == 0) return fail(c, CFATTN_ERR_ARG, "sequences must be positive");
    if (!offsets || !result || (rows && (!logp || !dlogp)) || ((rows || !per_token) && !advantages))
        return fail(c, CFATTN_ERR_ARG, "null buffer");
    if (!(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0))
        return fail(c, CFATTN_ERR_ARG, "clip_low must be in [0, 1] and clip_high not negative");
    if (reduction != CFOPS_POLICY_TOKEN_MEAN && reduction != CFOPS_POLICY_SEQUENCE_MEAN)
        return fail(c, CFATTN_ERR_ARG, "unknown reduction %d", reduction);
    CF_TRY(check_sequences(c, rows, seqs));
    int rc = CFATTN_OK;
    void* scratch = slot(c, cfattn_ctx::OPS_SEQ, cfattn::policy_scratch_bytes(rows, seqs), &rc);
    if (!scratch) return rc;
    cfattn::PolicyArgs a{};
    a.logp = logp, a.old_logp = old_logp, a.ref_logp = ref_logp, a.advantages = advantages, a.targets = targets;
    a.offsets = offsets, a.rows = (long)rows, a.seqs = (long)seqs, a.per_token = per_token != 0;
    a.sequence_mean = reduction == CFOPS_POLICY_SEQUENCE_MEAN, a.low = 1.0 - clip_low, a.high = 1.0 + clip_high;
    a.log_low = std::log1p(-clip_low), a.log_high = std::log1p(clip_high), a.kl_coef = kl_coef, a.dlogp = dlogp;
    a.result = reinterpret_cast<cfattn::PolicyResult*>(result);
    CF_HIP(c, cfattn::launch_policy(a, scratch, to_stream(stream)), "policy loss launch");
    return CFATTN_OK;
}

size_t cfops_adamw8_state_bytes(size_t n) { return cfattn::adamw8_state_bytes(n); }

int cfops_adamw8_update_multi(cfattn_ctx* c, size_t count, const cfops_adamw_tensor* tensors, uint64_t t, float lr,
                              float beta1, float beta2, float eps, void* stream) {
    CF_LOCK(c, stream);
    cfattn::Adamw8Step a{};
    a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.eps = eps;
    a.bc1 = 1.0f - powi_f32(beta1, (int)(int32_t)t);
    a.bc2 = 1.0f - powi_f32(beta2, (int)(int32_t)t);
    a.c1 = (float)(1.0 / (1.0 - std::pow((double)beta1, (double)t)));
    a.c2 = (float)(1.0 / std::sqrt(1.0 - std::pow((double)beta2, (double)t)));
    a.key = cfattn::adamw8_key(t);
    return adamw8_multi(c, count, tensors, cfattn::Adamw8Op::kUpdate, a, to_stream(stream));
}

int cfops_adamw8_pack_multi(cfattn_ctx* c, size_t count, const cfops_adamw_tensor* tensors, void* stream) {
    CF_LOCK(c, stream);
    return adamw8_multi(c, count, tensors, cfattn::Adamw8Op::kPack, {}, to_stream(stream));
}

int cfops_adamw8_unpack_multi(cfattn_ctx* c, size_t count, const cfops_adamw_tensor* tensors, void* stream) {
    CF_LOCK(c, stream);
    return adamw8_multi(c, count, tensors, cfattn::Adamw8Op::kUnpack, {}, to_stream(stream));
}

}  // extern "C"
