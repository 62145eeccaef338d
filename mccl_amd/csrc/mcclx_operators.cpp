// mcclx_operators.cpp -- the C entries of the training operators: argument checks and launches on the
// caller's stream.  Kernels: norm_kernels.hip, loss_kernels.hip.

#include <hip/hip_runtime.h>

#include <cmath>

#include "mcclx.h"
#include "mcclx_internal.h"
#include "operators.h"

namespace {

#define fail mcclx_fail

constexpr uint64_t kMostRows = (1ull << 32) - 1;  // the generator's counter has 32 bits for the row
constexpr uint64_t kMostCols = 1ull << 30;

bool known(int dtype) { return dtype == MCCLX_F32 || dtype == MCCLX_F16 || dtype == MCCLX_BF16; }
uint64_t size_of(int dtype) { return dtype == MCCLX_F32 ? 4 : 2; }

// The context's device is current while it lives.
struct OnDevice {
    int before = -1;
    bool ok = true;
    explicit OnDevice(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        if (before != device) ok = hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// One matrix or vector that a call is given: there, element aligned, its rows apart, and inside its allocation.
struct Checker {
    mcclx_ctx* ctx;
    int rc = MCCLX_OK;
    void rows(const char* what, const void* p, bool wanted, uint64_t size, uint64_t n, uint64_t cols, uint64_t* stride) {
        if (rc || (!p && !wanted)) return;
        if (!p) rc = fail(MCCLX_ERR_INVALID, "%s is null", what);
        else if ((uintptr_t)p % size) rc = fail(MCCLX_ERR_INVALID, "%s=%p is not element aligned", what, p);
        else if (*stride == 0) *stride = cols;
        if (!rc && *stride < cols)
            rc = fail(MCCLX_ERR_INVALID, "%s: rows of %llu elements lie %llu apart", what, (unsigned long long)cols,
                      (unsigned long long)*stride);
        else if (!rc && *stride > (1ull << 40))
            rc = fail(MCCLX_ERR_INVALID, "%s: rows lie %llu elements apart", what, (unsigned long long)*stride);
        // (2^56 elements are past every address; and the next product, in bytes, cannot wrap)
        else if (!rc && n > 1 && n - 1 > (1ull << 56) / (*stride ? *stride : 1))
            rc = fail(MCCLX_ERR_INVALID, "%s: %llu rows that lie %llu elements apart", what, (unsigned long long)n, (unsigned long long)*stride);
        if (!rc && n && mcclx_ctx_validates(ctx)) rc = mcclx_check_range(p, ((n - 1) * *stride + cols) * size, what);
    }
    void flat(const char* what, const void* p, bool wanted, uint64_t size, uint64_t n) {
        uint64_t stride = n;
        rows(what, p, wanted, size, 1, n, &stride);
    }
};

int check_shape(mcclx_ctx* ctx, int dtype, uint64_t rows, uint64_t cols) {
    if (!ctx) return fail(MCCLX_ERR_STATE, "context is null (mcclx_init not called)");
    if (!known(dtype)) return fail(MCCLX_ERR_UNSUPPORTED, "No kernel for dtype code %d", dtype);
    if (rows > kMostRows || cols > kMostCols)
        return fail(MCCLX_ERR_INVALID, "%llu rows of %llu elements: at most 2^32 - 1 of 2^30", (unsigned long long)rows,
                    (unsigned long long)cols);
    return MCCLX_OK;
}

int drop_args(double p, uint64_t seed, uint64_t offset, mcclx::DropArgs* d) {
    if (!(p >= 0.0 && p <= 1.0)) return fail(MCCLX_ERR_INVALID, "p=%g outside 0..1", p);
    d->threshold = p == 0.0 ? 0u : p == 1.0 ? 65536u : (uint32_t)std::nearbyint(p * 65536.0);
    if (p > 0.0 && d->threshold == 0) d->threshold = 1;
    if (p < 1.0 && d->threshold == 65536) d->threshold = 65535;
    d->factor = d->threshold == 65536 ? 0.f : (float)(65536.0 / (65536.0 - d->threshold));
    d->key[0] = (uint32_t)seed;
    d->key[1] = (uint32_t)(seed >> 32);
    d->offset[0] = (uint32_t)offset;
    d->offset[1] = (uint32_t)(offset >> 32);
    return MCCLX_OK;
}

int launched(mcclx_ctx* ctx, int n, hipError_t e) {
    if (n < 0) return fail(MCCLX_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(e));
    mcclx_ctx_launched(ctx, n);
    return MCCLX_OK;
}

int check_norm(mcclx_ctx* ctx, const mcclx_norm* a) {
    if (!ctx) return fail(MCCLX_ERR_STATE, "context is null (mcclx_init not called)");
    if (!a) return fail(MCCLX_ERR_INVALID, "arguments are null");
    if (int rc = check_shape(ctx, a->dtype, a->rows, a->cols)) return rc;
    if (a->param_dtype != a->dtype && a->param_dtype != MCCLX_F32)
        return fail(MCCLX_ERR_UNSUPPORTED, "layer norm: weight and bias of dtype code %d beside matrices of %d", a->param_dtype, a->dtype);
    if (a->cols == 0) return fail(MCCLX_ERR_INVALID, "layer norm of rows without elements");
    return MCCLX_OK;
}

int loss_args(mcclx_ctx* ctx, const mcclx_loss* a, mcclx::LossArgs* k) {
    if (!ctx) return fail(MCCLX_ERR_STATE, "context is null (mcclx_init not called)");
    if (!a) return fail(MCCLX_ERR_INVALID, "arguments are null");
    if (!known(a->dtype)) return fail(MCCLX_ERR_UNSUPPORTED, "No kernel for dtype code %d", a->dtype);
    if (a->reduction != MCCLX_LOSS_NONE && a->reduction != MCCLX_LOSS_MEAN && a->reduction != MCCLX_LOSS_SUM)
        return fail(MCCLX_ERR_INVALID, "reduction=%d unknown", a->reduction);
    if (a->tokens >= 1ull << 24 || a->vocab < 1 || a->vocab > 1ull << 24 || a->width < 1 || a->width > 1ull << 20)
        return fail(MCCLX_ERR_INVALID, "%llu tokens, a vocabulary of %llu, a width of %llu: below 2^24, 1 .. 2^24, 1 .. 2^20",
                    (unsigned long long)a->tokens, (unsigned long long)a->vocab, (unsigned long long)a->width);
    if (a->tokens * a->vocab > 1ull << 39)  // (a grid of all their tiles holds 2^32 lanes at most)
        return fail(MCCLX_ERR_INVALID, "%llu tokens of a vocabulary of %llu: 2^39 logits at most in one call", (unsigned long long)a->tokens,
                    (unsigned long long)a->vocab);
    *k = {};
    k->dtype = a->dtype;
    k->reduction = a->reduction;
    k->tokens = (uint32_t)a->tokens;
    k->vocab = (uint32_t)a->vocab;
    k->width = (uint32_t)a->width;
    k->hidden = a->hidden;
    k->weight = a->weight;
    k->hidden_ld = a->hidden_stride ? a->hidden_stride : a->width;
    k->weight_ld = a->weight_stride ? a->weight_stride : a->width;
    k->target = a->target;
    k->ignore_index = a->ignore_index;
    k->loss = a->loss;
    k->lse = a->lse;
    k->lse_in = a->lse;
    k->grad = a->grad;
    k->dhidden = a->dhidden;
    k->dweight = a->dweight;
    k->workspace = a->workspace;
    return MCCLX_OK;
}

int loss(mcclx_ctx* ctx, void* stream, const mcclx_loss* a, bool backward) {
    mcclx::LossArgs k;
    if (int rc = loss_args(ctx, a, &k)) return rc;
    const uint64_t size = size_of(a->dtype);
    const bool some = a->tokens > 0;
    const uint64_t each = a->reduction == MCCLX_LOSS_NONE ? a->tokens : 1;
    uint64_t out = a->width;
    Checker c{ctx};
    c.rows("hidden", a->hidden, some, size, a->tokens, a->width, &k.hidden_ld);
    c.rows("weight", a->weight, true, size, a->vocab, a->width, &k.weight_ld);
    c.flat("target", a->target, some, 8, a->tokens);
    c.flat("lse", a->lse, some, 4, a->tokens);
    if (backward) {
        c.flat("grad", a->grad, each > 0, 4, each);
        c.rows("dhidden", a->dhidden, false, size, a->tokens, a->width, &out);
        c.rows("dweight", a->dweight, false, size, a->vocab, a->width, &out);
    } else {
        c.flat("loss", a->loss, each > 0, 4, each);
    }
    if (c.rc) return c.rc;
    const int cus = mcclx_device_cus(ctx);
    const uint64_t need = mcclx::loss_workspace_bytes(k, backward, cus);
    c.flat("workspace", a->workspace, need > 0, 1, a->workspace_bytes);
    if (!c.rc && (uintptr_t)a->workspace % 256) c.rc = fail(MCCLX_ERR_INVALID, "workspace=%p is not aligned to 256 bytes", a->workspace);
    if (c.rc) return c.rc;
    if (a->workspace_bytes < need)
        return fail(MCCLX_ERR_INVALID, "workspace of %llu bytes, %llu are needed", (unsigned long long)a->workspace_bytes, (unsigned long long)need);
    OnDevice guard(mcclx_ctx_device(ctx));
    if (!guard.ok) return fail(MCCLX_ERR_HIP, "hipSetDevice(%d) failed", mcclx_ctx_device(ctx));
    hipError_t e = hipSuccess;
    return launched(ctx, mcclx::launch_loss(static_cast<hipStream_t>(stream), k, backward, cus, &e), e);
}

}  // namespace

extern "C" {

int mcclx_layer_norm_forward(mcclx_ctx* ctx, void* stream, const mcclx_norm* a) {
    if (int rc = check_norm(ctx, a)) return rc;
    if (!(a->eps >= 0.0) || !std::isfinite(a->eps)) return fail(MCCLX_ERR_INVALID, "eps=%g", a->eps);
    mcclx::NormForwardArgs k = {};
    if (int rc = drop_args(a->p, a->seed, a->offset, &k.drop)) return rc;
    const uint64_t size = size_of(a->dtype), psize = size_of(a->param_dtype);
    uint64_t xs = a->x_stride, rs = a->residual_stride, out = a->cols;
    const bool some = a->rows > 0;
    Checker c{ctx};
    c.rows("x", a->x, some, size, a->rows, a->cols, &xs);
    c.rows("residual", a->residual, false, size, a->rows, a->cols, &rs);
    c.rows("y", a->y, some, size, a->rows, a->cols, &out);
    c.rows("s", a->s, false, size, a->rows, a->cols, &out);
    c.flat("weight", a->weight, false, psize, a->cols);
    c.flat("bias", a->bias, false, psize, a->cols);
    c.flat("mean", a->mean, some, 4, a->rows);
    c.flat("rstd", a->rstd, some, 4, a->rows);
    if (c.rc || !some) return c.rc;
    k.x = a->x;
    k.residual = a->residual;
    k.weight = a->weight;
    k.bias = a->bias;
    k.y = a->y;
    k.s = a->s;
    k.mean = a->mean;
    k.rstd = a->rstd;
    k.x_stride = xs;
    k.residual_stride = rs;
    k.rows = a->rows;
    k.cols = (uint32_t)a->cols;
    k.eps = (float)a->eps;
    OnDevice guard(mcclx_ctx_device(ctx));
    if (!guard.ok) return fail(MCCLX_ERR_HIP, "hipSetDevice(%d) failed", mcclx_ctx_device(ctx));
    hipError_t e = hipSuccess;
    return launched(ctx, mcclx::launch_norm_forward(static_cast<hipStream_t>(stream), a->dtype, a->param_dtype, k, &e), e);
}

uint64_t mcclx_layer_norm_workspace_bytes(mcclx_ctx* ctx, uint64_t rows, uint64_t cols) {
    if (!ctx || rows > kMostRows || cols > kMostCols) return 0;
    return mcclx::norm_backward_scratch(rows, (uint32_t)cols, mcclx_device_cus(ctx));
}

int mcclx_layer_norm_backward(mcclx_ctx* ctx, void* stream, const mcclx_norm* a) {
    if (int rc = check_norm(ctx, a)) return rc;
    mcclx::NormBackwardArgs k = {};
    if (int rc = drop_args(a->p, a->seed, a->offset, &k.drop)) return rc;
    const uint64_t size = size_of(a->dtype), psize = size_of(a->param_dtype);
    uint64_t ss = a->s_stride, dys = a->dy_stride, dss = a->ds_stride, out = a->cols;
    const bool some = a->rows > 0;
    Checker c{ctx};
    c.rows("dy", a->dy, some, size, a->rows, a->cols, &dys);
    c.rows("s", a->s, some, size, a->rows, a->cols, &ss);
    c.rows("ds", a->ds, false, size, a->rows, a->cols, &dss);
    c.rows("dx", a->dx, false, size, a->rows, a->cols, &out);
    c.rows("dresidual", a->dresidual, false, size, a->rows, a->cols, &out);
    c.flat("weight", a->weight, false, psize, a->cols);
    c.flat("dweight", a->dweight, false, psize, a->cols);
    c.flat("dbias", a->dbias, false, psize, a->cols);
    c.flat("mean", a->mean, some, 4, a->rows);
    c.flat("rstd", a->rstd, some, 4, a->rows);
    if (c.rc) return c.rc;
    const int cus = mcclx_device_cus(ctx);
    k.parts = mcclx::norm_backward_parts(a->rows, (uint32_t)a->cols, cus);
    const uint64_t need = some ? mcclx::norm_backward_scratch(a->rows, (uint32_t)a->cols, cus) : 0;
    if (need) {
        if (a->workspace_bytes < need)
            return fail(MCCLX_ERR_INVALID, "workspace of %llu bytes, %llu are needed", (unsigned long long)a->workspace_bytes,
                        (unsigned long long)need);
        c.flat("workspace", a->workspace, true, 16, 1);  // (its alignment)
        c.flat("workspace", a->workspace, true, 1, need);
        if (c.rc) return c.rc;
    }
    k.dy = a->dy;
    k.ds = a->ds;
    k.x = a->s;
    k.weight = a->weight;
    k.mean = a->mean;
    k.rstd = a->rstd;
    k.dx = a->dx;
    k.dresidual = a->dresidual;
    k.dweight = a->dweight;
    k.dbias = a->dbias;
    k.partial = static_cast<float*>(a->workspace);
    k.dy_stride = dys;
    k.ds_stride = dss;
    k.x_stride = ss;
    k.rows = a->rows;
    k.cols = (uint32_t)a->cols;
    OnDevice guard(mcclx_ctx_device(ctx));
    if (!guard.ok) return fail(MCCLX_ERR_HIP, "hipSetDevice(%d) failed", mcclx_ctx_device(ctx));
    hipError_t e = hipSuccess;
    return launched(ctx, mcclx::launch_norm_backward(static_cast<hipStream_t>(stream), a->dtype, a->param_dtype, k, &e), e);
}

int mcclx_dropout(mcclx_ctx* ctx, void* stream, int dtype, uint64_t rows, uint64_t cols, const void* x, uint64_t x_stride,
                  const void* residual, uint64_t residual_stride, void* out, double p, uint64_t seed, uint64_t offset) {
    if (int rc = check_shape(ctx, dtype, rows, cols)) return rc;
    mcclx::DropoutArgs k = {};
    if (int rc = drop_args(p, seed, offset, &k.drop)) return rc;
    if (rows == 0 || cols == 0) return MCCLX_OK;
    uint64_t os = cols;
    Checker c{ctx};
    c.rows("x", x, true, size_of(dtype), rows, cols, &x_stride);
    c.rows("residual", residual, false, size_of(dtype), rows, cols, &residual_stride);
    c.rows("out", out, true, size_of(dtype), rows, cols, &os);
    if (c.rc) return c.rc;
    k.x = x;
    k.residual = residual;
    k.out = out;
    k.x_stride = x_stride;
    k.residual_stride = residual_stride;
    k.rows = rows;
    k.cols = (uint32_t)cols;
    OnDevice guard(mcclx_ctx_device(ctx));
    if (!guard.ok) return fail(MCCLX_ERR_HIP, "hipSetDevice(%d) failed", mcclx_ctx_device(ctx));
    hipError_t e = hipSuccess;
    return launched(ctx, mcclx::launch_dropout(static_cast<hipStream_t>(stream), dtype, k, mcclx_device_cus(ctx), &e), e);
}

int mcclx_linear_cross_entropy_forward(mcclx_ctx* ctx, void* stream, const mcclx_loss* a) { return loss(ctx, stream, a, false); }
int mcclx_linear_cross_entropy_backward(mcclx_ctx* ctx, void* stream, const mcclx_loss* a) { return loss(ctx, stream, a, true); }
uint64_t mcclx_linear_cross_entropy_workspace_bytes(mcclx_ctx* ctx, const mcclx_loss* a, int backward) {
    mcclx::LossArgs k;
    if (loss_args(ctx, a, &k)) return 0;
    return mcclx::loss_workspace_bytes(k, backward != 0, mcclx_device_cus(ctx));
}

}  // extern "C"
