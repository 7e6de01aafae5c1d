// C ABI of the row operators (include/srmi.h, "Row operators"): validation on the host, then the launches.
#include "common.h"

namespace srmi {

int linear_fwd(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, void* ws,
               hipStream_t s);
int linear_bwd(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw, void* db,
               void* ws, hipStream_t s);
size_t linear_workspace_bytes(const srmi_linear_desc& d, int pass);
bool linear_too_wide(const srmi_linear_desc& d);
int norm_fwd(const srmi_norm_desc& d, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, hipStream_t s);
int norm_bwd(const srmi_norm_desc& d, const void* x, const void* w, const float* mean, const float* rstd, const void* dy, void* dx,
             void* dw, void* db, float* ws, hipStream_t s);
size_t norm_workspace_bytes(const srmi_norm_desc& d);
int dropout(const void* x, const void* residual, void* y, long long n, double p, unsigned long long seed, unsigned long long offset,
            const unsigned long long* rng, int dtype, hipStream_t s);

static bool is_dtype(int v) { return v == SRMI_F32 || v == SRMI_BF16; }
static size_t dsize(int dtype) { return dtype == SRMI_BF16 ? 2 : 4; }

// pointers are aligned to their element; a linear call may promise 16 bytes for the products' operands
static bool element_aligned(const void* p, int dtype) { return ((uintptr_t)p & (dsize(dtype) - 1)) == 0; }
static bool linear_aligned(const srmi_linear_desc* d, const void* p) { return d->align >= 16 ? ((uintptr_t)p & 15) == 0 : element_aligned(p, d->dtype); }

static int check_linear(const srmi_linear_desc* d, const char* who) {
    if (!d) { set_error("%s: NULL descriptor", who); return SRMI_EINVAL; }
    if (d->M < 0 || d->N < 0 || d->K < 0 || d->M > SRMI_ROWS_MAX) {
        set_error("%s: bad sizes M=%lld N=%d K=%d", who, (long long)d->M, d->N, d->K);
        return SRMI_EINVAL;
    }
    if (!is_dtype(d->dtype)) { set_error("%s: bad dtype %d", who, d->dtype); return SRMI_EINVAL; }
    if (linear_too_wide(*d)) { set_error("%s: N=%d or K=%d over 2^22", who, d->N, d->K); return SRMI_EUNSUPPORTED; }
    switch (d->act) {
        case SRMI_ACT_NONE: case SRMI_ACT_LRELU: case SRMI_ACT_RELU: case SRMI_ACT_TANH: case SRMI_ACT_SIGMOID:
        case SRMI_ACT_GELU: case SRMI_ACT_GELU_TANH: case SRMI_ACT_SILU: break;
        default: set_error("%s: activation %d is not one of the row operators'", who, d->act); return SRMI_EUNSUPPORTED;
    }
    if (d->ldx < d->K || d->ldw < d->K || d->ldr < 0 || (d->ldr && d->ldr < d->N) || d->lddy < 0 || (d->lddy && d->lddy < d->N)) {
        set_error("%s: a row stride is shorter than its row (ldx=%lld ldw=%lld ldr=%lld lddy=%lld, K=%d N=%d)", who, (long long)d->ldx,
                  (long long)d->ldw, (long long)d->ldr, (long long)d->lddy, d->K, d->N);
        return SRMI_EINVAL;
    }
    return SRMI_OK;
}

static int check_norm(const srmi_norm_desc* d, const char* who) {
    if (!d) { set_error("%s: NULL descriptor", who); return SRMI_EINVAL; }
    if (d->rows < 0 || d->rows > SRMI_ROWS_MAX || d->C <= 0) {
        set_error("%s: bad sizes rows=%lld C=%d", who, (long long)d->rows, d->C);
        return SRMI_EINVAL;
    }
    if (d->C > SRMI_NORM_MAX_C) { set_error("%s: C=%d over 2^25", who, d->C); return SRMI_EUNSUPPORTED; }
    if (!is_dtype(d->dtype) || !is_dtype(d->param_dtype)) { set_error("%s: bad dtype", who); return SRMI_EINVAL; }
    if (!(d->eps >= 0.f)) { set_error("%s: eps must be >= 0", who); return SRMI_EINVAL; }
    if (d->ldx < d->C || d->lddy < 0 || (d->lddy && d->lddy < d->C)) {
        set_error("%s: a row stride is shorter than its row (ldx=%lld lddy=%lld, C=%d)", who, (long long)d->ldx, (long long)d->lddy, d->C);
        return SRMI_EINVAL;
    }
    return SRMI_OK;
}

}  // namespace srmi

using namespace srmi;

extern "C" {

int srmi_linear_workspace_bytes(const srmi_linear_desc* d, int32_t pass, size_t* bytes) {
    const int rc = check_linear(d, "linear_workspace_bytes");
    if (rc) return rc;
    if (!bytes || (pass != SRMI_PASS_FWD && pass != SRMI_PASS_BWD)) { set_error("linear_workspace_bytes: NULL argument or bad pass"); return SRMI_EINVAL; }
    *bytes = linear_workspace_bytes(*d, pass);
    return SRMI_OK;
}

int srmi_linear_fwd(const srmi_linear_desc* d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z,
                    void* ws, size_t ws_bytes, void* stream) {
    const int rc = check_linear(d, "linear_fwd");
    if (rc) return rc;
    if (d->M == 0 || d->N == 0) return SRMI_OK;
    if (!y || (d->K > 0 && (!x || !w))) { set_error("linear_fwd: NULL argument"); return SRMI_EINVAL; }
    if (residual && d->ldr < d->N) { set_error("linear_fwd: residual without its row stride"); return SRMI_EINVAL; }
    if (!linear_aligned(d, x) || !linear_aligned(d, w) || !element_aligned(bias, d->dtype) ||
        !element_aligned(residual, d->dtype) || !element_aligned(y, d->dtype) || !element_aligned(z, d->dtype)) {
        set_error("linear_fwd: an operand is not aligned to its element, or not as d->align says");
        return SRMI_EINVAL;
    }
    const size_t need = linear_workspace_bytes(*d, SRMI_PASS_FWD);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 255))) {
        set_error("linear_fwd: workspace of %zu bytes, 256-byte aligned, needed", need);
        return SRMI_EINVAL;
    }
    return linear_fwd(*d, x, w, bias, residual, y, z, ws, (hipStream_t)stream);
}

int srmi_linear_bwd(const srmi_linear_desc* d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw, void* db,
                    void* ws, size_t ws_bytes, void* stream) {
    const int rc = check_linear(d, "linear_bwd");
    if (rc) return rc;
    if (d->M > 0 && d->N > 0 && (!dy || d->lddy < d->N || (d->act != SRMI_ACT_NONE && !saved))) {
        set_error("linear_bwd: NULL dy / saved, or dy without its row stride");
        return SRMI_EINVAL;
    }
    if ((dw && d->M > 0 && d->K > 0 && !x) || (dx && d->N > 0 && d->K > 0 && !w)) { set_error("linear_bwd: NULL x or w"); return SRMI_EINVAL; }
    if (!linear_aligned(d, x) || !linear_aligned(d, w) || !element_aligned(saved, d->dtype) || !linear_aligned(d, dy) ||
        !element_aligned(dx, d->dtype) || !element_aligned(dw, d->dtype) || !element_aligned(db, d->dtype)) {
        set_error("linear_bwd: an operand is not aligned to its element, or not as d->align says");
        return SRMI_EINVAL;
    }
    const size_t need = linear_workspace_bytes(*d, SRMI_PASS_BWD);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 255))) {
        set_error("linear_bwd: workspace of %zu bytes, 256-byte aligned, needed", need);
        return SRMI_EINVAL;
    }
    return linear_bwd(*d, x, w, saved, dy, dx, dw, db, ws, (hipStream_t)stream);
}

int srmi_layer_norm_fwd(const srmi_norm_desc* d, const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                        void* stream) {
    const int rc = check_norm(d, "layer_norm_fwd");
    if (rc) return rc;
    if (d->rows == 0) return SRMI_OK;
    if (!x || !y || !mean != !rstd) { set_error("layer_norm_fwd: NULL argument (mean and rstd go together)"); return SRMI_EINVAL; }
    if (!element_aligned(x, d->dtype) || !element_aligned(y, d->dtype) || !element_aligned(weight, d->param_dtype) ||
        !element_aligned(bias, d->param_dtype) || !element_aligned(mean, SRMI_F32) || !element_aligned(rstd, SRMI_F32)) {
        set_error("layer_norm_fwd: an operand is not aligned to its element");
        return SRMI_EINVAL;
    }
    return norm_fwd(*d, x, weight, bias, y, mean, rstd, (hipStream_t)stream);
}

int srmi_layer_norm_workspace_bytes(const srmi_norm_desc* d, size_t* bytes) {
    const int rc = check_norm(d, "layer_norm_workspace_bytes");
    if (rc) return rc;
    if (!bytes) { set_error("layer_norm_workspace_bytes: NULL argument"); return SRMI_EINVAL; }
    *bytes = norm_workspace_bytes(*d);
    return SRMI_OK;
}

int srmi_layer_norm_bwd(const srmi_norm_desc* d, const void* x, const void* weight, const float* mean, const float* rstd, const void* dy,
                        void* dx, void* dweight, void* dbias, void* ws, size_t ws_bytes, void* stream) {
    const int rc = check_norm(d, "layer_norm_bwd");
    if (rc) return rc;
    if (!dweight && !dbias && (!dx || d->rows == 0)) return SRMI_OK;      // (gradients of the parameters are zeros then, and written)
    if (d->rows > 0 && (!x || !mean || !rstd || !dy || d->lddy < d->C)) { set_error("layer_norm_bwd: NULL argument, or dy without its row stride"); return SRMI_EINVAL; }
    if (!element_aligned(x, d->dtype) || !element_aligned(dy, d->dtype) || !element_aligned(dx, d->dtype) ||
        !element_aligned(weight, d->param_dtype) || !element_aligned(dweight, d->param_dtype) || !element_aligned(dbias, d->param_dtype) ||
        !element_aligned(mean, SRMI_F32) || !element_aligned(rstd, SRMI_F32)) {
        set_error("layer_norm_bwd: an operand is not aligned to its element");
        return SRMI_EINVAL;
    }
    if (dweight || dbias) {
        const size_t need = norm_workspace_bytes(*d);
        if (!ws || ws_bytes < need || ((uintptr_t)ws & 15)) { set_error("layer_norm_bwd: workspace of %zu bytes, 16-byte aligned, needed", need); return SRMI_EINVAL; }
    }
    return norm_bwd(*d, x, weight, mean, rstd, dy, dx, dweight, dbias, (float*)ws, (hipStream_t)stream);
}

int srmi_dropout(const void* x, const void* residual, void* y, size_t n, int32_t dtype, double p, uint64_t seed, uint64_t offset,
                 const uint64_t* rng, void* stream) {
    if (!is_dtype(dtype)) { set_error("dropout: bad dtype %d", dtype); return SRMI_EINVAL; }
    if (!(p >= 0.0 && p <= 1.0)) { set_error("dropout: p must be in [0, 1]"); return SRMI_EINVAL; }
    if (n > ((size_t)1 << 48)) { set_error("dropout: more than 2^48 elements"); return SRMI_EINVAL; }
    if (n == 0) return SRMI_OK;
    if (!x || !y) { set_error("dropout: NULL argument"); return SRMI_EINVAL; }
    if (!element_aligned(x, dtype) || !element_aligned(residual, dtype) || !element_aligned(y, dtype) || ((uintptr_t)rng & 7)) {
        set_error("dropout: an operand is not aligned to its element");
        return SRMI_EINVAL;
    }
    return dropout(x, residual, y, (long long)n, p, seed, offset, (const unsigned long long*)rng, dtype, (hipStream_t)stream);
}

}  // extern "C"
