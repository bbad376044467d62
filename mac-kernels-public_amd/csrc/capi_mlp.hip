// C ABI of the MLP side (include/qlin.h): argument checks and dispatch.  Host code only; the kernels
// live in add_norm.hip, gated_act.hip and w8a8.hip.
#include <cstdarg>
#include <cstdio>

#include "attention.h"
#include "mlp.h"

using namespace qlin;

namespace {

qlin_status fail(qlin_status s, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return report(s, buf);
}

qlin_status launched(hipError_t e, const char* what) {
    if (e == hipSuccess) return QLIN_OK;
    return fail(QLIN_EHIP, "%s: %s", what, hipGetErrorString(e));
}

bool is_float(int dt) { return dt == QLIN_DT_F32 || dt == QLIN_DT_F16 || dt == QLIN_DT_BF16; }

// Rows of one call: what the kernels' grids and 64-bit offsets count to with room to spare.
constexpr int64_t MOST_ROWS = (int64_t)1 << 31;

// t [T, W] with unit stride along the row (T, W < 0: any); written: rows may not overlap.
qlin_status rows_of(const qlin_tensor* t, const char* name, int64_t T, int64_t W, bool written, RowView& v) {
    if (!t) return fail(QLIN_EINVAL, "%s is missing", name);
    if (t->ndim != 2) return fail(QLIN_EINVAL, "%s must have 2 dimensions, it has %d", name, t->ndim);
    if (t->shape[0] < 0 || t->shape[1] < 0) return fail(QLIN_EINVAL, "%s has a negative size", name);
    if ((T >= 0 && t->shape[0] != T) || (W >= 0 && t->shape[1] != W))
        return fail(QLIN_EINVAL, "%s must be [%lld, %lld]", name, (long long)T, (long long)W);
    if (t->shape[0] && t->shape[1] && !t->data) return fail(QLIN_EINVAL, "%s is missing", name);
    if (t->shape[1] > 1 && t->stride[1] != 1) return fail(QLIN_EUNSUPPORTED, "%s needs unit stride along its rows", name);
    const int64_t ld = t->shape[0] > 1 ? t->stride[0] : 0;
    if (ld < 0) return fail(QLIN_EUNSUPPORTED, "%s has a negative stride", name);
    if (written && t->shape[0] > 1 && ld < t->shape[1]) return fail(QLIN_EINVAL, "%s has rows that overlap", name);
    v = {t->data, ld};
    return QLIN_OK;
}

// A contiguous vector of n elements, [n], [n, 1] or [1, n], of the given dtype (dtype < 0: any float).
qlin_status vector_of(const qlin_tensor* t, const char* name, int64_t n, int dtype) {
    if (!t) return fail(QLIN_EINVAL, "%s is missing", name);
    int64_t count = 1, stride = 1;
    for (int i = 0; i < t->ndim; ++i) {
        count *= t->shape[i];
        if (t->shape[i] > 1) stride = t->stride[i];
    }
    if (dtype < 0 ? !is_float(t->dtype) : t->dtype != dtype) return fail(QLIN_EUNSUPPORTED, "%s has an unsupported dtype", name);
    if (t->ndim > 2 || count != n || (t->ndim == 2 && t->shape[0] != 1 && t->shape[1] != 1)) return fail(QLIN_EINVAL, "%s has %lld elements, expected %lld", name, (long long)count, (long long)n);
    if (n > 0 && !t->data) return fail(QLIN_EINVAL, "%s is missing", name);
    if (n > 1 && stride != 1) return fail(QLIN_EUNSUPPORTED, "%s must be contiguous", name);
    return QLIN_OK;
}

qlin_status sizes_of(const qlin_tensor* t, const char* name, int64_t& T, int64_t& W) {
    if (!t) return fail(QLIN_EINVAL, "%s is missing", name);
    if (t->ndim != 2) return fail(QLIN_EINVAL, "%s must have 2 dimensions, it has %d", name, t->ndim);
    if (!is_float(t->dtype)) return fail(QLIN_EUNSUPPORTED, "%s dtype %d unsupported", name, t->dtype);
    T = t->shape[0];
    W = t->shape[1];
    if (T >= MOST_ROWS) return fail(QLIN_EUNSUPPORTED, "%s has too many rows", name);
    if (W > MLP_MAX_WIDTH) return fail(QLIN_EUNSUPPORTED, "rows of %lld values, more than %d", (long long)W, MLP_MAX_WIDTH);
    return QLIN_OK;
}

qlin_status group_of(int g, int64_t W) {
    if (g != 0 && g != 4 && g != 8 && g != 16 && g != 32 && g != 64 && g != 128 && g != 256)
        return fail(QLIN_EUNSUPPORTED, "ConvRot group %d unsupported", g);
    if (g && W % g) return fail(QLIN_EINVAL, "rows of %lld values are not a multiple of the ConvRot group %d", (long long)W, g);
    return QLIN_OK;
}

qlin_status codes_of(qlin_tensor* q, qlin_tensor* scale, int64_t T, int64_t W, int8_t*& qp, int64_t& ldq, float*& sp) {
    RowView v;
    if (qlin_status s = rows_of(q, "q", T, W, true, v)) return s;
    if (q->dtype != QLIN_DT_I8) return fail(QLIN_EUNSUPPORTED, "q must be int8");
    if (qlin_status s = vector_of(scale, "scale", T, QLIN_DT_F32)) return s;
    qp = (int8_t*)v.p;
    ldq = v.ld;
    sp = (float*)scale->data;
    return QLIN_OK;
}

qlin_status weight_of(const qlin_tensor* w, const char* name, int64_t W, const void*& p, int& dt) {
    p = nullptr;
    if (!w) return QLIN_OK;
    if (qlin_status s = vector_of(w, name, W, -1)) return s;
    p = w->data;
    dt = w->dtype;
    return QLIN_OK;
}

// The residual's side has x's dtype, or float32.
qlin_status side_dtype(int x, int h, const char* name) {
    if (h != x && h != QLIN_DT_F32) return fail(QLIN_EUNSUPPORTED, "%s must have x's dtype or float32", name);
    return QLIN_OK;
}

qlin_status norm_operands(const qlin_tensor* x, const qlin_tensor* residual, const qlin_tensor* weight, float eps,
                          qlin_tensor* h, AddNormArgs& a) {
    int64_t W;
    if (!(eps >= 0.0f)) return fail(QLIN_EINVAL, "eps must not be negative");
    if (qlin_status s = sizes_of(x, "x", a.T, W)) return s;
    a.W = (int)W;
    a.dtype = a.h_dtype = x->dtype;
    a.eps = eps;
    if (qlin_status s = rows_of(x, "x", -1, -1, false, a.x)) return s;
    if (!residual != !h) return fail(QLIN_EINVAL, "residual and h go together");
    if (residual) {
        a.h_dtype = residual->dtype;
        if (qlin_status s = side_dtype(a.dtype, a.h_dtype, "residual")) return s;
        if (qlin_status s = rows_of(residual, "residual", a.T, W, false, a.r)) return s;
        if (qlin_status s = rows_of(h, "h", a.T, W, true, a.h)) return s;
        if (h->dtype != residual->dtype) return fail(QLIN_EUNSUPPORTED, "h must have the residual's dtype");
    }
    return weight_of(weight, "weight", W, a.w, a.w_dt);
}

qlin_status act_operands(const qlin_tensor* gate, const qlin_tensor* up, int act, GatedActArgs& a) {
    int64_t W;
    if (act != QLIN_ACT_SILU && act != QLIN_ACT_GELU_TANH) return fail(QLIN_EUNSUPPORTED, "activation %d unsupported", act);
    if (qlin_status s = sizes_of(gate, "gate", a.T, W)) return s;
    a.W = (int)W;
    a.dtype = gate->dtype;
    a.act = act;
    if (qlin_status s = rows_of(gate, "gate", -1, -1, false, a.gate)) return s;
    if (!up) return QLIN_OK;
    if (up->dtype != gate->dtype) return fail(QLIN_EUNSUPPORTED, "up must have gate's dtype");
    return rows_of(up, "up", a.T, W, false, a.up);
}

// Rows like gate's, written.
qlin_status like_gate(qlin_tensor* t, const char* name, const GatedActArgs& a, RowView& v) {
    if (t && t->dtype != a.dtype) return fail(QLIN_EUNSUPPORTED, "%s must have gate's dtype", name);
    return rows_of(t, name, a.T, a.W, true, v);
}

}  // namespace

extern "C" {

qlin_status qlin_add_rms_norm(const qlin_tensor* x, const qlin_tensor* residual, const qlin_tensor* weight, float eps,
                              qlin_tensor* y, qlin_tensor* h, void* stream) {
    AddNormArgs a;
    if (qlin_status s = norm_operands(x, residual, weight, eps, h, a)) return s;
    if (qlin_status s = rows_of(y, "y", a.T, a.W, true, a.y)) return s;
    if (y->dtype != x->dtype) return fail(QLIN_EUNSUPPORTED, "y must have x's dtype");
    return launched(run_add_norm(a, (hipStream_t)stream), "norm");
}

qlin_status qlin_add_rms_norm_int8(const qlin_tensor* x, const qlin_tensor* residual, const qlin_tensor* weight, float eps,
                                   int convrot_groupsize, qlin_tensor* q, qlin_tensor* scale, qlin_tensor* h, void* stream) {
    AddNormArgs a;
    if (qlin_status s = norm_operands(x, residual, weight, eps, h, a)) return s;
    if (qlin_status s = group_of(convrot_groupsize, a.W)) return s;
    if (qlin_status s = codes_of(q, scale, a.T, a.W, a.q, a.ldq, a.scale)) return s;
    if (a.T > 0 && a.W == 0) return fail(QLIN_EUNSUPPORTED, "rows of no values have no scale");
    a.G = convrot_groupsize;
    return launched(run_add_norm(a, (hipStream_t)stream), "norm to int8");
}

qlin_status qlin_add_rms_norm_grad(const qlin_tensor* dy, const qlin_tensor* dh, const qlin_tensor* h, const qlin_tensor* weight,
                                   float eps, qlin_tensor* dx, qlin_tensor* dweight, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    AddNormGradArgs a;
    int64_t W;
    if (!(eps >= 0.0f)) return fail(QLIN_EINVAL, "eps must not be negative");
    if (qlin_status s = sizes_of(dy, "dy", a.T, W)) return s;
    a.W = (int)W;
    a.dtype = dy->dtype;
    a.eps = eps;
    if (qlin_status s = rows_of(dy, "dy", -1, -1, false, a.dy)) return s;
    if (qlin_status s = rows_of(h, "h", a.T, W, false, a.h)) return s;
    a.h_dtype = h->dtype;
    if (qlin_status s = side_dtype(a.dtype, a.h_dtype, "h")) return s;
    if (dh) {
        if (dh->dtype != h->dtype) return fail(QLIN_EUNSUPPORTED, "dh must have h's dtype");
        if (qlin_status s = rows_of(dh, "dh", a.T, W, false, a.dh)) return s;
    }
    if (qlin_status s = rows_of(dx, "dx", a.T, W, true, a.dx)) return s;
    if (dx->dtype != h->dtype) return fail(QLIN_EUNSUPPORTED, "dx must have h's dtype");
    if (qlin_status s = weight_of(weight, "weight", W, a.w, a.w_dt)) return s;
    const void* p;
    if (qlin_status s = weight_of(dweight, "dweight", W, p, a.dw_dt)) return s;
    a.dw = const_cast<void*>(p);
    if (a.dw && a.T) {
        const size_t need = ws_add_norm_grad(a.T, W);
        if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
            return fail(QLIN_EWORKSPACE, "workspace of %zu bytes, needs %zu (16-byte aligned)", workspace_bytes, need);
        a.part = (float*)workspace;
    }
    return launched(run_add_norm_grad(a, (hipStream_t)stream), "gradient of the norm");
}

qlin_status qlin_gated_act(const qlin_tensor* gate, const qlin_tensor* up, int act, qlin_tensor* y, void* stream) {
    GatedActArgs a;
    if (qlin_status s = act_operands(gate, up, act, a)) return s;
    if (qlin_status s = like_gate(y, "y", a, a.y)) return s;
    return launched(run_gated_act(a, (hipStream_t)stream), "gated activation");
}

qlin_status qlin_gated_act_int8(const qlin_tensor* gate, const qlin_tensor* up, int act, int convrot_groupsize, qlin_tensor* q,
                                qlin_tensor* scale, void* stream) {
    GatedActArgs a;
    if (qlin_status s = act_operands(gate, up, act, a)) return s;
    if (qlin_status s = group_of(convrot_groupsize, a.W)) return s;
    if (qlin_status s = codes_of(q, scale, a.T, a.W, a.q, a.ldq, a.scale)) return s;
    if (a.T > 0 && a.W == 0) return fail(QLIN_EUNSUPPORTED, "rows of no values have no scale");
    a.G = convrot_groupsize;
    return launched(run_gated_act(a, (hipStream_t)stream), "gated activation to int8");
}

qlin_status qlin_gated_act_grad(const qlin_tensor* dy, const qlin_tensor* gate, const qlin_tensor* up, int act,
                                qlin_tensor* dgate, qlin_tensor* dup, void* stream) {
    GatedActArgs a;
    if (qlin_status s = act_operands(gate, up, act, a)) return s;
    if (!dy || dy->dtype != a.dtype) return fail(dy ? QLIN_EUNSUPPORTED : QLIN_EINVAL, "dy must have gate's dtype");
    if (qlin_status s = rows_of(dy, "dy", a.T, a.W, false, a.dy)) return s;
    if (qlin_status s = like_gate(dgate, "dgate", a, a.dgate)) return s;
    if (!up != !dup) return fail(QLIN_EINVAL, "up and dup go together");
    if (up)
        if (qlin_status s = like_gate(dup, "dup", a, a.dup)) return s;
    return launched(run_gated_act_grad(a, (hipStream_t)stream), "gradient of the gated activation");
}

qlin_status qlin_w8a8_linear(const qlin_tensor* x, const qlin_tensor* x_scale, const qlin_tensor* qdata, const qlin_tensor* scale,
                             const qlin_tensor* bias, const qlin_tensor* residual, const qlin_tensor* residual_scale,
                             qlin_tensor* y, void* workspace, size_t workspace_bytes, void* stream) {
    W8A8Args a;
    RowView v;
    if (qlin_status s = rows_of(x, "x", -1, -1, false, v)) return s;
    if (x->dtype != QLIN_DT_I8) return fail(QLIN_EUNSUPPORTED, "x must be int8");
    a.M = x->shape[0];
    a.K = x->shape[1];
    a.x = (const int8_t*)v.p;
    a.ldx = v.ld;
    if (qlin_status s = rows_of(qdata, "qdata", -1, a.K, false, v)) {
        if (qdata && qdata->ndim == 2 && qdata->shape[1] != a.K)
            return fail(QLIN_EINVAL, "x has K=%lld, weight has K=%lld", (long long)a.K, (long long)qdata->shape[1]);
        return s;
    }
    if (qdata->dtype != QLIN_DT_I8) return fail(QLIN_EUNSUPPORTED, "qdata must be int8");
    a.N = qdata->shape[0];
    a.w = (const int8_t*)v.p;
    a.ldw = a.N > 1 ? v.ld : a.K;
    if (a.M == 1) a.ldx = a.K;
    if (a.K > W8A8_MAX_K) return fail(QLIN_EUNSUPPORTED, "K > %d", W8A8_MAX_K);
    if (a.M >= W8A8_MOST_ROWS || a.N >= W8A8_MOST_OUTPUTS || (a.N && a.M > W8A8_MOST_RESULTS / a.N))
        return fail(QLIN_EUNSUPPORTED, "%lld rows by %lld outputs are too many", (long long)a.M, (long long)a.N);
    if (qlin_status s = vector_of(x_scale, "x_scale", a.M, QLIN_DT_F32)) return s;
    if (qlin_status s = vector_of(scale, "scale", a.N, QLIN_DT_F32)) return s;
    a.sx = (const float*)x_scale->data;
    a.sw = (const float*)scale->data;
    if (bias) {
        if (qlin_status s = vector_of(bias, "bias", a.N, -1)) return s;
        a.bias = bias->data;
        a.bias_dt = bias->dtype;
    }
    if (qlin_status s = rows_of(y, "y", a.M, a.N, true, v)) return s;
    if (!is_float(y->dtype)) return fail(QLIN_EUNSUPPORTED, "y dtype %d unsupported", y->dtype);
    a.y = v.p;
    a.y_dt = y->dtype;
    a.ldy = a.M > 1 ? v.ld : a.N;
    if (residual) {
        if (qlin_status s = rows_of(residual, "residual", a.M, a.N, false, v)) return s;
        if (!is_float(residual->dtype)) return fail(QLIN_EUNSUPPORTED, "residual must be f32/f16/bf16");
        a.res.r = v.p;
        a.res.r_dt = residual->dtype;
        a.res.ldr = a.M > 1 ? v.ld : a.N;
        if (residual_scale) {
            if (qlin_status s = vector_of(residual_scale, "residual_scale", a.N, -1)) return s;
            a.res.rs = residual_scale->data;
            a.res.rs_dt = residual_scale->dtype;
        }
    } else if (residual_scale) {
        return fail(QLIN_EINVAL, "residual_scale given without residual");
    }
    if (a.M == 0 || a.N == 0) return QLIN_OK;
    if (a.K == 0) return fail(QLIN_EUNSUPPORTED, "rows of no values");
    const size_t need = ws_w8a8(a.M, a.N, a.K, w8a8_apart(a));
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256))
        return fail(QLIN_EWORKSPACE, "workspace of %zu bytes, needs %zu (256-byte aligned)", workspace_bytes, need);
    a.ws = workspace;
    return launched(run_w8a8(a, (hipStream_t)stream), "w8a8 linear");
}

}  // extern "C"
