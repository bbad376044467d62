// C ABI of the attention side (include/qlin.h): argument checks and dispatch.  Host code only;
// the kernels live in qk_rope.hip, paged_plan.hip and paged_attention.hip.
#include <cstdarg>
#include <cstdio>

#include "attention.h"

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
bool present(const qlin_tensor* t) { return t && t->data; }

// The stride of a dimension; nothing moves along one of a single element, whatever its stride says.
int64_t step(const qlin_tensor* t, int i) { return t->shape[i] > 1 ? t->stride[i] : 0; }

// Sizes that the kernels index with 32 bits.
constexpr int64_t INT_MOST = 0x7FFFFFFF;

// The memory of t is there for every index: no empty dimension of an absent pointer is looked at.
qlin_status has_data(const qlin_tensor* t, const char* name, int ndim) {
    if (!t) return fail(QLIN_EINVAL, "%s is missing", name);
    if (t->ndim != ndim) return fail(QLIN_EINVAL, "%s must have %d dimensions, it has %d", name, ndim, t->ndim);
    bool empty = false;
    for (int i = 0; i < ndim; ++i) {
        if (t->shape[i] < 0) return fail(QLIN_EINVAL, "%s has a negative size", name);
        empty |= t->shape[i] == 0;
    }
    if (!empty && !t->data) return fail(QLIN_EINVAL, "%s is missing", name);
    return QLIN_OK;
}

// [tokens, heads, D], unit stride along D.
qlin_status head_view(const qlin_tensor* t, const char* name, int dtype, int64_t T, int64_t H, int64_t D, HeadView& v) {
    if (qlin_status s = has_data(t, name, 3)) return s;
    if (t->dtype != dtype) return fail(QLIN_EUNSUPPORTED, "%s must have q's dtype", name);
    if (t->shape[0] != T || t->shape[1] != H || t->shape[2] != D)
        return fail(QLIN_EINVAL, "%s must be [%lld, %lld, %lld]", name, (long long)T, (long long)H, (long long)D);
    if (D > 1 && t->stride[2] != 1) return fail(QLIN_EUNSUPPORTED, "%s needs unit stride along the head", name);
    v = {t->data, step(t, 0), step(t, 1)};
    return QLIN_OK;
}

qlin_status cache_view(const qlin_tensor* t, const char* name, int dtype, int64_t H, int64_t D, int64_t& blocks,
                       int64_t& page, CacheView& v) {
    if (qlin_status s = has_data(t, name, 4)) return s;
    if (t->dtype != dtype) return fail(QLIN_EUNSUPPORTED, "%s must have q's dtype", name);
    if (blocks < 0) {
        blocks = t->shape[0];
        page = t->shape[1];
    }
    if (t->shape[0] != blocks || t->shape[1] != page || t->shape[2] != H || t->shape[3] != D)
        return fail(QLIN_EINVAL, "%s must be [%lld, %lld, %lld, %lld]", name, (long long)blocks, (long long)page, (long long)H,
                    (long long)D);
    if (page < 1) return fail(QLIN_EINVAL, "%s has pages of no token", name);
    if (page > INT_MOST || blocks > INT_MOST) return fail(QLIN_EUNSUPPORTED, "%s: too many blocks or places a block", name);
    if (D > 1 && t->stride[3] != 1) return fail(QLIN_EUNSUPPORTED, "%s needs unit stride along the head", name);
    v = {t->data, step(t, 0), step(t, 1), step(t, 2)};
    return QLIN_OK;
}

// A contiguous [n] of the given dtype (dtype < 0: any float).
qlin_status vector_of(const qlin_tensor* t, const char* name, int64_t n, int dtype) {
    if (qlin_status s = has_data(t, name, 1)) return s;
    if (dtype < 0 ? !is_float(t->dtype) : t->dtype != dtype) return fail(QLIN_EUNSUPPORTED, "%s has an unsupported dtype", name);
    if (t->shape[0] != n) return fail(QLIN_EINVAL, "%s has %lld elements, expected %lld", name, (long long)t->shape[0], (long long)n);
    if (n > 1 && t->stride[0] != 1) return fail(QLIN_EUNSUPPORTED, "%s must be contiguous", name);
    return QLIN_OK;
}

// Memory of rows of `width` bytes, `step` apart; a vector is one row.
struct Range {
    const char* name;
    uintptr_t p;
    int64_t width, rows, step;
};

Range range_of(const qlin_tensor* t, const char* name, int es) {
    if (t->ndim == 1) return {name, (uintptr_t)t->data, t->shape[0] * es, 1, 0};
    return {name, (uintptr_t)t->data, t->shape[1] * es, t->shape[0], step(t, 0) * es};
}

// Whether the vector v and the rows r share a byte.
bool share_memory(const Range& v, const Range& r) {
    if (v.width == 0 || r.width == 0 || r.rows == 0) return false;
    if (v.p + v.width <= r.p || v.p >= r.p + (r.rows - 1) * r.step + r.width) return false;
    if (v.p < r.p || r.rows == 1) return true;
    const int64_t at = (int64_t)(v.p - r.p), in = at % r.step;
    return in < r.width || (in + v.width > r.step && at / r.step + 1 < r.rows);
}

qlin_status turn_of(const qlin_tensor* positions, const qlin_tensor* inv_freq, const qlin_tensor* axis, int flags, int64_t T,
                    int64_t D, RopeTurn& r) {
    if (flags & ~(QLIN_ROPE_INTERLEAVED | QLIN_ROPE_INVERSE)) return fail(QLIN_EINVAL, "unknown flags %d", flags);
    r.interleaved = flags & QLIN_ROPE_INTERLEAVED;
    r.inverse = flags & QLIN_ROPE_INVERSE;
    if (!inv_freq) return fail(QLIN_EINVAL, "inv_freq is missing");
    const int64_t P = inv_freq->ndim == 1 ? inv_freq->shape[0] : -1;
    if (qlin_status s = vector_of(inv_freq, "inv_freq", P, QLIN_DT_F32)) return s;
    if (2 * P > D) return fail(QLIN_EINVAL, "inv_freq has %lld pairs, a head of %lld values holds %lld", (long long)P,
                               (long long)D, (long long)(D / 2));
    r.P = (int)P;
    r.inv_freq = (const float*)inv_freq->data;
    if (P == 0) return QLIN_OK;
    if (axis) {
        if (qlin_status s = vector_of(axis, "axis", P, QLIN_DT_I32)) return s;
        r.axis = (const int32_t*)axis->data;
    }
    if (!positions) return fail(QLIN_EINVAL, "positions is missing");
    const int nd = positions->ndim == 2 ? 2 : 1;
    if (qlin_status s = has_data(positions, "positions", nd)) return s;
    if (positions->dtype != QLIN_DT_I32 && positions->dtype != QLIN_DT_I64 && positions->dtype != QLIN_DT_F32)
        return fail(QLIN_EUNSUPPORTED, "positions must be int32, int64 or float32");
    if (positions->shape[nd - 1] != T || (nd == 2 && (positions->shape[0] < 1 || positions->shape[0] > INT_MOST)))
        return fail(QLIN_EINVAL, "positions must be [axes, %lld]", (long long)T);
    r.pos = positions->data;
    r.pos_dt = positions->dtype;
    r.pos_st = step(positions, nd - 1);
    r.pos_sa = nd == 2 ? step(positions, 0) : 0;
    r.axes = nd == 2 ? (int)positions->shape[0] : 1;
    return QLIN_OK;
}

// q [tokens, heads, D] sets the sizes of a call.
qlin_status head_sizes(const qlin_tensor* q, const char* name, int64_t& T, int64_t& H, int64_t& D) {
    if (qlin_status s = has_data(q, name, 3)) return s;
    if (!is_float(q->dtype)) return fail(QLIN_EUNSUPPORTED, "%s dtype %d unsupported", name, q->dtype);
    T = q->shape[0];
    H = q->shape[1];
    D = q->shape[2];
    if (D > ROPE_MAX_DIM) return fail(QLIN_EUNSUPPORTED, "heads of %lld values, more than %d", (long long)D, ROPE_MAX_DIM);
    if (H > ROPE_MAX_HEADS) return fail(QLIN_EUNSUPPORTED, "more than %d heads", ROPE_MAX_HEADS);
    if (T > INT_MOST / 2) return fail(QLIN_EUNSUPPORTED, "more than %lld tokens", (long long)(INT_MOST / 2));
    return QLIN_OK;
}

qlin_status weight_of(const qlin_tensor* w, const char* name, int64_t D, const void*& p, int& dt) {
    p = nullptr;
    if (!w) return QLIN_OK;
    if (qlin_status s = vector_of(w, name, D, -1)) return s;
    p = w->data;
    dt = w->dtype;
    return QLIN_OK;
}

// What the three forward entry points share: sizes, q (and k), weights and the rotation.
qlin_status forward_operands(const qlin_tensor* q, const qlin_tensor* k, const qlin_tensor* wq, const qlin_tensor* wk,
                             const qlin_tensor* positions, const qlin_tensor* inv_freq, const qlin_tensor* axis, int flags,
                             HeadRopeArgs& a) {
    int64_t H, D, Hk = 0;
    if (qlin_status s = head_sizes(q, "q", a.T, H, D)) return s;
    a.dtype = q->dtype;
    a.Hq = (int)H;
    a.D = (int)D;
    if (qlin_status s = head_view(q, "q", a.dtype, a.T, H, D, a.q)) return s;
    if (k) {
        Hk = k->ndim == 3 ? k->shape[1] : 0;
        if (Hk > ROPE_MAX_HEADS) return fail(QLIN_EUNSUPPORTED, "more than %d heads", ROPE_MAX_HEADS);
        if (qlin_status s = head_view(k, "k", a.dtype, a.T, Hk, D, a.k)) return s;
        a.Hk = (int)Hk;
    } else if (wk) {
        return fail(QLIN_EINVAL, "k_weight given without k");
    }
    if (qlin_status s = weight_of(wq, "q_weight", D, a.wq, a.wq_dt)) return s;
    if (qlin_status s = weight_of(wk, "k_weight", D, a.wk, a.wk_dt)) return s;
    return turn_of(positions, inv_freq, axis, flags, a.T, D, a.turn);
}

qlin_status forward_outputs(qlin_tensor* q_out, qlin_tensor* k_out, const qlin_tensor* k, HeadRopeArgs& a) {
    if (qlin_status s = head_view(q_out, "q_out", a.dtype, a.T, a.Hq, a.D, a.qo)) return s;
    if (!k != !k_out) return fail(QLIN_EINVAL, "k and k_out go together");
    if (k)
        if (qlin_status s = head_view(k_out, "k_out", a.dtype, a.T, a.Hk, a.D, a.ko)) return s;
    return QLIN_OK;
}

bool nothing(const HeadRopeArgs& a) { return a.T == 0 || a.D == 0 || a.Hq + a.Hk == 0; }

}  // namespace

extern "C" {

qlin_status qlin_axis_rope(const qlin_tensor* q, const qlin_tensor* k, const qlin_tensor* positions,
                           const qlin_tensor* inv_freq, const qlin_tensor* axis, int flags, qlin_tensor* q_out,
                           qlin_tensor* k_out, void* stream) {
    HeadRopeArgs a;
    if (qlin_status s = forward_operands(q, k, nullptr, nullptr, positions, inv_freq, axis, flags, a)) return s;
    if (qlin_status s = forward_outputs(q_out, k_out, k, a)) return s;
    if (nothing(a)) return QLIN_OK;
    return launched(run_head_rope(a, (hipStream_t)stream), "rotation");
}

qlin_status qlin_qk_norm_rope(const qlin_tensor* q, const qlin_tensor* k, const qlin_tensor* q_weight,
                              const qlin_tensor* k_weight, float eps, const qlin_tensor* positions,
                              const qlin_tensor* inv_freq, const qlin_tensor* axis, int flags, qlin_tensor* q_out,
                              qlin_tensor* k_out, void* stream) {
    HeadRopeArgs a;
    if (!(eps >= 0.0f)) return fail(QLIN_EINVAL, "eps must not be negative");
    a.norm = true;
    a.eps = eps;
    if (qlin_status s = forward_operands(q, k, q_weight, k_weight, positions, inv_freq, axis, flags, a)) return s;
    if (qlin_status s = forward_outputs(q_out, k_out, k, a)) return s;
    if (nothing(a)) return QLIN_OK;
    return launched(run_head_rope(a, (hipStream_t)stream), "head norms and rotation");
}

qlin_status qlin_qk_norm_rope_store(const qlin_tensor* q, const qlin_tensor* k, const qlin_tensor* v,
                                    const qlin_tensor* q_weight, const qlin_tensor* k_weight, float eps,
                                    const qlin_tensor* positions, const qlin_tensor* inv_freq, const qlin_tensor* axis,
                                    int flags, const qlin_tensor* slots, qlin_tensor* q_out, qlin_tensor* k_cache,
                                    qlin_tensor* v_cache, void* stream) {
    HeadRopeArgs a;
    if (eps != eps) return fail(QLIN_EINVAL, "eps is not a number");
    a.norm = eps >= 0.0f;
    a.eps = eps;
    if (!a.norm && (q_weight || k_weight)) return fail(QLIN_EINVAL, "weights given without the norms");
    if (!k) return fail(QLIN_EINVAL, "k is missing");
    if (qlin_status s = forward_operands(q, k, q_weight, k_weight, positions, inv_freq, axis, flags, a)) return s;
    if (qlin_status s = head_view(v, "v", a.dtype, a.T, a.Hk, a.D, a.v)) return s;
    if (qlin_status s = head_view(q_out, "q_out", a.dtype, a.T, a.Hq, a.D, a.qo)) return s;
    a.store = true;
    a.blocks = -1;
    if (qlin_status s = cache_view(k_cache, "k_cache", a.dtype, a.Hk, a.D, a.blocks, a.page, a.kc)) return s;
    if (qlin_status s = cache_view(v_cache, "v_cache", a.dtype, a.Hk, a.D, a.blocks, a.page, a.vc)) return s;
    if (qlin_status s = has_data(slots, "slots", 1)) return s;
    if (slots->dtype != QLIN_DT_I32 && slots->dtype != QLIN_DT_I64) return fail(QLIN_EUNSUPPORTED, "slots must be int32 or int64");
    if (slots->shape[0] != a.T) return fail(QLIN_EINVAL, "slots must be [%lld]", (long long)a.T);
    a.slots = slots->data;
    a.slots_dt = slots->dtype;
    a.slots_st = step(slots, 0);
    if (nothing(a)) return QLIN_OK;
    return launched(run_head_rope(a, (hipStream_t)stream), "head norms, rotation and cache");
}

qlin_status qlin_qk_norm_rope_grad(const qlin_tensor* dq_out, const qlin_tensor* dk_out, const qlin_tensor* q,
                                   const qlin_tensor* k, const qlin_tensor* q_weight, const qlin_tensor* k_weight, float eps,
                                   const qlin_tensor* positions, const qlin_tensor* inv_freq, const qlin_tensor* axis,
                                   int flags, qlin_tensor* dq, qlin_tensor* dk, qlin_tensor* dq_weight,
                                   qlin_tensor* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
    HeadRopeArgs f;
    if (!(eps >= 0.0f)) return fail(QLIN_EINVAL, "eps must not be negative");
    if (qlin_status s = forward_operands(q, k, q_weight, k_weight, positions, inv_freq, axis, flags, f)) return s;
    HeadGradArgs a;
    a.dtype = f.dtype; a.T = f.T; a.Hq = f.Hq; a.Hk = f.Hk; a.D = f.D; a.q = f.q; a.k = f.k; a.eps = eps;
    a.wq = f.wq; a.wk = f.wk; a.wq_dt = f.wq_dt; a.wk_dt = f.wk_dt; a.turn = f.turn;
    if (qlin_status s = head_view(dq_out, "dq_out", a.dtype, a.T, a.Hq, a.D, a.gq)) return s;
    if (qlin_status s = head_view(dq, "dq", a.dtype, a.T, a.Hq, a.D, a.dq)) return s;
    if (!k != !dk_out || !k != !dk || (!k && dk_weight)) return fail(QLIN_EINVAL, "k, dk_out and dk go together");
    if (k) {
        if (qlin_status s = head_view(dk_out, "dk_out", a.dtype, a.T, a.Hk, a.D, a.gk)) return s;
        if (qlin_status s = head_view(dk, "dk", a.dtype, a.T, a.Hk, a.D, a.dk)) return s;
    }
    const void* p;
    if (qlin_status s = weight_of(dq_weight, "dq_weight", a.D, p, a.dwq_dt)) return s;
    a.dwq = const_cast<void*>(p);
    if (qlin_status s = weight_of(dk_weight, "dk_weight", a.D, p, a.dwk_dt)) return s;
    a.dwk = const_cast<void*>(p);
    if (a.D == 0) return QLIN_OK;
    if (a.dwq || a.dwk) {
        if (!workspace || workspace_bytes < ws_head_grad(a.T, a.Hq + a.Hk, a.D) || (uintptr_t)workspace % 16)
            return fail(QLIN_EWORKSPACE, "workspace of %zu bytes, needs %zu (16-byte aligned)", workspace_bytes,
                        ws_head_grad(a.T, a.Hq + a.Hk, a.D));
        a.part = (float*)workspace;
    }
    return launched(run_head_grad(a, (hipStream_t)stream), "gradient of the head norms and rotation");
}

qlin_status qlin_paged_plan(const qlin_tensor* context, const qlin_tensor* added, const qlin_tensor* free_blocks,
                            int64_t page, qlin_tensor* block_table, qlin_tensor* slots, qlin_tensor* positions,
                            qlin_tensor* rows, qlin_tensor* starts, qlin_tensor* lengths, qlin_tensor* used, void* stream) {
    PagedPlanArgs a;
    if (page < 1 || page > INT_MOST) return fail(QLIN_EINVAL, "pages of %lld tokens", (long long)page);
    a.page = page;
    const int64_t B = context && context->ndim == 1 ? context->shape[0] : 0;
    if (qlin_status s = vector_of(context, "context", B, QLIN_DT_I32)) return s;
    if (B > QLIN_PLAN_MAX_REQUESTS) return fail(QLIN_EUNSUPPORTED, "%lld requests, more than %d", (long long)B, QLIN_PLAN_MAX_REQUESTS);
    if (qlin_status s = vector_of(added, "added", B, QLIN_DT_I32)) return s;
    a.F = free_blocks && free_blocks->ndim == 1 ? free_blocks->shape[0] : 0;
    if (qlin_status s = vector_of(free_blocks, "free_blocks", a.F, QLIN_DT_I32)) return s;
    if (qlin_status s = has_data(block_table, "block_table", 2)) return s;
    if (block_table->dtype != QLIN_DT_I32) return fail(QLIN_EUNSUPPORTED, "block_table must be int32");
    a.W = block_table->shape[1];
    if (block_table->shape[0] != B) return fail(QLIN_EINVAL, "block_table must have %lld rows", (long long)B);
    if (a.W > 1 && block_table->stride[1] != 1) return fail(QLIN_EUNSUPPORTED, "block_table needs unit column stride");
    if (B > 1 && a.W > 0 && block_table->stride[0] < a.W) return fail(QLIN_EINVAL, "block_table's rows overlap");
    a.ldt = step(block_table, 0);
    a.N = slots && slots->ndim == 1 ? slots->shape[0] : 0;
    if (a.N > INT_MOST - 4096) return fail(QLIN_EUNSUPPORTED, "too many places for tokens");
    if (qlin_status s = vector_of(slots, "slots", a.N, QLIN_DT_I64)) return s;
    if (qlin_status s = vector_of(positions, "positions", a.N, QLIN_DT_I32)) return s;
    if (qlin_status s = vector_of(rows, "rows", a.N, QLIN_DT_I32)) return s;
    if (qlin_status s = vector_of(starts, "starts", B + 1, QLIN_DT_I32)) return s;
    if (qlin_status s = vector_of(lengths, "lengths", B, QLIN_DT_I32)) return s;
    if (qlin_status s = vector_of(used, "used", 1, QLIN_DT_I32)) return s;
    // workgroups read the inputs while others write: what is written is nothing else's memory
    const Range table = range_of(block_table, "block_table", 4);
    const Range vectors[] = {range_of(context, "context", 4), range_of(added, "added", 4), range_of(free_blocks, "free_blocks", 4),
                             range_of(slots, "slots", 8), range_of(positions, "positions", 4), range_of(rows, "rows", 4),
                             range_of(starts, "starts", 4), range_of(lengths, "lengths", 4), range_of(used, "used", 4)};
    for (int i = 0; i < 9; ++i) {
        if (share_memory(vectors[i], table)) return fail(QLIN_EINVAL, "%s and block_table share memory", vectors[i].name);
        for (int j = 3; j < 9; ++j)
            if (i != j && share_memory(vectors[i], vectors[j]))
                return fail(QLIN_EINVAL, "%s and %s share memory", vectors[i].name, vectors[j].name);
    }
    a.B = (int)B;
    a.context = (const int32_t*)context->data; a.added = (const int32_t*)added->data;
    a.free_blocks = (const int32_t*)free_blocks->data; a.table = (int32_t*)block_table->data;
    a.slots = (int64_t*)slots->data; a.positions = (int32_t*)positions->data; a.rows = (int32_t*)rows->data;
    a.starts = (int32_t*)starts->data; a.lengths = (int32_t*)lengths->data; a.used = (int32_t*)used->data;
    return launched(run_paged_plan(a, (hipStream_t)stream), "paged plan");
}

qlin_status qlin_paged_attention(const qlin_tensor* q, const qlin_tensor* k_cache, const qlin_tensor* v_cache,
                                 const qlin_tensor* block_table, const qlin_tensor* lengths, float scale, int64_t window,
                                 qlin_tensor* out, void* workspace, size_t workspace_bytes, void* stream) {
    PagedAttentionArgs a;
    if (qlin_status s = has_data(q, "q", 3)) return s;
    a.dtype = q->dtype;
    if (a.dtype != QLIN_DT_F16 && a.dtype != QLIN_DT_BF16) return fail(QLIN_EUNSUPPORTED, "q dtype %d unsupported (f16, bf16)", a.dtype);
    const int64_t B = q->shape[0], H = q->shape[1], D = q->shape[2];
    if (D < 8 || D > PAGED_MAX_DIM || D % 8) return fail(QLIN_EUNSUPPORTED, "heads of %lld values (multiples of 8 up to %d)",
                                                         (long long)D, PAGED_MAX_DIM);
    if (B > INT_MOST / 2 || H > 65535) return fail(QLIN_EUNSUPPORTED, "too many rows or heads");
    if (qlin_status s = head_view(q, "q", a.dtype, B, H, D, a.q)) return s;
    if (qlin_status s = head_view(out, "out", a.dtype, B, H, D, a.out)) return s;
    const int64_t Hk = k_cache && k_cache->ndim == 4 ? k_cache->shape[2] : 0;
    a.blocks = -1;
    if (qlin_status s = cache_view(k_cache, "k_cache", a.dtype, Hk, D, a.blocks, a.page, a.kc)) return s;
    if (qlin_status s = cache_view(v_cache, "v_cache", a.dtype, Hk, D, a.blocks, a.page, a.vc)) return s;
    if (Hk < 1 || H % Hk) return fail(QLIN_EINVAL, "%lld heads over %lld kv heads", (long long)H, (long long)Hk);
    if (qlin_status s = has_data(block_table, "block_table", 2)) return s;
    if (block_table->dtype != QLIN_DT_I32) return fail(QLIN_EUNSUPPORTED, "block_table must be int32");
    if (block_table->shape[0] != B) return fail(QLIN_EINVAL, "block_table must have %lld rows", (long long)B);
    a.W = block_table->shape[1];
    if (a.W > 1 && block_table->stride[1] != 1) return fail(QLIN_EUNSUPPORTED, "block_table needs unit column stride");
    if (qlin_status s = vector_of(lengths, "lengths", B, QLIN_DT_I32)) return s;
    if (window < 0) return fail(QLIN_EINVAL, "window must not be negative");
    const int64_t strides[] = {a.q.st, a.q.sh, a.out.st, a.out.sh, a.kc.sb, a.kc.sp, a.kc.sh, a.vc.sb, a.vc.sp, a.vc.sh};
    for (int64_t v : strides)
        if (v % 8) return fail(QLIN_EUNSUPPORTED, "strides must be multiples of 8 values");
    const void* starts[] = {a.q.p, a.out.p, a.kc.p, a.vc.p};
    for (const void* p : starts)
        if ((uintptr_t)p % 16) return fail(QLIN_EUNSUPPORTED, "tensors must start 16-byte aligned");
    if (B == 0 || H == 0) return QLIN_OK;
    const size_t need = ws_paged_attention(B, H, Hk, D);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return fail(QLIN_EWORKSPACE, "workspace of %zu bytes, needs %zu (16-byte aligned)", workspace_bytes, need);
    a.B = B; a.H = (int)H; a.Hk = (int)Hk; a.D = (int)D;
    a.table = (const int32_t*)block_table->data;
    a.ldt = step(block_table, 0);
    a.lengths = (const int32_t*)lengths->data;
    a.scale = scale;
    a.window = window;
    a.ws = workspace;
    return launched(run_paged_attention(a, (hipStream_t)stream), "paged attention");
}

}  // extern "C"
