// Eager entry points for PyTorch: the plain linears (no LoRA, no residual), the attention side and the MLP side
// called straight from Python with torch tensors.  Each builds the qlin_tensor descriptors, takes the output and the
// workspace from torch's allocator and calls the C ABI (include/qlin.h) on the current stream,
// so an eager call costs one Python -> C++ crossing instead of the descriptor packing and ctypes
// marshalling of qlin/_lib.py.  The argument rules and declines are those of qlin/ops.py,
// qlin/attention.py and qlin/mlp.py, which run every other call (LoRA, residual) through ctypes.
//
// Errors leave as QlinStatusError("<status>:<message>"); qlin/ops.py turns a status into
// NoCapableBackendError (QLIN_EUNSUPPORTED), ValueError (QLIN_EINVAL, QLIN_EWORKSPACE) or
// QlinError, exactly as for its ctypes calls.
#include <torch/extension.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>

#include <string>
#include <unordered_map>
#include <vector>

#include "qlin.h"

namespace {

struct StatusError : std::exception {
    std::string what_;
    StatusError(int status, const std::string& msg) : what_(std::to_string(status) + ":" + msg) {}
    const char* what() const noexcept override { return what_.c_str(); }
};

[[noreturn]] void fail(int status, const std::string& msg) { throw StatusError(status, msg); }

void check(qlin_status st) {
    if (st != QLIN_OK) fail(st, qlin_last_error());
}

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return QLIN_DT_F32;
        case at::kHalf: return QLIN_DT_F16;
        case at::kBFloat16: return QLIN_DT_BF16;
        case at::kChar: return QLIN_DT_I8;
        case at::kByte: return QLIN_DT_U8;
        case at::kInt: return QLIN_DT_I32;
        case at::kFloat8_e4m3fn: return QLIN_DT_E4M3;
        case at::kLong: return QLIN_DT_I64;
        default: return -1;
    }
}

bool is_float(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// A descriptor of t; dtype -1 keeps t's own.
qlin_tensor desc(const at::Tensor& t, int dtype = -1) {
    qlin_tensor d{};
    d.data = t.data_ptr();
    d.dtype = dtype >= 0 ? dtype : dtype_of(t.scalar_type());
    const int64_t nd = t.dim();
    if (nd == 0) {
        d.ndim = 1;
        d.shape[0] = 1;
        d.stride[0] = 1;
        return d;
    }
    if (nd > 4) fail(QLIN_EINVAL, "at most 4 dims");
    d.ndim = (int32_t)nd;
    for (int64_t i = 0; i < nd; ++i) {
        d.shape[i] = t.size(i);
        d.stride[i] = t.stride(i);
    }
    return d;
}

const qlin_tensor* opt(const c10::optional<at::Tensor>& t, qlin_tensor& d) {
    if (!t.has_value()) return nullptr;
    d = desc(*t);
    return &d;
}

void on_device(const char* op, const at::Tensor& t, int& dev) {
    if (!t.is_cuda())
        fail(QLIN_EUNSUPPORTED, std::string("tensor on ") + t.device().str() + ", the kernels need a ROCm device");
    const int d = t.get_device();
    if (dev < 0) dev = d;
    else if (d != dev)
        fail(QLIN_EINVAL, std::string(op) + ": tensors on different devices (cuda:" + std::to_string(dev) + ", cuda:" +
                              std::to_string(d) + ")");
}

// x as a 2-D operand [M, K] the kernels take: unit column stride, rows at least K apart, 16-byte
// aligned start (a copy otherwise); `lead` gets the leading shape.
at::Tensor as_2d(const at::Tensor& x, int64_t k, std::vector<int64_t>& lead) {
    if (x.dim() < 1 || x.size(-1) != k)
        fail(QLIN_EINVAL, "x has " + std::to_string(x.dim() ? x.size(-1) : 0) + " input features, the weight has " +
                              std::to_string(k));
    lead.assign(x.sizes().begin(), x.sizes().end() - 1);
    at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
    if (x2.size(0) > 1 && (x2.stride(1) != 1 || x2.stride(0) < k)) x2 = x2.contiguous();
    if (reinterpret_cast<uintptr_t>(x2.data_ptr()) % 16) x2 = x2.clone(at::MemoryFormat::Contiguous);
    return x2;
}

at::Tensor output(const at::Tensor& x2, int64_t n, const c10::optional<at::ScalarType>& out_dtype) {
    const at::ScalarType dt = out_dtype.value_or(x2.scalar_type());
    if (!is_float(dt)) fail(QLIN_EUNSUPPORTED, "out_dtype unsupported");
    return at::empty({x2.size(0), n}, x2.options().dtype(dt));
}

at::Tensor shaped(const at::Tensor& y, std::vector<int64_t>& lead, int64_t n) {
    if (lead.size() == 1) return y;
    lead.push_back(n);
    return y.view(lead);
}

c10::optional<at::Tensor> bias_1d(const c10::optional<at::Tensor>& bias, int64_t n) {
    if (!bias.has_value()) return bias;
    const at::Tensor& b = *bias;
    if (b.numel() != n)
        fail(QLIN_EINVAL, "bias has " + std::to_string(b.numel()) + " elements, expected " + std::to_string(n));
    if (b.dim() == 1 && b.is_contiguous()) return bias;
    return b.reshape({n}).contiguous();
}

// One workspace per (device, stream), grown on demand: calls on one stream run in order, so they
// can share it.  During HIP-graph capture every call takes its own buffer from the graph's pool
// (a cached buffer could be replaced after the capture while the graph still uses it).
struct WsKey {
    int dev;
    hipStream_t stream;
    bool operator==(const WsKey& o) const { return dev == o.dev && stream == o.stream; }
};
struct WsHash {
    size_t operator()(const WsKey& k) const { return std::hash<void*>()(k.stream) ^ (size_t)k.dev; }
};
std::unordered_map<WsKey, at::Tensor, WsHash>& ws_cache() {
    static std::unordered_map<WsKey, at::Tensor, WsHash> cache;
    return cache;
}

at::Tensor workspace_for(size_t nbytes, const at::Tensor& like, hipStream_t stream) {
    nbytes = nbytes ? nbytes : 1;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &cap) != hipSuccess) fail(QLIN_EHIP, "hipStreamIsCapturing failed");
    const auto opts = like.options().dtype(at::kByte);
    if (cap != hipStreamCaptureStatusNone) return at::empty({(int64_t)nbytes}, opts);
    const WsKey key{(int)like.get_device(), stream};
    auto& cache = ws_cache();
    auto it = cache.find(key);
    if (it == cache.end() || (size_t)it->second.numel() < nbytes) {
        at::Tensor w = at::empty({(int64_t)std::max<size_t>(nbytes, 1u << 20)}, opts);
        cache[key] = w;
        return w;
    }
    return it->second;
}

hipStream_t current_stream(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// (qk, block bytes) per ggml type id, given once by the Python package (its GGUF_TYPES table).
std::unordered_map<int64_t, std::pair<int64_t, int64_t>>& gguf_table() {
    static std::unordered_map<int64_t, std::pair<int64_t, int64_t>> t;
    return t;
}

void set_gguf_types(const std::unordered_map<int64_t, std::pair<int64_t, int64_t>>& types) { gguf_table() = types; }

at::Tensor gguf_linear(const at::Tensor& x, const at::Tensor& weight, int64_t tid, int64_t n, int64_t k,
                       const c10::optional<at::Tensor>& bias, const c10::optional<at::ScalarType>& out_dtype) {
    int dev = -1;
    on_device("gguf_linear", x, dev);
    on_device("gguf_linear", weight, dev);
    if (bias.has_value()) on_device("gguf_linear", *bias, dev);
    const auto it = gguf_table().find(tid);
    if (it == gguf_table().end()) fail(QLIN_EUNSUPPORTED, "ggml type " + std::to_string(tid) + " unsupported");
    if (weight.scalar_type() != at::kByte) fail(QLIN_EUNSUPPORTED, "weight must be the uint8 block bytes");
    if (!weight.is_contiguous()) fail(QLIN_EUNSUPPORTED, "weight bytes must be contiguous");
    const int64_t qk = it->second.first, ts = it->second.second;
    if (k % qk || weight.numel() != n * (k / qk) * ts)
        fail(QLIN_EINVAL, "weight has " + std::to_string(weight.numel()) + " bytes, expected " +
                              std::to_string(n * (k / qk) * ts) + " for (" + std::to_string(n) + ", " + std::to_string(k) +
                              ")");
    if (!is_float(x.scalar_type())) fail(QLIN_EUNSUPPORTED, "x dtype unsupported");
    std::vector<int64_t> lead;
    const at::Tensor x2 = as_2d(x, k, lead);
    at::Tensor y = output(x2, n, out_dtype);
    if (x2.size(0) == 0 || n == 0) return shaped(y, lead, n);
    const auto b = bias_1d(bias, n);
    const hipStream_t st = current_stream(x2);
    const at::Tensor ws = workspace_for(
        qlin_workspace_size(QLIN_OP_GGUF_LINEAR, x2.size(0), n, k, (int)tid, dtype_of(x2.scalar_type())), x2, st);
    qlin_tensor dx = desc(x2), dy = desc(y), db;
    check(qlin_gguf_linear(&dx, weight.data_ptr(), (int)tid, n, k, opt(b, db), &dy, ws.data_ptr(), (size_t)ws.numel(), st));
    return shaped(y, lead, n);
}

at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& qdata, const at::Tensor& scale,
                       const c10::optional<at::Tensor>& bias, const c10::optional<at::ScalarType>& out_dtype,
                       int64_t convrot_groupsize) {
    int dev = -1;
    on_device("int8_linear", x, dev);
    on_device("int8_linear", qdata, dev);
    on_device("int8_linear", scale, dev);
    if (bias.has_value()) on_device("int8_linear", *bias, dev);
    if (qdata.scalar_type() != at::kChar || qdata.dim() != 2) fail(QLIN_EUNSUPPORTED, "qdata must be a 2-D int8 tensor");
    if (!is_float(x.scalar_type())) fail(QLIN_EUNSUPPORTED, "x dtype unsupported");
    const int64_t n = qdata.size(0), k = qdata.size(1);
    std::vector<int64_t> lead;
    const at::Tensor x2 = as_2d(x, k, lead);
    at::Tensor y = output(x2, n, out_dtype);
    if (x2.size(0) == 0 || n == 0) return shaped(y, lead, n);
    const at::Tensor s = (scale.dim() == 1 || (scale.numel() != 1 && scale.numel() != n)) ? scale : scale.reshape({-1});
    const auto b = bias_1d(bias, n);
    const hipStream_t st = current_stream(x2);
    const at::Tensor ws = workspace_for(qlin_workspace_size(QLIN_OP_INT8_LINEAR, x2.size(0), n, k, (int)convrot_groupsize,
                                                            dtype_of(x2.scalar_type())),
                                        x2, st);
    qlin_tensor dx = desc(x2), dq = desc(qdata), ds = desc(s), dy = desc(y), db;
    check(qlin_int8_linear(&dx, &dq, &ds, opt(b, db), &dy, (int)convrot_groupsize, ws.data_ptr(), (size_t)ws.numel(), st));
    return shaped(y, lead, n);
}

at::Tensor f32_1d(const at::Tensor& t) {
    if (t.dim() == 1 && t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
    return t.reshape({-1}).to(at::kFloat).contiguous();
}

at::Tensor w4a8_int8_linear(const at::Tensor& x, const at::Tensor& qdata, const at::Tensor& s_rel,
                            const at::Tensor& s_channel, const c10::optional<at::Tensor>& codebook,
                            const c10::optional<at::Tensor>& bias, int64_t group_size, int64_t convrot_groupsize,
                            const c10::optional<at::ScalarType>& out_dtype) {
    int dev = -1;
    for (const at::Tensor* t : {&x, &qdata, &s_rel, &s_channel}) on_device("w4a8_int8_linear", *t, dev);
    if (codebook.has_value()) on_device("w4a8_int8_linear", *codebook, dev);
    if (bias.has_value()) on_device("w4a8_int8_linear", *bias, dev);
    if (!is_float(x.scalar_type())) fail(QLIN_EUNSUPPORTED, "x dtype unsupported");
    if (qdata.dim() != 2 || s_rel.dim() != 2) fail(QLIN_EINVAL, "qdata and s_rel must be 2-D");
    const int64_t k = s_rel.size(1) * group_size;
    const int64_t bits = k ? (qdata.size(1) * 8) / k : 0;
    if ((bits != 4 && bits != 6) || qdata.size(1) * 8 != bits * k)
        fail(QLIN_EINVAL, "qdata [" + std::to_string(qdata.size(0)) + ", " + std::to_string(qdata.size(1)) +
                              "] does not hold 4- or 6-bit codes for K=" + std::to_string(k));
    const int64_t n = qdata.size(0);
    int srdt;
    switch (s_rel.scalar_type()) {
        case at::kFloat8_e4m3fn: srdt = QLIN_DT_E4M3; break;
        case at::kHalf: case at::kBFloat16: case at::kFloat: srdt = dtype_of(s_rel.scalar_type()); break;
        default: fail(QLIN_EUNSUPPORTED, "s_rel dtype unsupported");
    }
    std::vector<int64_t> lead;
    const at::Tensor x2 = as_2d(x, k, lead);
    at::Tensor y = output(x2, n, out_dtype);
    if (x2.size(0) == 0 || n == 0) return shaped(y, lead, n);
    const at::Tensor q = (qdata.scalar_type() == at::kChar || qdata.scalar_type() == at::kByte) ? qdata : qdata.view(at::kChar);
    c10::optional<at::Tensor> cb;
    if (codebook.has_value()) cb = f32_1d(*codebook);
    const at::Tensor sch = f32_1d(s_channel);
    const auto b = bias_1d(bias, n);
    const hipStream_t st = current_stream(x2);
    const at::Tensor ws = workspace_for(qlin_workspace_size(QLIN_OP_W4A8_LINEAR, x2.size(0), n, k,
                                                            (int)(bits | group_size << 8), dtype_of(x2.scalar_type())),
                                        x2, st);
    qlin_tensor dx = desc(x2), dq = desc(q), dsr = desc(s_rel, srdt), dsc = desc(sch), dy = desc(y), dcb, db;
    check(qlin_w4a8_linear(&dx, &dq, &dsr, &dsc, opt(cb, dcb), opt(b, db), &dy, (int)bits, (int)group_size,
                           (int)convrot_groupsize, ws.data_ptr(), (size_t)ws.numel(), st));
    return shaped(y, lead, n);
}

// ---- the attention side (qlin/attention.py) ----
using OptTensor = c10::optional<at::Tensor>;

// t with unit stride along its last dimension (a copy if need be).
at::Tensor dense(const at::Tensor& t) {
    return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// [.., heads, D] as [tokens, heads, D].
at::Tensor heads_of(const char* op, const at::Tensor& t, const char* name) {
    if (t.dim() < 3)
        fail(QLIN_EINVAL, std::string(op) + ": " + name + " must be [.., heads, D], it has " + std::to_string(t.dim()) +
                              " dimensions");
    if (t.dim() == 3) return dense(t);
    int64_t tokens = 1;  // -1 has no meaning to reshape without values
    for (int64_t i = 0; i < t.dim() - 2; ++i) tokens *= t.size(i);
    return dense(t.reshape({tokens, t.size(-2), t.size(-1)}));
}

at::Tensor packed(const at::Tensor& t, c10::optional<at::ScalarType> dt = c10::nullopt) {
    const at::Tensor u = !dt || t.scalar_type() == *dt ? t : t.to(*dt);
    return u.is_contiguous() ? u : u.contiguous();
}

// An optional tensor's descriptor, with the tensor kept alive until the call has been made.
struct Opt {
    at::Tensor t;
    qlin_tensor d{};
    bool there = false;
    Opt() = default;
    explicit Opt(const at::Tensor& x) : t(x), d(desc(x)), there(true) {}
    qlin_tensor* p() { return there ? &d : nullptr; }
};

Opt vec(const OptTensor& t, c10::optional<at::ScalarType> dt = c10::nullopt) { return t ? Opt(packed(*t, dt)) : Opt(); }

void all_on_device(const char* op, std::initializer_list<const OptTensor*> ts) {
    int dev = -1;
    for (const OptTensor* t : ts)
        if (t->has_value()) on_device(op, **t, dev);
}

// An output like x [tokens, heads, D], contiguous.
at::Tensor like(const at::Tensor& x) { return at::empty(x.sizes(), x.options()); }

pybind11::object as(const Opt& o, const OptTensor& shape) {
    if (!o.there) return pybind11::none();
    return pybind11::cast(shape->dim() == 3 ? o.t : o.t.view(shape->sizes()));
}

// The forward call with or without the norms (eps < 0: without).
pybind11::tuple rope_forward(const char* op, const at::Tensor& q, const OptTensor& k, const OptTensor& wq, const OptTensor& wk,
                             bool norm, double eps, const at::Tensor& positions, const at::Tensor& inv_freq,
                             const OptTensor& axis, int64_t flags) {
    const OptTensor qt = q, pt = positions, ft = inv_freq;
    all_on_device(op, {&qt, &k, &wq, &wk, &pt, &ft, &axis});
    Opt q3(heads_of(op, q, "q")), k3, qo(like(q3.t)), ko, pos(positions), freq = vec(ft, at::kFloat), ax = vec(axis, at::kInt);
    if (k) {
        k3 = Opt(heads_of(op, *k, "k"));
        ko = Opt(like(k3.t));
    }
    const hipStream_t st = current_stream(q);
    if (norm) {
        Opt a = vec(wq), b = vec(wk);
        check(qlin_qk_norm_rope(q3.p(), k3.p(), a.p(), b.p(), (float)eps, pos.p(), freq.p(), ax.p(), (int)flags, qo.p(), ko.p(), st));
    } else {
        check(qlin_axis_rope(q3.p(), k3.p(), pos.p(), freq.p(), ax.p(), (int)flags, qo.p(), ko.p(), st));
    }
    return pybind11::make_tuple(as(qo, qt), as(ko, k));
}

pybind11::tuple axis_rope(const at::Tensor& q, const OptTensor& k, const at::Tensor& positions, const at::Tensor& inv_freq,
                          const OptTensor& axis, int64_t flags) {
    return rope_forward("axis_rope", q, k, c10::nullopt, c10::nullopt, false, 0.0, positions, inv_freq, axis, flags);
}

pybind11::tuple qk_norm_rope(const at::Tensor& q, const OptTensor& k, const OptTensor& wq, const OptTensor& wk, double eps,
                             const at::Tensor& positions, const at::Tensor& inv_freq, const OptTensor& axis, int64_t flags) {
    return rope_forward("qk_norm_rope", q, k, wq, wk, true, eps, positions, inv_freq, axis, flags);
}

at::Tensor qk_norm_rope_store(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& wq,
                              const OptTensor& wk, double eps, const at::Tensor& positions, const at::Tensor& inv_freq,
                              const OptTensor& axis, int64_t flags, const at::Tensor& slots, const at::Tensor& k_cache,
                              const at::Tensor& v_cache) {
    const char* op = "qk_norm_rope_store";
    const OptTensor qt = q, kt = k, vt = v, pt = positions, ft = inv_freq, st_ = slots, kc = k_cache, vc = v_cache;
    all_on_device(op, {&qt, &kt, &vt, &wq, &wk, &pt, &ft, &axis, &st_, &kc, &vc});
    Opt q3(heads_of(op, q, "q")), k3(heads_of(op, k, "k")), v3(heads_of(op, v, "v")), qo(like(q3.t)), pos(positions);
    Opt freq = vec(ft, at::kFloat), ax = vec(axis, at::kInt), a = vec(wq), b = vec(wk), s(slots), dk(k_cache), dv(v_cache);
    check(qlin_qk_norm_rope_store(q3.p(), k3.p(), v3.p(), a.p(), b.p(), (float)eps, pos.p(), freq.p(), ax.p(), (int)flags, s.p(),
                                  qo.p(), dk.p(), dv.p(), current_stream(q)));
    return q.dim() == 3 ? qo.t : qo.t.view(q.sizes());
}

pybind11::tuple qk_norm_rope_grad(const at::Tensor& gq, const OptTensor& gk, const at::Tensor& q, const OptTensor& k,
                                  const OptTensor& wq, const OptTensor& wk, double eps, const at::Tensor& positions,
                                  const at::Tensor& inv_freq, const OptTensor& axis, int64_t flags, bool wq_grad, bool wk_grad) {
    const char* op = "qk_norm_rope_grad";
    const OptTensor gt = gq, qt = q, pt = positions, ft = inv_freq;
    all_on_device(op, {&gt, &gk, &qt, &k, &wq, &wk, &pt, &ft, &axis});
    Opt q3(heads_of(op, q, "q")), k3, dq(like(q3.t)), dk, g3(heads_of(op, gq, "dq_out")), h3, pos(positions);
    Opt freq = vec(ft, at::kFloat), ax = vec(axis, at::kInt), a = vec(wq), b = vec(wk), da, db;
    if (k) {
        k3 = Opt(heads_of(op, *k, "k"));
        dk = Opt(like(k3.t));
    }
    if (gk) h3 = Opt(heads_of(op, *gk, "dk_out"));
    if (wq_grad && wq) da = Opt(at::empty_like(a.t));
    if (wk_grad && wk) db = Opt(at::empty_like(b.t));
    const hipStream_t st = current_stream(q);
    at::Tensor ws;
    if (da.there || db.there)
        ws = workspace_for(qlin_workspace_size(QLIN_OP_QK_NORM_ROPE_GRAD, q3.t.size(0), q3.t.size(1) + (k ? k3.t.size(1) : 0),
                                               q3.t.size(2), 0, q3.d.dtype),
                           q, st);
    check(qlin_qk_norm_rope_grad(g3.p(), h3.p(), q3.p(), k3.p(), a.p(), b.p(), (float)eps, pos.p(), freq.p(), ax.p(), (int)flags,
                                 dq.p(), dk.p(), da.p(), db.p(), ws.defined() ? ws.data_ptr() : nullptr,
                                 ws.defined() ? (size_t)ws.numel() : 0, st));
    const auto weight = [](const Opt& o) { return o.there ? pybind11::cast(o.t) : pybind11::object(pybind11::none()); };
    return pybind11::make_tuple(as(dq, qt), as(dk, k), weight(da), weight(db));
}

// n values of `base` [..], from the `first` on.
at::Tensor part_of(const at::Tensor& base, int64_t first, int64_t n) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(base.storage()), base.key_set(),
                                                            base.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(first);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
}

pybind11::tuple paged_plan(const at::Tensor& context, const at::Tensor& added, const at::Tensor& table,
                           const at::Tensor& free_blocks, int64_t page, int64_t tokens) {
    const char* op = "paged_plan";
    const OptTensor ct = context, at_ = added, tt = table, ft = free_blocks;
    all_on_device(op, {&ct, &at_, &tt, &ft});
    if (tokens < 0) fail(QLIN_EINVAL, std::string(op) + ": tokens must not be negative");
    const int64_t B = context.dim() == 1 ? context.size(0) : 0;
    // One allocation for the int32 results of the tokens and one for those of the requests, each a tensor of its own over a
    // part of it: what a caller keeps of a step (lengths) holds no memory of its tokens, and no memory has two dtypes.
    const auto fresh = [&](int64_t n, at::ScalarType dt) { return at::Tensor(at::detail::empty_cuda({n}, dt, context.device(), c10::nullopt)); };
    const at::Tensor slots = fresh(tokens, at::kLong), t2 = fresh(2 * tokens, at::kInt), r2 = fresh(2 * B + 2, at::kInt);
    const at::Tensor positions = part_of(t2, 0, tokens), rows = part_of(t2, tokens, tokens), starts = part_of(r2, 0, B + 1),
                     lengths = part_of(r2, B + 1, B), used = part_of(r2, 2 * B + 1, 1);
    qlin_tensor dc = desc(context), da = desc(added), df = desc(free_blocks), dt = desc(table), ds = desc(slots),
                dp = desc(positions), dr = desc(rows), dst = desc(starts), dl = desc(lengths), du = desc(used);
    check(qlin_paged_plan(&dc, &da, &df, page, &dt, &ds, &dp, &dr, &dst, &dl, &du, current_stream(context)));
    return pybind11::make_tuple(slots, positions, rows, starts, lengths, used);
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table,
                           const at::Tensor& lengths, double scale, int64_t window, const OptTensor& out) {
    const char* op = "paged_attention";
    const OptTensor qt = q, kt = k_cache, vt = v_cache, tt = table, lt = lengths;
    all_on_device(op, {&qt, &kt, &vt, &tt, &lt, &out});
    if (q.dim() != 3 || k_cache.dim() != 4)
        fail(QLIN_EINVAL, std::string(op) + ": q must be [rows, heads, D] and the caches [blocks, page, kv heads, D]");
    const at::Tensor q3 = dense(q), o = out ? *out : like(q);
    const hipStream_t st = current_stream(q);
    const at::Tensor ws = workspace_for(qlin_workspace_size(QLIN_OP_PAGED_ATTENTION, q.size(0), q.size(1), q.size(2),
                                                            (int)k_cache.size(2), dtype_of(q.scalar_type())),
                                        q, st);
    qlin_tensor dq = desc(q3), dk = desc(k_cache), dv = desc(v_cache), dt = desc(table), dl = desc(lengths), d_o = desc(o);
    check(qlin_paged_attention(&dq, &dk, &dv, &dt, &dl, (float)scale, window, &d_o, ws.data_ptr(), (size_t)ws.numel(), st));
    return o;
}

// ---- the MLP side (qlin/mlp.py) ----

// [.., values] as [rows, values] with unit stride along a row (a copy if need be).
at::Tensor rows_of(const char* op, const at::Tensor& t, const char* name, const at::Tensor* shape = nullptr) {
    if (t.dim() < 1) fail(QLIN_EINVAL, std::string(op) + ": " + name + " must be [.., values]");
    if (shape && t.sizes() != shape->sizes()) fail(QLIN_EINVAL, std::string(op) + ": " + name + " has another shape than the rows before it");
    if (t.dim() == 2) return dense(t);
    int64_t rows = 1;
    for (int64_t i = 0; i < t.dim() - 1; ++i) rows *= t.size(i);
    return dense(t.reshape({rows, t.size(-1)}));
}

// A new tensor, straight from the device's allocator: small calls are bound by the host.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dt, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, dt, like.device(), c10::nullopt));
}

// A new tensor shaped like x [.., values], and its rows.
struct Fresh {
    at::Tensor t;
    Opt rows;
    Fresh() = default;
    Fresh(const at::Tensor& x, const at::Tensor& x2, at::ScalarType dt) : t(fresh(x.sizes(), dt, x)), rows(x.dim() == 2 ? t : t.view(x2.sizes())) {}
};

// int8 codes like x and a scale a row.
struct Codes {
    at::Tensor q, scale;
    Opt dq, ds;
    Codes(const at::Tensor& x, const at::Tensor& x2) : q(fresh(x.sizes(), at::kChar, x)) {
        std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = 1;
        scale = fresh(sizes, at::kFloat, x);
        dq = Opt(x.dim() == 2 ? q : q.view(x2.sizes()));
        ds = Opt(x.dim() == 2 ? scale : scale.view({x2.size(0), 1}));
    }
};

pybind11::tuple add_rms_norm(const at::Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps) {
    const char* op = "add_rms_norm";
    const OptTensor xt = x;
    all_on_device(op, {&xt, &residual, &weight});
    Opt x2(rows_of(op, x, "x")), r2, w = vec(weight);
    if (residual) r2 = Opt(rows_of(op, *residual, "residual", &x));
    Fresh y(x, x2.t, x.scalar_type()), h;
    if (residual) h = Fresh(x, x2.t, residual->scalar_type());
    check(qlin_add_rms_norm(x2.p(), r2.p(), w.p(), (float)eps, y.rows.p(), h.rows.p(), current_stream(x)));
    return pybind11::make_tuple(y.t, residual ? h.t : x);
}

pybind11::tuple add_rms_norm_int8(const at::Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps, int64_t group) {
    const char* op = "add_rms_norm_int8";
    const OptTensor xt = x;
    all_on_device(op, {&xt, &residual, &weight});
    Opt x2(rows_of(op, x, "x")), r2, w = vec(weight);
    if (residual) r2 = Opt(rows_of(op, *residual, "residual", &x));
    Codes c(x, x2.t);
    Fresh h;
    if (residual) h = Fresh(x, x2.t, residual->scalar_type());
    check(qlin_add_rms_norm_int8(x2.p(), r2.p(), w.p(), (float)eps, (int)group, c.dq.p(), c.ds.p(), h.rows.p(), current_stream(x)));
    return pybind11::make_tuple(c.q, c.scale, residual ? h.t : x);
}

pybind11::tuple add_rms_norm_grad(const at::Tensor& dy, const OptTensor& dh, const at::Tensor& h, const OptTensor& weight, double eps,
                                  bool weight_grad) {
    const char* op = "add_rms_norm_grad";
    const OptTensor gt = dy, ht = h;
    all_on_device(op, {&gt, &dh, &ht, &weight});
    Opt g2(rows_of(op, dy, "dy")), h2(rows_of(op, h, "h", &dy)), d2, w = vec(weight), dw;
    if (dh) d2 = Opt(rows_of(op, *dh, "dh", &dy));
    Fresh dx(h, h2.t, h.scalar_type());
    const hipStream_t st = current_stream(dy);
    at::Tensor ws;
    if (weight_grad && weight) {
        dw = Opt(fresh(w.t.sizes(), w.t.scalar_type(), w.t));
        ws = workspace_for(qlin_workspace_size(QLIN_OP_ADD_RMS_NORM_GRAD, g2.t.size(0), 0, g2.t.size(1), 0, g2.d.dtype), dy, st);
    }
    check(qlin_add_rms_norm_grad(g2.p(), d2.p(), h2.p(), w.p(), (float)eps, dx.rows.p(), dw.p(), ws.defined() ? ws.data_ptr() : nullptr,
                                 ws.defined() ? (size_t)ws.numel() : 0, st));
    return pybind11::make_tuple(dx.t, dw.there ? pybind11::cast(dw.t) : pybind11::object(pybind11::none()));
}

at::Tensor gated_act(const at::Tensor& gate, const OptTensor& up, int64_t act) {
    const char* op = "gated_act";
    const OptTensor gt = gate;
    all_on_device(op, {&gt, &up});
    Opt g2(rows_of(op, gate, "gate")), u2;
    if (up) u2 = Opt(rows_of(op, *up, "up", &gate));
    Fresh y(gate, g2.t, gate.scalar_type());
    check(qlin_gated_act(g2.p(), u2.p(), (int)act, y.rows.p(), current_stream(gate)));
    return y.t;
}

pybind11::tuple gated_act_int8(const at::Tensor& gate, const OptTensor& up, int64_t act, int64_t group) {
    const char* op = "gated_act_int8";
    const OptTensor gt = gate;
    all_on_device(op, {&gt, &up});
    Opt g2(rows_of(op, gate, "gate")), u2;
    if (up) u2 = Opt(rows_of(op, *up, "up", &gate));
    Codes c(gate, g2.t);
    check(qlin_gated_act_int8(g2.p(), u2.p(), (int)act, (int)group, c.dq.p(), c.ds.p(), current_stream(gate)));
    return pybind11::make_tuple(c.q, c.scale);
}

pybind11::tuple gated_act_grad(const at::Tensor& dy, const at::Tensor& gate, const OptTensor& up, int64_t act) {
    const char* op = "gated_act_grad";
    const OptTensor gt = gate, dt = dy;
    all_on_device(op, {&dt, &gt, &up});
    Opt g2(rows_of(op, gate, "gate")), d2(rows_of(op, dy, "dy", &gate)), u2;
    const int64_t n = g2.t.size(1);
    if (!up) {
        Fresh d(gate, g2.t, gate.scalar_type());
        check(qlin_gated_act_grad(d2.p(), g2.p(), nullptr, (int)act, d.rows.p(), nullptr, current_stream(gate)));
        return pybind11::make_tuple(d.t, pybind11::none());
    }
    u2 = Opt(rows_of(op, *up, "up", &gate));
    std::vector<int64_t> sizes(gate.sizes().begin(), gate.sizes().end());
    sizes.back() = 2 * n;
    const at::Tensor both = fresh(sizes, gate.scalar_type(), gate), flat = both.view({g2.t.size(0), 2 * n});
    Opt a(flat.narrow(1, 0, n)), b(flat.narrow(1, n, n));
    check(qlin_gated_act_grad(d2.p(), g2.p(), u2.p(), (int)act, a.p(), b.p(), current_stream(gate)));
    return pybind11::make_tuple(both.narrow(-1, 0, n), both.narrow(-1, n, n));
}

at::Tensor w8a8_int8_linear(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& qdata, const at::Tensor& scale,
                            const OptTensor& bias, const c10::optional<at::ScalarType>& out_dtype, const OptTensor& residual,
                            const OptTensor& residual_scale) {
    const char* op = "w8a8_int8_linear";
    const OptTensor xt = x, xst = x_scale, qt = qdata, st_ = scale;
    all_on_device(op, {&xt, &xst, &qt, &st_, &bias, &residual, &residual_scale});
    Opt x2(rows_of(op, x, "x"));
    if (qdata.dim() != 2) fail(QLIN_EUNSUPPORTED, "qdata must be a 2-D int8 tensor");
    const int64_t m = x2.t.size(0), k = x2.t.size(1), n = qdata.size(0);
    const auto count = [&](const at::Tensor& t, const char* name, int64_t want) {
        if (t.numel() != want)
            fail(QLIN_EINVAL, std::string(op) + ": " + name + " has " + std::to_string(t.numel()) + " elements, expected " + std::to_string(want));
    };
    count(x_scale, "x_scale", m);
    if (scale.numel() != 1) count(scale, "scale", n);
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = n;
    Opt r, rs;
    if (residual) {
        if (residual->sizes() != at::IntArrayRef(sizes)) fail(QLIN_EINVAL, std::string(op) + ": residual has another shape than the output");
        r = Opt(rows_of(op, *residual, "residual"));
        if (r.t.size(0) > 1 && r.t.stride(0) < n) r = Opt(r.t.contiguous());
        if (residual_scale) {
            count(*residual_scale, "residual_scale", n);
            rs = Opt(residual_scale->reshape({n}).contiguous());
        }
    } else if (residual_scale) {
        fail(QLIN_EINVAL, std::string(op) + ": residual_scale given without residual");
    }
    const at::ScalarType dt = out_dtype.value_or(residual ? residual->scalar_type() : at::kBFloat16);
    if (!is_float(dt)) fail(QLIN_EUNSUPPORTED, "out_dtype unsupported");
    const at::Tensor y = fresh(sizes, dt, x);
    const at::Tensor w = dense(qdata);
    at::Tensor ws_ = f32_1d(scale);
    if (ws_.numel() != n) ws_ = ws_.expand({n}).contiguous();
    const auto b = bias_1d(bias, n);
    const auto off = [k](const at::Tensor& t) {
        const int64_t ld = t.size(0) > 1 ? t.stride(0) : 0;
        return k % 16 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 || ld % 16 || ld >= (1 << 24));
    };
    const int param = (off(x2.t) ? QLIN_W8A8_X_ROWS : 0) | (off(w) ? QLIN_W8A8_W_ROWS : 0) |
                      (n > 1 && w.stride(0) != k ? QLIN_W8A8_W_APART : 0);
    const hipStream_t st = current_stream(x);
    const size_t need = qlin_workspace_size(QLIN_OP_W8A8_LINEAR, m, n, k, param, 0);
    const at::Tensor room = need ? workspace_for(need, x, st) : at::Tensor();
    Opt xs(f32_1d(x_scale)), dw(w), ds(ws_), yo(x.dim() == 2 ? y : y.view({m, n}));
    qlin_tensor db;
    check(qlin_w8a8_linear(x2.p(), xs.p(), dw.p(), ds.p(), opt(b, db), r.p(), rs.p(), yo.p(), need ? room.data_ptr() : nullptr,
                           need ? (size_t)room.numel() : 0, st));
    return y;
}

// The cached workspace for (device of `like`, current stream), at least nbytes (for the ctypes
// calls of qlin/ops.py, so that both routes share one buffer per stream).
at::Tensor workspace(int64_t nbytes, const at::Tensor& like) {
    return workspace_for((size_t)std::max<int64_t>(nbytes, 1), like, current_stream(like));
}

void release_workspaces() { ws_cache().clear(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    static pybind11::exception<StatusError> status_error(m, "QlinStatusError", PyExc_RuntimeError);
    pybind11::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const StatusError& e) {
            status_error(e.what());
        }
    });
    m.def("set_gguf_types", &set_gguf_types);
    m.def("gguf_linear", &gguf_linear);
    m.def("int8_linear", &int8_linear);
    m.def("w4a8_int8_linear", &w4a8_int8_linear);
    m.def("axis_rope", &axis_rope);
    m.def("qk_norm_rope", &qk_norm_rope);
    m.def("qk_norm_rope_store", &qk_norm_rope_store);
    m.def("qk_norm_rope_grad", &qk_norm_rope_grad);
    m.def("paged_plan", &paged_plan);
    m.def("paged_attention", &paged_attention);
    m.def("add_rms_norm", &add_rms_norm);
    m.def("add_rms_norm_int8", &add_rms_norm_int8);
    m.def("add_rms_norm_grad", &add_rms_norm_grad);
    m.def("gated_act", &gated_act);
    m.def("gated_act_int8", &gated_act_int8);
    m.def("gated_act_grad", &gated_act_grad);
    m.def("w8a8_int8_linear", &w8a8_int8_linear);
    m.def("workspace", &workspace);
    m.def("release_workspaces", &release_workspaces);
}
