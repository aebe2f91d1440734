// host_ops.cpp -- the host side of the training-step operators in native code:
// the checks of their arguments, their output and workspace tensors, and the
// calls of libmgopt's entry points (include/mgopt_ops.h) by address.  Each
// operator is one call from Python; on the small shapes, where the host's work
// is what a call costs, torch operators and ctypes conversions around each
// launch took several times as long.

#include <torch/extension.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <tuple>
#include <vector>

#include "mgopt_ops.h"

namespace {

using at::Tensor;
using c10::optional;

struct Entries {
    decltype(&mgopt_embedding) embedding = nullptr;
    decltype(&mgopt_embedding_grad_workspace) embedding_grad_workspace = nullptr;
    decltype(&mgopt_embedding_grad) embedding_grad = nullptr;
    decltype(&mgopt_gated_act) gated_act = nullptr;
    decltype(&mgopt_gated_act_backward) gated_act_backward = nullptr;
    decltype(&mgopt_qk_norm_rope) qk_norm_rope = nullptr;
    decltype(&mgopt_qk_norm_rope_workspace) qk_norm_rope_workspace = nullptr;
    decltype(&mgopt_qk_norm_rope_backward) qk_norm_rope_backward = nullptr;
    decltype(&mgopt_policy_workspace) policy_workspace = nullptr;
    decltype(&mgopt_token_log_probs) token_log_probs = nullptr;
    decltype(&mgopt_policy_loss) policy_loss = nullptr;
    decltype(&mgopt_policy_loss_backward) policy_loss_backward = nullptr;
    decltype(&mgopt_last_error) last_error = nullptr;
    PyObject* error = nullptr;  // the package's MgoptError
} lib;

// Binds the entry points by name; the error class is kept for the process.
void bind_ops(const py::dict& addresses, const py::object& error) {
    auto take = [&](auto& fn, const char* name) {
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>());
    };
    take(lib.embedding, "mgopt_embedding");
    take(lib.embedding_grad_workspace, "mgopt_embedding_grad_workspace");
    take(lib.embedding_grad, "mgopt_embedding_grad");
    take(lib.gated_act, "mgopt_gated_act");
    take(lib.gated_act_backward, "mgopt_gated_act_backward");
    take(lib.qk_norm_rope, "mgopt_qk_norm_rope");
    take(lib.qk_norm_rope_workspace, "mgopt_qk_norm_rope_workspace");
    take(lib.qk_norm_rope_backward, "mgopt_qk_norm_rope_backward");
    take(lib.policy_workspace, "mgopt_policy_workspace");
    take(lib.token_log_probs, "mgopt_token_log_probs");
    take(lib.policy_loss, "mgopt_policy_loss");
    take(lib.policy_loss_backward, "mgopt_policy_loss_backward");
    take(lib.last_error, "mgopt_last_error");
    Py_XDECREF(lib.error);
    lib.error = error.inc_ref().ptr();
}

void check(int rc, const char* what) {
    if (rc == 0) return;
    const std::string text = std::string(what) + " failed with status " + std::to_string(rc) + ": " + lib.last_error();
    PyErr_SetString(lib.error, text.c_str());
    throw py::error_already_set();
}

int32_t code_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case c10::ScalarType::Float: return MGOPT_F32;
        case c10::ScalarType::Half: return MGOPT_F16;
        case c10::ScalarType::BFloat16: return MGOPT_BF16;
        default:
            throw py::type_error(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) +
                                 "; expected float32, float16 or bfloat16");
    }
}

[[noreturn]] void refuse(const std::string& text) { throw py::value_error(text); }

std::string shape_of(at::IntArrayRef sizes) {
    std::string s = "(";
    for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
    return s + ")";
}
std::string shape_of(const Tensor& t) { return shape_of(t.sizes()); }

// Whether two shapes of one count name the same elements in the same order:
// equal but for dimensions of one, or one of them a flat list.
bool same_order(at::IntArrayRef a, at::IntArrayRef b) {
    const auto real = [](at::IntArrayRef s) {
        std::vector<int64_t> r;
        for (const int64_t n : s)
            if (n != 1) r.push_back(n);
        return r;
    };
    if (a == b) return true;
    const std::vector<int64_t> x = real(a), y = real(b);
    return x.size() <= 1 || y.size() <= 1 || x == y;
}

// On a GPU, and on the first operand's.
void on_gpu(const Tensor& t, const char* name) {
    if (!t.is_cuda()) throw std::runtime_error(std::string(name) + " is not on a GPU; there is no CPU path");
}
void beside(const Tensor& t, const Tensor& first, const char* name) {
    on_gpu(t, name);
    if (t.device() != first.device()) refuse(std::string(name) + " is on another GPU than the operands before it");
}
void same_dtype(const Tensor& t, const Tensor& first, const char* name) {
    if (t.scalar_type() != first.scalar_type())
        throw py::type_error(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + " beside " +
                             c10::toString(first.scalar_type()));
}

// A caller's tensor that a kernel has overwritten: its version moves on, as after
// any operation in place, so that a backward pass that saved it raises instead of
// reading the new values.  Tensors of inference mode have no version.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void* as_stream(uint64_t s) { return reinterpret_cast<void*>(static_cast<uintptr_t>(s)); }

// A tensor of dimension >= 1 as rows of its last dimension, one stride apart;
// a copy where its strides are no such rows.
struct Rows {
    Tensor t;
    int64_t rows, width, stride;
};
Rows rows_of(const Tensor& x) {
    const int64_t d = x.dim(), width = x.size(d - 1);
    int64_t rows = 1, stride = width;
    bool plain = width <= 1 || x.stride(d - 1) == 1, started = false;
    int64_t next = 0;  // the stride the next dimension out has to have
    for (int64_t i = d - 2; i >= 0; --i) {
        const int64_t n = x.size(i);
        rows *= n;
        if (n == 1) continue;
        if (!started) stride = next = x.stride(i), started = true;
        plain = plain && x.stride(i) == next;
        next *= n;
    }
    if (plain) return {x, rows, width, stride};
    return {x.contiguous(), rows, width, width};
}

// ------------------------------------------------------------- embedding

Tensor ids_of(const Tensor& ids, const Tensor& first) {
    beside(ids, first, "ids");
    if (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) throw py::type_error("ids must be int64 or int32");
    return ids.contiguous();
}

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, const optional<py::object>& dtype, uint64_t stream) {
    on_gpu(weight, "weight");
    const int32_t code = code_of(weight, "weight");
    if (weight.dim() != 2 || weight.size(0) < 1 || weight.size(1) < 1)
        refuse("weight needs shape (rows, width), got " + shape_of(weight));
    if (!std::isfinite(scale)) refuse("the scale must be finite");
    const c10::DeviceGuard guard(weight.device());
    const Tensor i = ids_of(ids, weight), w = weight.contiguous();
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(weight.size(1));
    auto options = weight.options();
    if (dtype.has_value()) options = options.dtype(torch::python::detail::py_object_to_dtype(*dtype));
    Tensor out = at::empty(shape, options);
    check(lib.embedding(i.data_ptr(), static_cast<int32_t>(i.element_size()), i.numel(), w.data_ptr(), code, w.size(0),
                        w.size(1), static_cast<float>(scale), out.data_ptr(), code_of(out, "the output"), as_stream(stream)),
          "embedding");
    return out;
}

void embedding_grad(const Tensor& grad, const Tensor& ids, const Tensor& grad_out, double scale,
                    const optional<int64_t>& padding_idx, bool accumulate, uint64_t stream) {
    on_gpu(grad, "grad");
    const int32_t code = code_of(grad, "grad");
    if (grad.dim() != 2 || grad.size(0) < 1 || grad.size(1) < 1 || !grad.is_contiguous())
        refuse("grad needs shape (rows, width) and to be contiguous, got " + shape_of(grad));
    beside(grad_out, grad, "grad_out");
    const int32_t out_code = code_of(grad_out, "grad_out");
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(grad.size(1));
    if (grad_out.sizes() != at::IntArrayRef(shape))
        refuse("grad_out needs the ids' shape and grad's width, got " + shape_of(grad_out) + " for ids " + shape_of(ids) +
               " and grad " + shape_of(grad));
    if (!std::isfinite(scale)) refuse("the scale must be finite");
    int64_t padding = -1;
    if (padding_idx.has_value()) {
        padding = *padding_idx < 0 ? *padding_idx + grad.size(0) : *padding_idx;
        if (padding < 0 || padding >= grad.size(0))
            refuse("padding_idx " + std::to_string(*padding_idx) + " is outside " + std::to_string(grad.size(0)) + " rows");
    }
    const c10::DeviceGuard guard(grad.device());
    const Tensor i = ids_of(ids, grad), g = grad_out.contiguous();
    const int64_t rows = grad.size(0), width = grad.size(1);
    Tensor work = at::empty({lib.embedding_grad_workspace(i.numel(), rows, width)}, grad.options().dtype(at::kByte));
    check(lib.embedding_grad(i.data_ptr(), static_cast<int32_t>(i.element_size()), i.numel(), g.data_ptr(), out_code,
                             grad.data_ptr(), code, rows, width, static_cast<float>(scale), padding, accumulate,
                             work.data_ptr(), as_stream(stream)),
          "embedding_grad_");
    written(grad);
}

// ------------------------------------------------------------- gated_act

int32_t activation(const std::string& act) {
    if (act == "silu") return MGOPT_ACT_SILU;
    if (act == "gelu_tanh") return MGOPT_ACT_GELU_TANH;
    refuse("unknown activation '" + act + "': 'silu' or 'gelu_tanh'");
}

// (y, codes, scales); without pack, codes and scales are undefined (None).
std::tuple<Tensor, optional<Tensor>, optional<Tensor>> gated_act(const Tensor& gate, const optional<Tensor>& up,
                                                                 const std::string& act, bool pack, uint64_t stream) {
    const int32_t kind = activation(act);
    on_gpu(gate, "gate");
    const int32_t dtype = code_of(gate, "gate");
    if (gate.dim() < 1 || gate.size(-1) < 1) refuse("gate needs a last dimension of at least 1, got " + shape_of(gate));
    if (up.has_value()) {
        beside(*up, gate, "up");
        same_dtype(*up, gate, "up");
        if (up->sizes() != gate.sizes()) refuse("gate and up differ in shape: " + shape_of(gate) + ", " + shape_of(*up));
    }
    const c10::DeviceGuard guard(gate.device());
    const Rows g = rows_of(gate), u = up.has_value() ? rows_of(*up) : Rows{};
    Tensor y = at::empty(gate.sizes(), gate.options());
    optional<Tensor> codes, scales;
    if (pack) {
        const int64_t groups = (g.width + MGOPT_ACT_GROUP - 1) / MGOPT_ACT_GROUP, inputs = up.has_value() ? 2 : 1;
        codes = at::empty({inputs, g.rows, groups * MGOPT_ACT_GROUP}, gate.options().dtype(at::kChar));
        scales = at::empty({inputs, g.rows, groups}, gate.options().dtype(at::kFloat));
    }
    check(lib.gated_act(g.t.data_ptr(), g.stride, up.has_value() ? u.t.data_ptr() : nullptr,
                        up.has_value() ? u.stride : 0, dtype, g.rows, g.width, kind, y.data_ptr(),
                        pack ? codes->data_ptr<int8_t>() : nullptr, pack ? scales->data_ptr<float>() : nullptr,
                        as_stream(stream)),
          "gated_act");
    return {y, codes, scales};
}

// (d_gate, d_up or None, y or None); shape: the activation's, None where it is not known
std::tuple<Tensor, optional<Tensor>, optional<Tensor>> gated_act_backward(const Tensor& grad_out, const Tensor& codes,
                                                                          const Tensor& scales, const std::string& act,
                                                                          const optional<std::vector<int64_t>>& shape,
                                                                          bool want_y, uint64_t stream) {
    const int32_t kind = activation(act);
    on_gpu(grad_out, "grad_out");
    const int32_t dtype = code_of(grad_out, "grad_out");
    beside(codes, grad_out, "codes");
    beside(scales, grad_out, "scales");
    if (grad_out.dim() < 1 || grad_out.size(-1) < 1) refuse("grad_out needs a last dimension of at least 1");
    const c10::DeviceGuard guard(grad_out.device());
    const Rows g = rows_of(grad_out);
    const int64_t groups = (g.width + MGOPT_ACT_GROUP - 1) / MGOPT_ACT_GROUP;
    if (codes.scalar_type() != at::kChar || scales.scalar_type() != at::kFloat || !codes.is_contiguous() ||
        !scales.is_contiguous() || codes.dim() != 3 || scales.dim() != 3 || codes.size(0) < 1 || codes.size(0) > 2 ||
        codes.size(1) != g.rows || codes.size(2) != groups * MGOPT_ACT_GROUP || scales.size(0) != codes.size(0) ||
        scales.size(1) != g.rows || scales.size(2) != groups)
        refuse("the checkpoint is not one of rows like grad_out's " + shape_of(grad_out) + ": codes " + shape_of(codes) +
               ", scales " + shape_of(scales));
    if (shape.has_value()) {
        const at::IntArrayRef kept(*shape), lead = grad_out.sizes().slice(0, grad_out.dim() - 1);
        if (kept.empty() || kept.back() != g.width || !same_order(kept.slice(0, kept.size() - 1), lead))
            refuse("the checkpoint is not one of rows like grad_out's " + shape_of(grad_out) + ": the activation had shape " +
                   shape_of(kept));
    }
    const bool gated = codes.size(0) == 2;
    Tensor d_gate = at::empty(grad_out.sizes(), grad_out.options());
    optional<Tensor> d_up, y;
    if (gated) d_up = at::empty(grad_out.sizes(), grad_out.options());
    if (want_y) y = at::empty(grad_out.sizes(), grad_out.options());
    check(lib.gated_act_backward(g.t.data_ptr(), g.stride, codes.data_ptr<int8_t>(), scales.data_ptr<float>(), gated,
                                 dtype, g.rows, g.width, kind, d_gate.data_ptr(), g.width,
                                 gated ? d_up->data_ptr() : nullptr, g.width, want_y ? y->data_ptr() : nullptr,
                                 as_stream(stream)),
          "gated_act_backward");
    return {d_gate, d_up, y};
}

// ----------------------------------------------------------- qk_norm_rope

// t with contiguous last dimension, and its strides by batch, token and head.
Tensor heads_in(const Tensor& t, int64_t (&stride)[3], bool heads_first) {
    const Tensor u = t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous();
    stride[0] = u.stride(0);
    stride[1] = u.stride(heads_first ? 2 : 1);
    stride[2] = u.stride(heads_first ? 1 : 2);
    return u;
}

// The arguments both passes share, with the tensors that keep them alive.
struct Rope {
    mgopt_qk_args a{};
    Tensor q, k, wq, wk, cos, sin, positions;
};
Rope rope_args(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos, const Tensor& sin,
               const optional<Tensor>& positions, double eps, bool interleaved) {
    Rope r;
    mgopt_qk_args& a = r.a;
    on_gpu(q, "q");
    a.dtype = code_of(q, "q");
    beside(k, q, "k");
    same_dtype(k, q, "k");
    if (q.dim() != 4 || k.dim() != 4 || q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.size(3) != k.size(3) ||
        q.size(2) < 1 || k.size(2) < 1 || q.size(3) < 1)
        refuse("q and k need shapes (batch, length, heads, dim) that differ in heads only, got " + shape_of(q) + " and " +
               shape_of(k));
    const int64_t dim = q.size(3);
    if (dim > MGOPT_MAX_HEAD_DIM) refuse("heads of more than " + std::to_string(MGOPT_MAX_HEAD_DIM) + " elements");
    beside(wq, q, "q_weight");
    beside(wk, q, "k_weight");
    a.weight_dtype = code_of(wq, "q_weight");
    same_dtype(wk, wq, "k_weight");
    if (wq.dim() != 1 || wk.dim() != 1 || wq.size(0) != dim || wk.size(0) != dim)
        refuse("q_weight and k_weight need shape (" + std::to_string(dim) + ",), got " + shape_of(wq) + " and " + shape_of(wk));
    beside(cos, q, "cos");
    beside(sin, q, "sin");
    if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat) throw py::type_error("cos and sin must be float32");
    if (cos.dim() != 2 || cos.sizes() != sin.sizes() || 2 * cos.size(1) > dim)
        refuse("cos and sin need one shape (positions, rotary / 2) with rotary at most dim, got " + shape_of(cos) + " and " +
               shape_of(sin));
    if (!(eps >= 0.0)) refuse("eps must not be negative");
    a.batch = q.size(0), a.length = q.size(1), a.dim = static_cast<int32_t>(dim);
    if (positions.has_value()) {
        beside(*positions, q, "positions");
        if (positions->scalar_type() != at::kLong && positions->scalar_type() != at::kInt)
            throw py::type_error("positions must be int64 or int32");
        const bool per_batch = positions->dim() == 2;
        if (!(positions->dim() == 1 || (per_batch && (positions->size(0) == a.batch || positions->size(0) == 1))) ||
            positions->size(-1) != a.length)
            refuse("positions need shape (length,) or (batch, length), got " + shape_of(*positions) + " for " + shape_of(q));
        r.positions = positions->contiguous();
        a.positions_dev = r.positions.data_ptr();
        a.position_bytes = static_cast<int32_t>(r.positions.element_size());
        a.position_stride = per_batch && r.positions.size(0) > 1 ? a.length : 0;
    }
    r.q = heads_in(q, a.q.x_stride, false), r.k = heads_in(k, a.k.x_stride, false);
    r.wq = wq.contiguous(), r.wk = wk.contiguous(), r.cos = cos.contiguous(), r.sin = sin.contiguous();
    a.q.x_dev = r.q.data_ptr(), a.k.x_dev = r.k.data_ptr();
    a.q.weight_dev = r.wq.data_ptr(), a.k.weight_dev = r.wk.data_ptr();
    a.q.heads = static_cast<int32_t>(q.size(2)), a.k.heads = static_cast<int32_t>(k.size(2));
    a.cos_dev = r.cos.data_ptr<float>(), a.sin_dev = r.sin.data_ptr<float>();
    a.table_rows = cos.size(0), a.rotary = static_cast<int32_t>(2 * cos.size(1));
    a.interleaved = interleaved, a.eps = static_cast<float>(eps);
    return r;
}

std::vector<int64_t> heads_shape(const Tensor& t, bool heads_first) {
    return heads_first ? std::vector<int64_t>{t.size(0), t.size(2), t.size(1), t.size(3)} : t.sizes().vec();
}

py::tuple qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos,
                       const Tensor& sin, const optional<Tensor>& positions, double eps, bool interleaved, bool heads_first,
                       uint64_t stream) {
    Rope r = rope_args(q, k, wq, wk, cos, sin, positions, eps, interleaved);
    const c10::DeviceGuard guard(q.device());
    Tensor oq = at::empty(heads_shape(q, heads_first), q.options()), ok = at::empty(heads_shape(k, heads_first), k.options());
    heads_in(oq, r.a.q.out_stride, heads_first), heads_in(ok, r.a.k.out_stride, heads_first);
    r.a.q.out_dev = oq.data_ptr(), r.a.k.out_dev = ok.data_ptr();
    check(lib.qk_norm_rope(&r.a, as_stream(stream)), "qk_norm_rope");
    return py::make_tuple(oq, ok);
}

py::tuple qk_norm_rope_backward(const Tensor& gq, const Tensor& gk, const Tensor& q, const Tensor& k, const Tensor& wq,
                                const Tensor& wk, const Tensor& cos, const Tensor& sin, const optional<Tensor>& positions,
                                double eps, bool interleaved, bool heads_first, uint64_t stream) {
    Rope r = rope_args(q, k, wq, wk, cos, sin, positions, eps, interleaved);
    mgopt_qk_args& a = r.a;
    beside(gq, q, "grad_q");
    beside(gk, q, "grad_k");
    same_dtype(gq, q, "grad_q");
    same_dtype(gk, q, "grad_k");
    if (gq.sizes() != at::IntArrayRef(heads_shape(q, heads_first)) || gk.sizes() != at::IntArrayRef(heads_shape(k, heads_first)))
        refuse("grad_q and grad_k need the outputs' shapes, got " + shape_of(gq) + " and " + shape_of(gk));
    const c10::DeviceGuard guard(q.device());
    const Tensor cq = heads_in(gq, a.q.grad_stride, heads_first), ck = heads_in(gk, a.k.grad_stride, heads_first);
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    Tensor dwq = at::empty(wq.sizes(), wq.options()), dwk = at::empty(wk.sizes(), wk.options());
    Tensor work = at::empty({lib.qk_norm_rope_workspace(a.dim)}, q.options().dtype(at::kByte));
    heads_in(dq, a.q.d_x_stride, false), heads_in(dk, a.k.d_x_stride, false);
    a.q.grad_dev = cq.data_ptr(), a.k.grad_dev = ck.data_ptr();
    a.q.d_x_dev = dq.data_ptr(), a.k.d_x_dev = dk.data_ptr();
    a.q.d_weight_dev = dwq.data_ptr(), a.k.d_weight_dev = dwk.data_ptr();
    a.workspace_dev = work.data_ptr();
    check(lib.qk_norm_rope_backward(&a, as_stream(stream)), "qk_norm_rope_backward");
    return py::make_tuple(dq, dk, dwq, dwk);
}

// ------------------------------------------------------------ policy_loss

// One value per row, in the rows' order.
Tensor per_row(const Tensor& t, const Tensor& logits, int64_t rows, const char* name) {
    beside(t, logits, name);
    if (t.numel() != rows)
        refuse(std::string(name) + " has " + std::to_string(t.numel()) + " values for " + std::to_string(rows) + " rows");
    if (!same_order(t.sizes(), logits.sizes().slice(0, logits.dim() - 1)))
        refuse(std::string(name) + " has shape " + shape_of(t) + " for logits " + shape_of(logits));
    return t.contiguous();
}
Tensor float_per_row(const Tensor& t, const Tensor& logits, int64_t rows, const char* name) {
    if (t.scalar_type() != at::kFloat)
        throw py::type_error(std::string(name) + " must be float32, got " + c10::toString(t.scalar_type()));
    return per_row(t, logits, rows, name);
}

// The arguments all three entry points share, with the tensors that keep them alive.
struct Policy {
    mgopt_policy_args a{};
    Rows logits;
    Tensor targets, mask, log_probs;
};
Policy policy_args(const Tensor& logits, const Tensor& targets, const optional<Tensor>& mask, double temperature) {
    Policy p;
    on_gpu(logits, "logits");
    p.a.dtype = code_of(logits, "logits");
    if (logits.dim() < 1 || logits.size(-1) < 1) refuse("logits need a last dimension of at least 1, got " + shape_of(logits));
    if (!(temperature >= 0x1p-120 && temperature <= 0x1p120)) refuse("the temperature must lie between 2^-120 and 2^120");
    p.logits = rows_of(logits);
    const int64_t rows = p.logits.rows;
    if (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt)
        throw py::type_error("targets must be int64 or int32");
    p.targets = per_row(targets, logits, rows, "targets");
    if (mask.has_value()) {
        if (mask->scalar_type() != at::kBool && mask->scalar_type() != at::kFloat)
            throw py::type_error("mask must be bool or float32");
        p.mask = per_row(*mask, logits, rows, "mask");
        p.a.mask_kind = mask->scalar_type() == at::kBool ? MGOPT_MASK_BYTES : MGOPT_MASK_F32;
        p.a.mask_dev = p.mask.data_ptr();
    }
    p.a.logits_dev = p.logits.t.data_ptr();
    p.a.logits_stride = p.logits.stride;
    p.a.targets_dev = p.targets.data_ptr();
    p.a.target_bytes = static_cast<int32_t>(p.targets.element_size());
    p.a.rows = rows;
    p.a.vocab = p.logits.width;
    p.a.temperature = temperature;
    return p;
}

std::vector<int64_t> all_but_last(const Tensor& t) { return {t.sizes().begin(), t.sizes().end() - 1}; }

Tensor token_log_probs(const Tensor& logits, const Tensor& targets, const optional<Tensor>& mask, double temperature,
                       uint64_t stream) {
    Policy p = policy_args(logits, targets, mask, temperature);
    const c10::DeviceGuard guard(logits.device());
    Tensor out = at::empty(all_but_last(logits), logits.options().dtype(at::kFloat));
    p.a.log_probs_dev = out.data_ptr<float>();
    Tensor work;
    if (p.a.rows < 128) {  // few rows, which may be cut in slices
        work = at::empty({lib.policy_workspace(p.a.rows)}, logits.options().dtype(at::kByte));
        p.a.workspace_dev = work.data_ptr();
    }
    check(lib.token_log_probs(&p.a, as_stream(stream)), "token_log_probs");
    return out;
}

// The loss's inputs beside the logits, as one call's arguments.
struct Loss {
    Policy p;
    Tensor old_logp, advantages, ref, scale;
};
Loss loss_args(const Tensor& logits, const Tensor& targets, const Tensor& old_logp, const Tensor& advantages,
               const optional<Tensor>& ref, const optional<Tensor>& mask, double clip_low, double clip_high, double kl_coef,
               double temperature, const optional<Tensor>& scale) {
    Loss l;
    l.p = policy_args(logits, targets, mask, temperature);
    mgopt_policy_args& a = l.p.a;
    if (!(clip_low >= 0.0) || !(clip_high >= 0.0)) refuse("the clip range must not be negative");
    l.old_logp = float_per_row(old_logp, logits, a.rows, "old_logp");
    l.advantages = float_per_row(advantages, logits, a.rows, "advantages");
    a.old_logp_dev = l.old_logp.data_ptr<float>();
    a.advantages_dev = l.advantages.data_ptr<float>();
    if (ref.has_value()) {
        l.ref = float_per_row(*ref, logits, a.rows, "ref_logp");
        a.ref_logp_dev = l.ref.data_ptr<float>();
    }
    if (scale.has_value()) {
        beside(*scale, logits, "grad_scale");
        if (scale->scalar_type() != at::kFloat || scale->numel() != 1) refuse("grad_scale must be one float32 value");
        l.scale = *scale;
        a.grad_scale_dev = l.scale.data_ptr<float>();
    }
    a.clip_low = clip_low, a.clip_high = clip_high, a.kl_coef = kl_coef;
    return l;
}

// Element i of a tensor as a scalar tensor that shares its memory alone: no view
// of it to autograd, with a version of its own.  Callers change a loss in place,
// which autograd forbids on one of several views that an autograd function returns.
Tensor scalar_of(const Tensor& t, int64_t i) {
    Tensor s = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
    s.unsafeGetTensorImpl()->set_storage_offset(t.storage_offset() + i);
    s.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef{}, at::IntArrayRef{});
    return s;
}

// (loss, log_probs, policy, kl, clip_fraction, gradient or None, workspace)
py::tuple policy_loss(const Tensor& logits, const Tensor& targets, const Tensor& old_logp, const Tensor& advantages,
                      const optional<Tensor>& ref, const optional<Tensor>& mask, double clip_low, double clip_high,
                      double kl_coef, double temperature, const optional<Tensor>& scale, bool want_grad,
                      const optional<Tensor>& out, uint64_t stream) {
    Loss l = loss_args(logits, targets, old_logp, advantages, ref, mask, clip_low, clip_high, kl_coef, temperature, scale);
    mgopt_policy_args& a = l.p.a;
    const c10::DeviceGuard guard(logits.device());
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor log_probs = at::empty(all_but_last(logits), f32), results = at::empty({4}, f32);  // loss, policy, kl, clip_fraction
    Tensor work = at::empty({lib.policy_workspace(a.rows)}, logits.options().dtype(at::kByte));
    a.log_probs_dev = log_probs.data_ptr<float>();
    a.workspace_dev = work.data_ptr();
    optional<Tensor> grad;
    if (want_grad) {
        if (out.has_value()) {
            beside(*out, logits, "out");
            same_dtype(*out, logits, "out");
            if (out->sizes() != logits.sizes()) refuse("out has shape " + shape_of(*out) + ", logits " + shape_of(logits));
            const Rows r = rows_of(*out);
            if (!r.t.is_same(*out)) refuse("out needs rows that are contiguous and evenly spaced");
            if (r.rows > 1 && r.stride < r.width) refuse("out's rows overlap");
            // over the logits exactly, or beside them
            const char *x = static_cast<const char*>(a.logits_dev), *d = static_cast<const char*>(out->data_ptr());
            const auto bytes = [&](int64_t stride) { return ((a.rows - 1) * stride + a.vocab) * logits.element_size(); };
            if (a.rows > 0 && x < d + bytes(r.stride) && d < x + bytes(a.logits_stride) &&
                !(x == d && r.stride == a.logits_stride))
                refuse("out overlaps the logits and is not them");
            grad = *out;
            a.d_logits_stride = r.stride;
        } else {
            grad = at::empty(logits.sizes(), logits.options());
            a.d_logits_stride = a.vocab;
        }
        a.d_logits_dev = grad->data_ptr();
    }
    float* const r = results.data_ptr<float>();
    check(lib.policy_loss(&a, r, r + 1, as_stream(stream)), "policy_loss");
    if (want_grad && out.has_value()) written(*out);
    return py::make_tuple(scalar_of(results, 0), log_probs, scalar_of(results, 1), scalar_of(results, 2),
                          scalar_of(results, 3), grad, work);
}

Tensor policy_loss_backward(const Tensor& logits, const Tensor& targets, const Tensor& old_logp, const Tensor& advantages,
                            const optional<Tensor>& ref, const optional<Tensor>& mask, double clip_low, double clip_high,
                            double kl_coef, double temperature, const Tensor& scale, const Tensor& log_probs,
                            const Tensor& work, uint64_t stream) {
    Loss l = loss_args(logits, targets, old_logp, advantages, ref, mask, clip_low, clip_high, kl_coef, temperature, scale);
    mgopt_policy_args& a = l.p.a;
    const c10::DeviceGuard guard(logits.device());
    Tensor grad = at::empty(logits.sizes(), logits.options());
    a.log_probs_dev = log_probs.data_ptr<float>();
    a.workspace_dev = work.data_ptr();
    a.d_logits_dev = grad.data_ptr();
    a.d_logits_stride = a.vocab;
    check(lib.policy_loss_backward(&a, as_stream(stream)), "policy_loss_backward");
    return grad;
}

}  // namespace

void define_ops(py::module_& m) {
    m.def("bind_ops", &bind_ops);
    m.def("embedding", &embedding);
    m.def("embedding_grad", &embedding_grad);
    m.def("gated_act", &gated_act);
    m.def("gated_act_backward", &gated_act_backward);
    m.def("qk_norm_rope", &qk_norm_rope);
    m.def("qk_norm_rope_backward", &qk_norm_rope_backward);
    m.def("token_log_probs", &token_log_probs);
    m.def("policy_loss", &policy_loss);
    m.def("policy_loss_backward", &policy_loss_backward);
}
