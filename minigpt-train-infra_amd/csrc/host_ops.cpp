// host_ops.cpp -- the host side of the training-step operators in native code:
// the checks of their arguments, their output and workspace tensors, and the
// calls of libmgopt's entry points (include/mgopt_ops.h) by address.  Each
// operator is one call from Python; on the small shapes, where the host's work
// is what a call costs, torch operators and ctypes conversions around each
// launch took several times as long.

#include <torch/extension.h>

#include <cstdint>
#include <string>
#include <tuple>
#include <vector>

#include "mgopt_ops.h"

namespace {

using at::Tensor;
using c10::optional;

struct Entries {
    decltype(&mgopt_gated_act) gated_act = nullptr;
    decltype(&mgopt_gated_act_backward) gated_act_backward = nullptr;
    decltype(&mgopt_last_error) last_error = nullptr;
    PyObject* error = nullptr;  // the package's MgoptError
} lib;

// Binds the entry points by name; the error class is kept for the process.
void bind_ops(const py::dict& addresses, const py::object& error) {
    auto take = [&](auto& fn, const char* name) {
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>());
    };
    take(lib.gated_act, "mgopt_gated_act");
    take(lib.gated_act_backward, "mgopt_gated_act_backward");
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

std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
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

// (d_gate, d_up or None, y or None)
std::tuple<Tensor, optional<Tensor>, optional<Tensor>> gated_act_backward(const Tensor& grad_out, const Tensor& codes,
                                                                          const Tensor& scales, const std::string& act,
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

}  // namespace

void define_ops(py::module_& m) {
    m.def("bind_ops", &bind_ops);
    m.def("gated_act", &gated_act);
    m.def("gated_act_backward", &gated_act_backward);
}
