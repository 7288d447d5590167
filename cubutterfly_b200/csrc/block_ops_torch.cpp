// block_ops_torch.cpp -- the block operators on torch tensors: argument
// checks, output allocation, autograd nodes and the calls of the C entry
// points, as a CPython extension (cubutterfly_b200._block_ops).
//
// It lies between cubutterfly_b200.block_ops and the C ABI because the
// smallest calls, a token of a few requests, are bounded by the host: through
// ctypes and a Python autograd function one call cost 20 to 34 us and a
// forward with its backward 190 us, of which the kernels are 2 to 15.
// The C entry points are handed over as addresses by the frontend that loaded
// the library, so this file links against torch alone.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <mutex>
#include <string>
#include <vector>

#include <cubutterfly/cubutterfly_b200.h>

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

constexpr int64_t kChunk = 16;  // tokens per state kept for the backward of the scan

// ---- the C ABI ----------------------------------------------------------------------------------
struct Abi {
    decltype(&cubutterflyB200BlockNormForward) norm_forward = nullptr;
    decltype(&cubutterflyB200BlockNormBackward) norm_backward = nullptr;
    decltype(&cubutterflyB200BlockNormGetWorkspaceSize) norm_workspace = nullptr;
    decltype(&cubutterflyB200GatedScanForward) scan_forward = nullptr;
    decltype(&cubutterflyB200GatedScanBackward) scan_backward = nullptr;
    decltype(&cubutterflyB200GatedScanGetWorkspaceSize) scan_workspace = nullptr;
    decltype(&cubutterflyB200GatedScanStep) scan_step = nullptr;
    decltype(&cubutterflyB200GatedDeltaForward) delta_forward = nullptr;
    decltype(&cubutterflyB200GatedDeltaBackward) delta_backward = nullptr;
    decltype(&cubutterflyB200GatedDeltaGetWorkspaceSize) delta_workspace = nullptr;
    decltype(&cubutterflyB200GatedDeltaStep) delta_step = nullptr;
    decltype(&cubutterflyB200QkNormForward) qk_forward = nullptr;
    decltype(&cubutterflyB200QkNormBackward) qk_backward = nullptr;
    decltype(&cubutterflyB200QkNormGetWorkspaceSize) qk_workspace = nullptr;
    PyObject* fail = nullptr;  // called with a status: raises the frontend's error
} abi;

void bind(const std::vector<uintptr_t>& entries, py::object fail) {
    size_t at = 0;
    auto take = [&](auto& entry) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(entries.at(at++)); };
    take(abi.norm_forward);
    take(abi.norm_backward);
    take(abi.norm_workspace);
    take(abi.scan_forward);
    take(abi.scan_backward);
    take(abi.scan_workspace);
    take(abi.scan_step);
    take(abi.delta_forward);
    take(abi.delta_backward);
    take(abi.delta_workspace);
    take(abi.delta_step);
    take(abi.qk_forward);
    take(abi.qk_backward);
    take(abi.qk_workspace);
    Py_XDECREF(abi.fail);
    abi.fail = fail.release().ptr();
}

void check(cubutterflyStatus_t status) {
    if (status == CUBUTTERFLY_STATUS_SUCCESS) return;
    py::gil_scoped_acquire gil;
    PyObject* r = PyObject_CallFunction(abi.fail, "i", static_cast<int>(status));
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "block operator failed");
    throw py::error_already_set();
}

// ---- checks -------------------------------------------------------------------------------------
// Messages are put together from text alone: numbers go through
// std::to_string, since inserting one into the stream behind these macros
// crashed here.
#define REQUIRE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

std::string text(at::IntArrayRef shape) {
    std::string s = "[";
    for (size_t d = 0; d < shape.size(); ++d) s += (d ? ", " : "") + std::to_string(shape[d]);
    return s + "]";
}

int data_type(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return CUBUTTERFLY_DATA_BF16;
        case at::kHalf: return CUBUTTERFLY_DATA_FP16;
        case at::kFloat: return CUBUTTERFLY_DATA_FP32;
        default: return -1;
    }
}

// Refuses what these calls, which stand outside torch's dispatcher, would drop
// without a word: a tangent, the record of a trace, and what a subclass or a
// transform keeps elsewhere than in storage of the tensor's own (its data pointer
// may be null, which here means an argument left out).
void check_plain(const Tensor& t, const char* what) {
    const bool proxies = c10::impl::TorchDispatchModeTLS::any_modes_set() &&
                         c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
    REQUIRE(!proxies && !torch::jit::tracer::isTracing(), what,
            " is being traced: the block operators cannot be recorded, only run or captured in a CUDA graph");
    REQUIRE(t.has_storage() && !t._is_zerotensor() && !t.unsafeGetTensorImpl()->is_python_dispatch(), what,
            " must be a CUDA tensor with storage of its own, not a wrapper of others");
    REQUIRE(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), what,
            " carries a forward-mode tangent: the block operators have reverse-mode gradients only");
}

// A view that is negated lazily (the imaginary part of a conjugate, say) is taken as a copy, whose memory holds its values.
// Gradients that come to a node:
variable_list plain_gradients(variable_list&& grads) {
    for (auto& g : grads)
        if (g.defined() && g.is_neg()) g = g.resolve_neg();
    return std::move(grads);
}

// A CUDA tensor out of an argument; None where `optional`.
Tensor tensor_of(py::handle h, const char* what, bool optional = false) {
    if (optional && h.is_none()) return {};
    REQUIRE(THPVariable_Check(h.ptr()), what, " must be a CUDA tensor");
    const Tensor& t = THPVariable_Unpack(h.ptr());
    check_plain(t, what);
    REQUIRE(t.is_cuda(), what, " must be a CUDA tensor");
    return t.is_neg() ? t.resolve_neg() : t;
}
// A pool of states, which is written where it lies.
Tensor pool_of(py::handle h, const char* what) {
    REQUIRE(!THPVariable_Check(h.ptr()) || !THPVariable_Unpack(h.ptr()).is_neg(), what,
            " must not be a lazily negated view: its memory does not hold its values");
    return tensor_of(h, what);
}
void check_type(const Tensor& t, const char* what) {
    REQUIRE(data_type(t.scalar_type()) >= 0, what, " does not support dtype ", c10::toString(t.scalar_type()));
}
void check_like(const Tensor& t, const char* what, const Tensor& x, at::IntArrayRef shape) {
    REQUIRE(t.device() == x.device(), what, " is on ", t.device().str(), ", not on ", x.device().str());
    REQUIRE(t.sizes() == shape, what, " must have shape ", text(shape), ", got ", text(t.sizes()));
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

struct Rows {
    Tensor t;  // as given, or a contiguous copy
    int64_t stride = 0;
};
// `t` as rows of `dim` consecutive values one stride apart: as it is, where its
// leading dimensions merge into one of separate rows, else copied.  Rows that
// coincide or overlap (a broadcast dimension has stride zero, as the gradient of
// a sum over it has) are copied.
Rows rows_of(const Tensor& t, int64_t dim) {
    if (t.is_contiguous()) return {t, dim};
    bool fits = t.size(-1) == 1 || t.stride(-1) == 1, seen = false;
    int64_t stride = dim, expected = 0;  // of the dimensions before the last, merged from the inner one
    for (int64_t d = t.dim() - 2; d >= 0 && fits; --d) {
        if (t.size(d) == 1) continue;
        if (seen)
            fits = t.stride(d) == expected;
        else
            stride = t.stride(d);
        seen = true;
        expected = t.stride(d) * t.size(d);
    }
    if (fits && stride >= dim) return {t, stride};
    return {t.contiguous(), dim};
}

struct Tokens {
    Tensor t;
    int64_t batch = 0, token = 0;
};
// Strides of a (batch, tokens, dim) or (tokens, dim) tensor with adjacent channels.
Tokens tokens_of(const Tensor& t, int64_t dim) {
    const int64_t length = t.size(-2), batch = t.dim() == 3 ? t.size(0) : 1;
    const int64_t token = length > 1 ? t.stride(-2) : dim;
    if ((dim > 1 && t.stride(-1) != 1) || token < dim) {
        Tensor c = t.contiguous();
        return {c, batch > 1 ? c.stride(0) : 0, dim};
    }
    return {t, batch > 1 ? t.stride(0) : 0, token};
}

// Keeps errors of a second differentiation where they belong: at its use.
variable_list once(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    auto node = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate twice through ") + name + ", which is differentiable once",
        static_cast<int64_t>(grads.size()));
    for (auto& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    return (*node)(std::move(grads));
}

bool any_requires_grad(std::initializer_list<const Tensor*> list) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : list)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Tensor i of a node's inputs, saved.
SavedVariable saved(const Tensor& t) { return t.defined() ? SavedVariable(t, false) : SavedVariable(); }

// ---- block norm ---------------------------------------------------------------------------------
struct NormCall {
    int64_t dim = 0, rows = 0, gate_rows = 0;
    at::ScalarType block = at::kFloat, stream = at::kFloat;
    int flags = 0, activation = 0;
    double scale = 1.0, eps = 0.0;

    // The six inputs x, y, gate, pre, post, scale; copies are kept in `alive`.
    cubutterflyB200BlockNorm_t pack(const variable_list& in, std::vector<Tensor>& alive) const {
        cubutterflyB200BlockNorm_t a{};
        a.struct_size = sizeof(a);
        a.rows = rows;
        a.dim = dim;
        a.gate_rows = gate_rows;
        a.data_type = data_type(block);
        a.residual_type = data_type(stream);
        auto type = [&](const Tensor& t) { return t.defined() ? data_type(t.scalar_type()) : a.data_type; };
        a.pre_type = type(in[3]);
        a.post_type = type(in[4]);
        a.scale_type = type(in[5]);
        a.gate_type = type(in[2]);
        a.flags = flags;
        a.activation = activation;
        a.residual_scale = scale;
        a.epsilon = eps;
        auto place = [&](const Tensor& t, const void** p, size_t* stride) {
            if (!t.defined()) return;
            Rows r = rows_of(t, dim);
            *p = r.t.data_ptr();
            *stride = r.stride;
            alive.push_back(std::move(r.t));
        };
        place(in[0], &a.x, &a.x_row);
        place(in[1], &a.y, &a.y_row);
        place(in[2], &a.gate, &a.gate_row);
        a.pre_weight = pointer(in[3]);
        a.post_weight = pointer(in[4]);
        a.scale = pointer(in[5]);
        return a;
    }
    // residual (undefined without y), normed (undefined without the norm), and with `keep` both norms' factors
    void forward(const variable_list& in, bool keep, Tensor* residual, Tensor* normed, Tensor* rms) const {
        const Tensor& x = in[0];
        const auto options = x.options().requires_grad(false);
        if (in[1].defined()) *residual = at::empty(x.sizes(), options);
        if (flags & CUBUTTERFLY_B200_PRE_NORM) *normed = at::empty(x.sizes(), options.dtype(block));
        if (keep) *rms = at::empty({2, rows}, options.dtype(at::kFloat));
        if (rows == 0) return;
        std::vector<Tensor> alive;
        cubutterflyB200BlockNorm_t a = pack(in, alive);
        a.residual = pointer(*residual);
        a.normed = pointer(*normed);
        if (keep) {
            a.post_rms = rms->data_ptr<float>();
            a.pre_rms = a.post_rms + rows;
        }
        const c10::cuda::CUDAGuard guard(x.device());
        check(abi.norm_forward(&a, c10::cuda::getCurrentCUDAStream()));
    }
    variable_list backward(const variable_list& in, const Tensor& rms, const Tensor& d_residual,
                           const Tensor& d_normed) const {
        variable_list grads(in.size());
        const bool zero = rows == 0 || (!d_residual.defined() && !d_normed.defined());
        for (size_t i = 0; i < in.size(); ++i)
            if (in[i].defined())
                grads[i] = zero ? at::zeros(in[i].sizes(), in[i].options()) : at::empty(in[i].sizes(), in[i].options());
        if (zero) return grads;
        std::vector<Tensor> alive;
        cubutterflyB200BlockNorm_t a = pack(in, alive);
        size_t bytes = 0;
        check(abi.norm_workspace(&a, &bytes));
        const Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, in[0].options().dtype(at::kByte));
        const Rows dr = d_residual.defined() ? rows_of(d_residual, dim) : Rows{};
        const Rows dn = d_normed.defined() ? rows_of(d_normed, dim) : Rows{};
        a.post_rms = rms.data_ptr<float>();
        a.pre_rms = a.post_rms + rows;
        a.d_residual = pointer(dr.t);
        a.d_residual_row = dr.stride;
        a.d_normed = pointer(dn.t);
        a.d_normed_row = dn.stride;
        a.d_x = pointer(grads[0]);
        a.d_y = pointer(grads[1]);
        a.d_gate = pointer(grads[2]);
        a.d_pre_weight = pointer(grads[3]);
        a.d_post_weight = pointer(grads[4]);
        a.d_scale = pointer(grads[5]);
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = bytes;
        const c10::cuda::CUDAGuard guard(in[0].device());
        check(abi.norm_backward(&a, c10::cuda::getCurrentCUDAStream()));
        return grads;
    }
};

struct BlockNormBackward : Node {
    NormCall call;
    std::vector<SavedVariable> inputs;
    SavedVariable rms;

    variable_list apply(variable_list&& incoming) override {
        const variable_list grads = plain_gradients(std::move(incoming));
        variable_list in;
        Tensor r;
        {
            // another thread's backward over the same graph may release them meanwhile
            const std::lock_guard<std::mutex> lock(mutex_);
            for (const auto& v : inputs) in.push_back(v.unpack());
            r = rms.unpack();
        }
        // the outputs that exist, in order: the residual (with y), the normed rows
        const bool has_residual = in[1].defined();
        const Tensor d_residual = has_residual ? grads[0] : Tensor();
        const Tensor d_normed = call.flags & CUBUTTERFLY_B200_PRE_NORM ? grads[has_residual ? 1 : 0] : Tensor();
        variable_list out;
        {
            at::NoGradGuard no_grad;
            out = call.backward(in, r, d_residual, d_normed);
        }
        for (size_t i = 0; i < out.size(); ++i)
            if (!task_should_compute_output(i)) out[i] = Tensor();
        return once(std::move(out), "block_norm");
    }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : inputs) v.reset_data();
        rms.reset_data();
    }
    std::string name() const override { return "BlockNormBackward"; }
};

// How many gate rows a gate broadcast to x's shape has: 1, one per group of leading indices, or one per row.
int64_t gate_rows_of(const Tensor& gate, const Tensor& x, int64_t rows) {
    const auto shape = gate.sizes(), full = x.sizes();
    REQUIRE(!shape.empty() && shape.size() <= full.size() && shape.back() == full.back(), "block_norm: gate of shape ",
            text(shape), " does not broadcast over ", text(full));
    if (shape == full) return std::max<int64_t>(rows, 1);
    std::vector<int64_t> wide(full.size() - shape.size(), 1);
    wide.insert(wide.end(), shape.begin(), shape.end());
    size_t lead = 0;
    int64_t n = 1;
    while (lead + 1 < full.size() && wide[lead] == full[lead]) n *= wide[lead++];
    for (size_t d = lead; d + 1 < full.size(); ++d)
        REQUIRE(wide[d] == 1, "block_norm: gate of shape ", text(shape), " must be one per channel, or equal to x's ", text(full),
                " in its leading dimensions and 1 in the others");
    return n;
}

py::object wrap(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

py::object block_norm(py::handle hx, py::handle hy, py::handle hpre, py::handle hpost, py::handle hgate,
                      const std::string& activation, py::handle hscale, double eps, bool pre_norm, bool post_norm,
                      bool rotate, py::handle hdtype) {
    const Tensor x = tensor_of(hx, "block_norm: x"), y = tensor_of(hy, "block_norm: y", true);
    check_type(x, "block_norm: x");
    REQUIRE(x.dim() >= 1 && x.size(-1) >= 1, "block_norm requires a non-empty last dimension");
    NormCall call;
    call.dim = x.size(-1);
    call.rows = x.numel() / call.dim;
    call.stream = x.scalar_type();
    Tensor gate = tensor_of(hgate, "block_norm: gate", true), pre = tensor_of(hpre, "block_norm: pre_weight", true),
           post = tensor_of(hpost, "block_norm: post_weight", true), scale;
    if (THPVariable_Check(hscale.ptr())) {
        scale = tensor_of(hscale, "block_norm: residual_scale");
    } else {
        call.scale = hscale.cast<double>();
        REQUIRE(std::isfinite(call.scale), "block_norm: residual_scale must be finite");
    }
    const bool typed = !hdtype.is_none();
    const at::ScalarType dtype = typed ? torch::python::detail::py_object_to_dtype(py::reinterpret_borrow<py::object>(hdtype))
                                       : call.stream;
    if (!y.defined()) {
        REQUIRE(!gate.defined() && !post.defined(), "block_norm: gate and post_weight need a block output y");
        REQUIRE(!scale.defined() && call.scale == 1.0, "block_norm: residual_scale needs a block output y");
        REQUIRE(pre_norm, "block_norm: without y and pre_norm there is nothing to compute");
        call.block = dtype;
        post_norm = false;
        REQUIRE(data_type(dtype) >= 0, "block_norm does not support dtype ", c10::toString(dtype));
    } else {
        check_type(y, "block_norm: y");
        check_like(y, "block_norm: y", x, x.sizes());
        call.block = y.scalar_type();
        REQUIRE(!typed || dtype == call.block, "block_norm: dtype is y's when y is given");
    }
    REQUIRE(call.stream == call.block || call.stream == at::kFloat,
            "block_norm: the residual stream must have the block's type ", c10::toString(call.block),
            " or float32, got ", c10::toString(call.stream));
    REQUIRE((!post.defined() || post_norm) && (!pre.defined() || pre_norm),
            "block_norm: a weight of a norm that is turned off");
    REQUIRE(!rotate || pre_norm, "block_norm: rotate needs pre_norm");
    REQUIRE(std::isfinite(eps) && eps >= 0, "block_norm: eps must be finite and not negative");
    call.eps = eps;
    if (activation == "none") {
        call.activation = CUBUTTERFLY_B200_GATE_LINEAR;
    } else if (activation == "sigmoid") {
        call.activation = CUBUTTERFLY_B200_GATE_SIGMOID;
    } else {
        REQUIRE(activation == "silu", "block_norm: gate_activation must be one of none, sigmoid, silu");
        call.activation = CUBUTTERFLY_B200_GATE_SILU;
    }
    call.flags = (post_norm ? CUBUTTERFLY_B200_POST_NORM : 0) | (pre_norm ? CUBUTTERFLY_B200_PRE_NORM : 0) |
                 (rotate ? CUBUTTERFLY_B200_ROTATE : 0);
    auto vector = [&](Tensor& v, const char* what) {
        if (!v.defined()) return;
        check_like(v, what, x, {call.dim});
        REQUIRE(v.scalar_type() == call.block || v.scalar_type() == at::kFloat, what, " does not support dtype ",
                c10::toString(v.scalar_type()));
        v = v.contiguous();
    };
    vector(pre, "block_norm: pre_weight");
    vector(post, "block_norm: post_weight");
    vector(scale, "block_norm: residual_scale");
    if (gate.defined()) {
        REQUIRE(gate.device() == x.device(), "block_norm: gate is on ", gate.device().str(), ", not on ",
                x.device().str());
        REQUIRE(gate.scalar_type() == call.block || gate.scalar_type() == at::kFloat,
                "block_norm: gate does not support dtype ", c10::toString(gate.scalar_type()));
        call.gate_rows = gate_rows_of(gate, x, call.rows);
        REQUIRE(call.gate_rows != call.rows || call.rows <= 1 || gate.scalar_type() == call.block,
                "block_norm: a gate per row must have the block's type ", c10::toString(call.block));
    }
    const bool differentiable = any_requires_grad({&x, &y, &gate, &pre, &post, &scale});
    Tensor residual, normed, rms;
    variable_list in{x, y, gate, pre, post, scale};
    std::shared_ptr<BlockNormBackward> node;
    if (differentiable) {
        node = std::shared_ptr<BlockNormBackward>(new BlockNormBackward(), torch::autograd::deleteNode);
        node->call = call;
        node->set_next_edges(torch::autograd::collect_next_edges(x, y, gate, pre, post, scale));
        for (const auto& t : in) node->inputs.push_back(saved(t));
    }
    {
        at::NoGradGuard no_grad;
        call.forward(in, differentiable, &residual, &normed, &rms);
    }
    if (differentiable) {
        node->rms = saved(rms);
        if (residual.defined()) torch::autograd::set_history(residual, node);
        if (normed.defined()) torch::autograd::set_history(normed, node);
    }
    return py::make_tuple(y.defined() ? wrap(residual) : py::reinterpret_borrow<py::object>(hx), wrap(normed));
}

// ---- gated scan ---------------------------------------------------------------------------------
struct ScanCall {
    int64_t batch = 0, length = 0, dim = 0, sequences = 0;
    at::ScalarType type = at::kFloat;
    double exponent = 8.0;

    bool empty() const { return batch == 0 || length == 0; }

    // The inputs x, recurrence gate, input gate, decay, initial state; copies are kept in `alive`.
    cubutterflyB200GatedScan_t pack(const variable_list& in, const Tensor& offsets, std::vector<Tensor>& alive) const {
        cubutterflyB200GatedScan_t a{};
        a.struct_size = sizeof(a);
        a.batch = batch;
        a.length = length;
        a.dim = dim;
        a.sequences = sequences;
        a.data_type = data_type(type);
        a.exponent = exponent;
        auto place = [&](const Tensor& t, const void** p, size_t* b, size_t* s) {
            Tokens k = tokens_of(t, dim);
            *p = k.t.data_ptr();
            *b = k.batch;
            *s = k.token;
            alive.push_back(std::move(k.t));
        };
        place(in[0], &a.x, &a.x_batch, &a.x_token);
        place(in[1], &a.recurrence_gate, &a.recurrence_batch, &a.recurrence_token);
        place(in[2], &a.input_gate, &a.input_batch, &a.input_token);
        a.decay = floats(in[3]);
        a.initial_state = floats(in[4]);
        a.offsets = offsets.defined() ? offsets.data_ptr<int>() : nullptr;
        return a;
    }
    void forward(const variable_list& in, const Tensor& offsets, bool keep, Tensor* h, Tensor* final,
                 Tensor* chunk_states) const {
        const auto options = in[0].options().requires_grad(false);
        const auto wide = options.dtype(at::kFloat);
        const int64_t states = offsets.defined() ? sequences : batch;
        *h = at::empty(in[0].sizes(), options);
        if (empty()) {  // no tokens: the states stay as they are
            *final = at::zeros({states, dim}, wide);
            if (in[4].defined()) final->copy_(in[4]);
            return;
        }
        *final = at::empty({states, dim}, wide);
        if (keep) *chunk_states = at::empty({batch * ((length + kChunk - 1) / kChunk), dim}, wide);
        std::vector<Tensor> alive;
        cubutterflyB200GatedScan_t a = pack(in, offsets, alive);
        a.h = h->data_ptr();
        a.final_state = floats(*final);
        a.chunk_states = floats(*chunk_states);
        const c10::cuda::CUDAGuard guard(in[0].device());
        check(abi.scan_forward(&a, c10::cuda::getCurrentCUDAStream()));
    }
    variable_list backward(const variable_list& in, const Tensor& offsets, const Tensor& chunk_states, Tensor d_h,
                           Tensor d_final) const {
        variable_list grads(5);
        for (int i = 0; i < 5; ++i)
            if (in[i].defined()) grads[i] = at::empty(in[i].sizes(), in[i].options());
        if (empty()) {
            grads[3].zero_();
            if (in[4].defined()) {
                if (d_final.defined())
                    grads[4].copy_(d_final);
                else
                    grads[4].zero_();
            }
            return grads;
        }
        if (!d_h.defined()) d_h = at::zeros(in[0].sizes(), in[0].options());
        if (d_final.defined()) d_final = d_final.contiguous();
        std::vector<Tensor> alive;
        cubutterflyB200GatedScan_t a = pack(in, offsets, alive);
        size_t bytes = 0;
        check(abi.scan_workspace(&a, &bytes));
        const Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, in[0].options().dtype(at::kByte));
        const Tokens dh = tokens_of(d_h, dim);
        a.chunk_states = floats(chunk_states);
        a.d_h = dh.t.data_ptr();
        a.dh_batch = dh.batch;
        a.dh_token = dh.token;
        a.d_final_state = floats(d_final);
        a.d_x = pointer(grads[0]);
        a.d_recurrence_gate = pointer(grads[1]);
        a.d_input_gate = pointer(grads[2]);
        a.d_decay = floats(grads[3]);
        a.d_initial_state = floats(grads[4]);
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = bytes;
        const c10::cuda::CUDAGuard guard(in[0].device());
        check(abi.scan_backward(&a, c10::cuda::getCurrentCUDAStream()));
        return grads;
    }
};

struct GatedScanBackward : Node {
    ScanCall call;
    std::vector<SavedVariable> inputs;
    SavedVariable offsets, chunk_states;

    variable_list apply(variable_list&& incoming) override {
        const variable_list grads = plain_gradients(std::move(incoming));
        variable_list out(5);
        if (grads[0].defined() || grads[1].defined()) {
            variable_list in;
            Tensor o, states;
            {
                const std::lock_guard<std::mutex> lock(mutex_);
                for (const auto& v : inputs) in.push_back(v.unpack());
                o = offsets.unpack();
                states = chunk_states.unpack();
            }
            at::NoGradGuard no_grad;
            out = call.backward(in, o, states, grads[0], grads[1]);
            for (size_t i = 0; i < out.size(); ++i)
                if (!task_should_compute_output(i)) out[i] = Tensor();
        }
        return once(std::move(out), "gated_scan");
    }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : inputs) v.reset_data();
        offsets.reset_data();
        chunk_states.reset_data();
    }
    std::string name() const override { return "GatedScanBackward"; }
};

void check_exponent(double exponent, const char* what) {
    REQUIRE(std::isfinite(exponent) && exponent > 0, what, ": exponent must be finite and positive");
}

py::object gated_scan(py::handle hx, py::handle hr, py::handle hi, py::handle hdecay, double exponent,
                      py::handle hinitial, py::handle hoffsets) {
    const Tensor x = tensor_of(hx, "gated_scan: x");
    check_type(x, "gated_scan: x");
    Tensor offsets = tensor_of(hoffsets, "gated_scan: offsets", true);
    ScanCall call;
    if (offsets.defined()) {
        REQUIRE(offsets.scalar_type() == at::kInt, "gated_scan: offsets does not support dtype ",
                c10::toString(offsets.scalar_type()));
        REQUIRE(offsets.device() == x.device(), "gated_scan: offsets is on ", offsets.device().str(), ", not on ",
                x.device().str());
        REQUIRE(offsets.dim() == 1 && offsets.numel() >= 2, "gated_scan: offsets must hold n + 1 values, n at least 1");
        REQUIRE(x.dim() == 2 || (x.dim() == 3 && x.size(0) == 1), "gated_scan: a packed batch is (T, D) or (1, T, D)");
        offsets = offsets.contiguous();
        call.sequences = offsets.numel() - 1;
    } else {
        REQUIRE(x.dim() == 3, "gated_scan: x must be (B, S, D), or packed with offsets");
    }
    REQUIRE(x.size(-1) >= 1, "gated_scan requires a non-empty last dimension");
    call.batch = x.dim() == 3 ? x.size(0) : 1;
    call.length = x.size(-2);
    call.dim = x.size(-1);
    call.type = x.scalar_type();
    call.exponent = exponent;
    check_exponent(exponent, "gated_scan");
    const Tensor r = tensor_of(hr, "gated_scan: recurrence_gate"), i = tensor_of(hi, "gated_scan: input_gate");
    check_like(r, "gated_scan: recurrence_gate", x, x.sizes());
    check_like(i, "gated_scan: input_gate", x, x.sizes());
    REQUIRE(r.scalar_type() == call.type && i.scalar_type() == call.type, "gated_scan: the gates must have x's dtype ",
            c10::toString(call.type));
    Tensor decay = tensor_of(hdecay, "gated_scan: decay");
    check_type(decay, "gated_scan: decay");
    check_like(decay, "gated_scan: decay", x, {call.dim});
    decay = decay.to(at::kFloat).contiguous();
    Tensor initial = tensor_of(hinitial, "gated_scan: initial_state", true);
    if (initial.defined()) {
        REQUIRE(initial.scalar_type() == at::kFloat, "gated_scan: initial_state does not support dtype ",
                c10::toString(initial.scalar_type()));
        check_like(initial, "gated_scan: initial_state", x, {offsets.defined() ? call.sequences : call.batch, call.dim});
        initial = initial.contiguous();
    }
    const bool differentiable = any_requires_grad({&x, &r, &i, &decay, &initial});
    variable_list in{x, r, i, decay, initial};
    std::shared_ptr<GatedScanBackward> node;
    if (differentiable) {
        node = std::shared_ptr<GatedScanBackward>(new GatedScanBackward(), torch::autograd::deleteNode);
        node->call = call;
        node->set_next_edges(torch::autograd::collect_next_edges(x, r, i, decay, initial));
        for (const auto& t : in) node->inputs.push_back(saved(t));
        node->offsets = saved(offsets);
    }
    Tensor h, final, chunk_states;
    {
        at::NoGradGuard no_grad;
        call.forward(in, offsets, differentiable, &h, &final, &chunk_states);
    }
    if (differentiable) {
        node->chunk_states = saved(chunk_states);
        torch::autograd::set_history(h, node);
        torch::autograd::set_history(final, node);
    }
    return py::make_tuple(h, final);
}

Tensor gated_scan_step(py::handle hstate, py::handle hx, py::handle hr, py::handle hi, py::handle hdecay,
                       double exponent, py::handle hslots, py::handle hnew) {
    const Tensor x = tensor_of(hx, "gated_scan_step: x");
    check_type(x, "gated_scan_step: x");
    REQUIRE(x.dim() == 2 && x.size(1) >= 1, "gated_scan_step: x must be (B, D)");
    const int64_t batch = x.size(0), dim = x.size(1);
    const Tensor r = tensor_of(hr, "gated_scan_step: recurrence_gate"), i = tensor_of(hi, "gated_scan_step: input_gate");
    check_like(r, "gated_scan_step: recurrence_gate", x, x.sizes());
    check_like(i, "gated_scan_step: input_gate", x, x.sizes());
    REQUIRE(r.scalar_type() == x.scalar_type() && i.scalar_type() == x.scalar_type(),
            "gated_scan_step: the gates must have x's dtype ", c10::toString(x.scalar_type()));
    Tensor decay = tensor_of(hdecay, "gated_scan_step: decay");
    check_type(decay, "gated_scan_step: decay");
    check_like(decay, "gated_scan_step: decay", x, {dim});
    const Tensor state = pool_of(hstate, "gated_scan_step: state");
    const Tensor next = hnew.is_none() ? state : pool_of(hnew, "gated_scan_step: new_state");
    for (const Tensor* t : {&state, &next}) {
        REQUIRE(t->scalar_type() == at::kFloat, "gated_scan_step: a state pool does not support dtype ",
                c10::toString(t->scalar_type()));
        REQUIRE(t->device() == x.device(), "gated_scan_step: a state pool is on ", t->device().str(), ", not on ",
                x.device().str());
        REQUIRE(t->dim() == 2 && t->size(1) == dim && t->is_contiguous(),
                "gated_scan_step: a state pool must be contiguous and (slots, ", std::to_string(dim), ")");
    }
    REQUIRE(next.sizes() == state.sizes(), "gated_scan_step: new_state must have the shape of state");
    Tensor slots = tensor_of(hslots, "gated_scan_step: slots", true);
    if (slots.defined()) {
        REQUIRE(slots.scalar_type() == at::kInt, "gated_scan_step: slots does not support dtype ",
                c10::toString(slots.scalar_type()));
        check_like(slots, "gated_scan_step: slots", x, {batch});
        slots = slots.contiguous();
    } else {
        REQUIRE(state.size(0) >= batch, "gated_scan_step: ", std::to_string(batch),
                " requests without slots need a pool of as many rows");
    }
    REQUIRE(!any_requires_grad({&state, &next, &x, &r, &i, &decay}), "gated_scan_step is inference only: an input requires grad");
    check_exponent(exponent, "gated_scan_step");
    at::NoGradGuard no_grad;
    decay = decay.to(at::kFloat).contiguous();
    Tensor h = at::empty({batch, dim}, x.options().requires_grad(false));
    if (batch == 0) return h;
    const Rows kx = rows_of(x, dim), kr = rows_of(r, dim), ki = rows_of(i, dim);
    cubutterflyB200GatedScanStep_t a{};
    a.struct_size = sizeof(a);
    a.batch = batch;
    a.dim = dim;
    a.pool = state.size(0);
    a.data_type = data_type(x.scalar_type());
    a.exponent = exponent;
    a.x = kx.t.data_ptr();
    a.recurrence_gate = kr.t.data_ptr();
    a.input_gate = ki.t.data_ptr();
    a.x_row = kx.stride;
    a.recurrence_row = kr.stride;
    a.input_row = ki.stride;
    a.decay = floats(decay);
    a.state = floats(state);
    a.new_state = floats(next);
    a.slots = slots.defined() ? slots.data_ptr<int>() : nullptr;
    a.h = h.data_ptr();
    const c10::cuda::CUDAGuard guard(x.device());
    check(abi.scan_step(&a, c10::cuda::getCurrentCUDAStream()));
    // a backward that kept this pool has to see that it changed
    if (!next.is_inference()) next.unsafeGetTensorImpl()->bump_version();
    return h;
}

// ---- gated delta rule ---------------------------------------------------------------------------
// A (batch, tokens, heads, channels) tensor with adjacent channels, or a copy that has them; packed ones have one
// batch row, tensors of gates no channels, and tensors of a step no tokens.
struct Heads {
    Tensor t;
    cubutterflyB200HeadTensor_t h{};
};
Heads heads_of(const Tensor& t, bool batched, bool tokens, bool channels) {
    Heads r{t, {}};
    if (channels && t.size(-1) > 1 && t.stride(-1) != 1) r.t = t.contiguous();
    int64_t d = 0;
    r.h.batch = batched ? r.t.stride(d++) : 0;
    r.h.token = tokens ? r.t.stride(d++) : 0;
    r.h.head = r.t.stride(d);
    r.h.data = r.t.data_ptr();
    return r;
}

struct DeltaSizes {
    int64_t k_heads = 0, heads = 0, k_dim = 0, v_dim = 0;
};
// Shapes, types and devices of q, k, v and the gates, whose leading dimensions are `lead`.
DeltaSizes check_delta(const std::string& name, const Tensor& q, const Tensor& k, const Tensor& v,
                       const Tensor& log_decay, const Tensor& beta) {
    const size_t n = q.dim();
    DeltaSizes s{q.size(-2), v.size(-2), q.size(-1), v.size(-1)};
    REQUIRE(s.k_heads >= 1 && s.heads >= 1 && s.k_dim >= 1 && s.v_dim >= 1, name, " requires non-empty heads");
    REQUIRE(s.k_dim <= 128 && s.v_dim <= 128, name, ": heads of keys and of values are limited to 128 channels, got ",
            std::to_string(s.k_dim), " and ", std::to_string(s.v_dim));
    REQUIRE(s.heads % s.k_heads == 0, name, ": the ", std::to_string(s.heads), " heads of v must be a multiple of the ",
            std::to_string(s.k_heads), " of k");
    std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
    check_like(k, (name + ": k").c_str(), q, shape);
    shape[n - 2] = s.heads;
    shape[n - 1] = s.v_dim;
    check_like(v, (name + ": v").c_str(), q, shape);
    shape.pop_back();
    check_like(log_decay, (name + ": log_decay").c_str(), q, shape);
    check_like(beta, (name + ": beta").c_str(), q, shape);
    REQUIRE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), name,
            ": k and v must have q's dtype ", c10::toString(q.scalar_type()));
    for (const Tensor* t : {&log_decay, &beta})
        REQUIRE(t->scalar_type() == q.scalar_type() || t->scalar_type() == at::kFloat, name,
                ": a gate must have q's dtype ", c10::toString(q.scalar_type()), " or float32, got ",
                c10::toString(t->scalar_type()));
    return s;
}
double scale_of(py::handle h, int64_t k_dim, const char* what) {
    const double scale = h.is_none() ? 1.0 / std::sqrt(static_cast<double>(k_dim)) : h.cast<double>();
    REQUIRE(std::isfinite(scale), what, ": scale must be finite");
    return scale;
}

struct DeltaCall {
    DeltaSizes sizes;
    int64_t batch = 0, length = 0, sequences = 0;
    bool batched = false;        // the tensors have a batch dimension
    at::ScalarType type = at::kFloat;
    double scale = 1.0;

    bool empty() const { return batch == 0 || length == 0; }
    Tensor workspace(const cubutterflyB200GatedDelta_t& a, bool backward, const Tensor& like) const {
        size_t bytes = 0;
        check(abi.delta_workspace(&a, backward, &bytes));
        return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte).requires_grad(false));
    }
    // The inputs q, k, v, log_decay, beta, initial state; copies are kept in `alive`.
    cubutterflyB200GatedDelta_t pack(const variable_list& in, const Tensor& offsets, std::vector<Tensor>& alive) const {
        cubutterflyB200GatedDelta_t a{};
        a.struct_size = sizeof(a);
        a.batch = batch;
        a.length = length;
        a.k_heads = sizes.k_heads;
        a.heads = sizes.heads;
        a.k_dim = sizes.k_dim;
        a.v_dim = sizes.v_dim;
        a.sequences = sequences;
        a.data_type = data_type(type);
        a.log_decay_type = data_type(in[3].scalar_type());
        a.beta_type = data_type(in[4].scalar_type());
        a.scale = scale;
        cubutterflyB200HeadTensor_t* const places[] = {&a.q, &a.k, &a.v, &a.log_decay, &a.beta};
        for (int i = 0; i < 5; ++i) {
            Heads h = heads_of(in[i], batched, true, i < 3);
            *places[i] = h.h;
            alive.push_back(std::move(h.t));
        }
        a.initial_state = floats(in[5]);
        a.offsets = offsets.defined() ? offsets.data_ptr<int>() : nullptr;
        return a;
    }
    void forward(const variable_list& in, const Tensor& offsets, Tensor* o, Tensor* final) const {
        const auto options = in[2].options().requires_grad(false);
        const auto wide = options.dtype(at::kFloat);
        const int64_t states = offsets.defined() ? sequences : batch;
        const std::vector<int64_t> shape{states, sizes.heads, sizes.k_dim, sizes.v_dim};
        *o = at::empty(in[2].sizes(), options);
        if (empty()) {  // no tokens: the states stay as they are
            *final = at::zeros(shape, wide);
            if (in[5].defined()) final->copy_(in[5]);
            return;
        }
        const c10::cuda::CUDAGuard guard(in[0].device());
        *final = at::empty(shape, wide);
        std::vector<Tensor> alive;
        cubutterflyB200GatedDelta_t a = pack(in, offsets, alive);
        a.o = o->data_ptr();
        a.final_state = floats(*final);
        const Tensor space = workspace(a, false, in[0]);
        a.workspace = space.data_ptr();
        a.workspace_bytes = space.numel();
        check(abi.delta_forward(&a, c10::cuda::getCurrentCUDAStream()));
    }
    variable_list backward(const variable_list& in, const Tensor& offsets, Tensor d_o, Tensor d_final) const {
        variable_list grads(6);
        for (int i = 0; i < 6; ++i)
            if (in[i].defined()) grads[i] = at::empty(in[i].sizes(), in[i].options().requires_grad(false));
        if (empty()) {
            if (in[5].defined()) {
                if (d_final.defined())
                    grads[5].copy_(d_final);
                else
                    grads[5].zero_();
            }
            return grads;
        }
        const c10::cuda::CUDAGuard guard(in[0].device());
        if (!d_o.defined()) d_o = at::zeros(in[2].sizes(), in[2].options().requires_grad(false));
        if (d_final.defined()) d_final = d_final.contiguous();
        std::vector<Tensor> alive;
        cubutterflyB200GatedDelta_t a = pack(in, offsets, alive);
        const Heads h = heads_of(d_o, batched, true, true);
        a.d_o = h.h;
        a.d_final_state = floats(d_final);
        a.d_q = pointer(grads[0]);
        a.d_k = pointer(grads[1]);
        a.d_v = pointer(grads[2]);
        a.d_log_decay = pointer(grads[3]);
        a.d_beta = pointer(grads[4]);
        a.d_initial_state = floats(grads[5]);
        const Tensor space = workspace(a, true, in[0]);
        a.workspace = space.data_ptr();
        a.workspace_bytes = space.numel();
        check(abi.delta_backward(&a, c10::cuda::getCurrentCUDAStream()));
        return grads;
    }
};

struct GatedDeltaBackward : Node {
    DeltaCall call;
    std::vector<SavedVariable> inputs;
    SavedVariable offsets;

    variable_list apply(variable_list&& incoming) override {
        const variable_list grads = plain_gradients(std::move(incoming));
        variable_list out(6);
        if (grads[0].defined() || grads[1].defined()) {
            variable_list in;
            Tensor o;
            {
                const std::lock_guard<std::mutex> lock(mutex_);
                for (const auto& v : inputs) in.push_back(v.unpack());
                o = offsets.unpack();
            }
            at::NoGradGuard no_grad;
            out = call.backward(in, o, grads[0], grads[1]);
            for (size_t i = 0; i < out.size(); ++i)
                if (!task_should_compute_output(i)) out[i] = Tensor();
        }
        return once(std::move(out), "gated_delta");
    }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : inputs) v.reset_data();
        offsets.reset_data();
    }
    std::string name() const override { return "GatedDeltaBackward"; }
};

py::object gated_delta(py::handle hq, py::handle hk, py::handle hv, py::handle hdecay, py::handle hbeta,
                       py::handle hscale, py::handle hinitial, py::handle hoffsets) {
    const Tensor q = tensor_of(hq, "gated_delta: q");
    check_type(q, "gated_delta: q");
    const Tensor k = tensor_of(hk, "gated_delta: k"), v = tensor_of(hv, "gated_delta: v");
    const Tensor decay = tensor_of(hdecay, "gated_delta: log_decay"), beta = tensor_of(hbeta, "gated_delta: beta");
    Tensor offsets = tensor_of(hoffsets, "gated_delta: offsets", true);
    DeltaCall call;
    if (offsets.defined()) {
        REQUIRE(offsets.scalar_type() == at::kInt, "gated_delta: offsets does not support dtype ",
                c10::toString(offsets.scalar_type()));
        REQUIRE(offsets.device() == q.device(), "gated_delta: offsets is on ", offsets.device().str(), ", not on ",
                q.device().str());
        REQUIRE(offsets.dim() == 1 && offsets.numel() >= 2, "gated_delta: offsets must hold n + 1 values, n at least 1");
        REQUIRE(q.dim() == 3 || (q.dim() == 4 && q.size(0) == 1),
                "gated_delta: a packed batch is (T, heads, K) or (1, T, heads, K)");
        offsets = offsets.contiguous();
        call.sequences = offsets.numel() - 1;
    } else {
        REQUIRE(q.dim() == 4, "gated_delta: q must be (B, S, heads, K), or packed with offsets");
    }
    REQUIRE(v.dim() == q.dim(), "gated_delta: v must have as many dimensions as q");
    call.sizes = check_delta("gated_delta", q, k, v, decay, beta);
    call.batched = q.dim() == 4;
    call.batch = call.batched ? q.size(0) : 1;
    call.length = q.size(-3);
    call.type = q.scalar_type();
    call.scale = scale_of(hscale, call.sizes.k_dim, "gated_delta");
    Tensor initial = tensor_of(hinitial, "gated_delta: initial_state", true);
    if (initial.defined()) {
        REQUIRE(initial.scalar_type() == at::kFloat, "gated_delta: initial_state does not support dtype ",
                c10::toString(initial.scalar_type()));
        check_like(initial, "gated_delta: initial_state", q,
                   {offsets.defined() ? call.sequences : call.batch, call.sizes.heads, call.sizes.k_dim, call.sizes.v_dim});
        initial = initial.contiguous();
    }
    const bool differentiable = any_requires_grad({&q, &k, &v, &decay, &beta, &initial});
    variable_list in{q, k, v, decay, beta, initial};
    std::shared_ptr<GatedDeltaBackward> node;
    if (differentiable) {
        node = std::shared_ptr<GatedDeltaBackward>(new GatedDeltaBackward(), torch::autograd::deleteNode);
        node->call = call;
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, v, decay, beta, initial));
        for (const auto& t : in) node->inputs.push_back(saved(t));
        node->offsets = saved(offsets);
    }
    Tensor o, final;
    {
        at::NoGradGuard no_grad;
        call.forward(in, offsets, &o, &final);
    }
    if (differentiable) {
        torch::autograd::set_history(o, node);
        torch::autograd::set_history(final, node);
    }
    return py::make_tuple(o, final);
}

Tensor gated_delta_step(py::handle hstate, py::handle hq, py::handle hk, py::handle hv, py::handle hdecay,
                        py::handle hbeta, py::handle hscale, py::handle hslots, py::handle hnew) {
    const Tensor q = tensor_of(hq, "gated_delta_step: q");
    check_type(q, "gated_delta_step: q");
    const Tensor k = tensor_of(hk, "gated_delta_step: k"), v = tensor_of(hv, "gated_delta_step: v");
    const Tensor decay = tensor_of(hdecay, "gated_delta_step: log_decay"), beta = tensor_of(hbeta, "gated_delta_step: beta");
    REQUIRE(q.dim() == 3 && v.dim() == 3, "gated_delta_step: q must be (B, heads, K) and v (B, heads, V)");
    const DeltaSizes sizes = check_delta("gated_delta_step", q, k, v, decay, beta);
    const int64_t batch = q.size(0);
    const Tensor state = pool_of(hstate, "gated_delta_step: state");
    const Tensor next = hnew.is_none() ? state : pool_of(hnew, "gated_delta_step: new_state");
    for (const Tensor* t : {&state, &next}) {
        REQUIRE(t->scalar_type() == at::kFloat, "gated_delta_step: a state pool does not support dtype ",
                c10::toString(t->scalar_type()));
        REQUIRE(t->device() == q.device(), "gated_delta_step: a state pool is on ", t->device().str(), ", not on ",
                q.device().str());
        REQUIRE(t->dim() == 4 && t->size(1) == sizes.heads && t->size(2) == sizes.k_dim && t->size(3) == sizes.v_dim &&
                    t->is_contiguous(),
                "gated_delta_step: a state pool must be contiguous and (slots, ", std::to_string(sizes.heads), ", ",
                std::to_string(sizes.k_dim), ", ", std::to_string(sizes.v_dim), ")");
    }
    REQUIRE(next.sizes() == state.sizes(), "gated_delta_step: new_state must have the shape of state");
    Tensor slots = tensor_of(hslots, "gated_delta_step: slots", true);
    if (slots.defined()) {
        REQUIRE(slots.scalar_type() == at::kInt, "gated_delta_step: slots does not support dtype ",
                c10::toString(slots.scalar_type()));
        check_like(slots, "gated_delta_step: slots", q, {batch});
        slots = slots.contiguous();
    } else {
        REQUIRE(state.size(0) >= batch, "gated_delta_step: ", std::to_string(batch),
                " requests without slots need a pool of as many states");
    }
    REQUIRE(!any_requires_grad({&state, &next, &q, &k, &v, &decay, &beta}),
            "gated_delta_step is inference only: an input requires grad");
    const double scale = scale_of(hscale, sizes.k_dim, "gated_delta_step");
    at::NoGradGuard no_grad;
    Tensor o = at::empty({batch, sizes.heads, sizes.v_dim}, v.options().requires_grad(false));
    if (batch == 0) return o;
    const c10::cuda::CUDAGuard guard(q.device());
    const Heads places[] = {heads_of(q, true, false, true), heads_of(k, true, false, true), heads_of(v, true, false, true),
                            heads_of(decay, true, false, false), heads_of(beta, true, false, false)};
    cubutterflyB200GatedDeltaStep_t a{};
    a.struct_size = sizeof(a);
    a.batch = batch;
    a.k_heads = sizes.k_heads;
    a.heads = sizes.heads;
    a.k_dim = sizes.k_dim;
    a.v_dim = sizes.v_dim;
    a.pool = state.size(0);
    a.data_type = data_type(q.scalar_type());
    a.log_decay_type = data_type(decay.scalar_type());
    a.beta_type = data_type(beta.scalar_type());
    a.scale = scale;
    a.q = places[0].h;
    a.k = places[1].h;
    a.v = places[2].h;
    a.log_decay = places[3].h;
    a.beta = places[4].h;
    a.state = floats(state);
    a.new_state = floats(next);
    a.slots = slots.defined() ? slots.data_ptr<int>() : nullptr;
    a.o = o.data_ptr();
    check(abi.delta_step(&a, c10::cuda::getCurrentCUDAStream()));
    if (!next.is_inference()) next.unsafeGetTensorImpl()->bump_version();
    return o;
}

// ---- norm of queries and keys -------------------------------------------------------------------
struct QkCall {
    int64_t batch = 1, tokens = 1, q_heads = 0, k_heads = 0, dim = 0, rotary = 0, axis_count = 0, period = 0;
    at::ScalarType type = at::kFloat;
    int flags = 0;
    double eps = 0.0;

    // (..., heads, dim) as (batch, tokens, heads, dim): `tokens` is the last leading dimension, the others merge into
    // one, or the tensor is copied.
    Heads place(const Tensor& t) const {
        Heads r{t, {}};
        const int64_t n = t.dim() - 2;           // leading dimensions
        bool fits = t.size(-1) == 1 || t.stride(-1) == 1, seen = false;
        int64_t stride = 0, expected = 0;
        for (int64_t d = n - 2; d >= 0 && fits; --d) {
            if (t.size(d) == 1) continue;
            if (seen)
                fits = t.stride(d) == expected;
            else
                stride = t.stride(d);
            seen = true;
            expected = t.stride(d) * t.size(d);
        }
        if (!fits) {
            r.t = t.contiguous();
            stride = n >= 2 ? r.t.stride(n - 2) : 0;
        }
        r.h.batch = stride;
        r.h.token = n >= 1 ? r.t.stride(n - 1) : 0;
        r.h.head = r.t.stride(n);
        r.h.data = r.t.data_ptr();
        return r;
    }
    // The inputs q, k, their weights; positions, frequencies and axes; copies are kept in `alive`.
    cubutterflyB200QkNorm_t pack(const variable_list& in, const variable_list& turn, std::vector<Tensor>& alive) const {
        cubutterflyB200QkNorm_t a{};
        a.struct_size = sizeof(a);
        a.batch = batch;
        a.tokens = tokens;
        a.q_heads = q_heads;
        a.k_heads = k_heads;
        a.dim = dim;
        a.rotary = rotary;
        a.axis_count = axis_count;
        a.positions_axis = a.positions_period = period;
        a.data_type = data_type(type);
        auto weight = [&](const Tensor& t) { return t.defined() ? data_type(t.scalar_type()) : a.data_type; };
        a.q_weight_type = weight(in[2]);
        a.k_weight_type = weight(in[3]);
        a.flags = flags;
        a.epsilon = eps;
        Heads q = place(in[0]), k = place(in[1]);
        a.q = q.h;
        a.k = k.h;
        alive.push_back(std::move(q.t));
        alive.push_back(std::move(k.t));
        a.q_weight = pointer(in[2]);
        a.k_weight = pointer(in[3]);
        a.positions = pointer(turn[0]);
        a.frequencies = floats(turn[1]);
        a.axes = turn[2].defined() ? turn[2].data_ptr<int>() : nullptr;
        return a;
    }
    bool empty() const { return batch == 0 || tokens == 0; }
    void forward(const variable_list& in, const variable_list& turn, Tensor* q, Tensor* k) const {
        *q = at::empty(in[0].sizes(), in[0].options().requires_grad(false));
        *k = at::empty(in[1].sizes(), in[1].options().requires_grad(false));
        if (empty()) return;
        const c10::cuda::CUDAGuard guard(in[0].device());
        std::vector<Tensor> alive;
        cubutterflyB200QkNorm_t a = pack(in, turn, alive);
        a.q_out = q->data_ptr();
        a.k_out = k->data_ptr();
        check(abi.qk_forward(&a, c10::cuda::getCurrentCUDAStream()));
    }
    variable_list backward(const variable_list& in, const variable_list& turn, Tensor d_q, Tensor d_k) const {
        variable_list grads(4);
        for (int i = 0; i < 4; ++i)
            if (in[i].defined())
                grads[i] = empty() ? at::zeros(in[i].sizes(), in[i].options().requires_grad(false))
                                   : at::empty(in[i].sizes(), in[i].options().requires_grad(false));
        if (empty()) return grads;
        const c10::cuda::CUDAGuard guard(in[0].device());
        if (!d_q.defined()) d_q = at::zeros(in[0].sizes(), in[0].options().requires_grad(false));
        if (!d_k.defined()) d_k = at::zeros(in[1].sizes(), in[1].options().requires_grad(false));
        std::vector<Tensor> alive;
        cubutterflyB200QkNorm_t a = pack(in, turn, alive);
        const Heads hq = place(d_q), hk = place(d_k);
        a.d_q_out = hq.h;
        a.d_k_out = hk.h;
        a.d_q = pointer(grads[0]);
        a.d_k = pointer(grads[1]);
        a.d_q_weight = pointer(grads[2]);
        a.d_k_weight = pointer(grads[3]);
        size_t bytes = 0;
        check(abi.qk_workspace(&a, &bytes));
        Tensor space;
        if (bytes) {
            space = at::empty({static_cast<int64_t>(bytes)}, in[0].options().dtype(at::kByte).requires_grad(false));
            a.workspace = space.data_ptr();
            a.workspace_bytes = bytes;
        }
        check(abi.qk_backward(&a, c10::cuda::getCurrentCUDAStream()));
        return grads;
    }
};

struct QkNormBackward : Node {
    QkCall call;
    std::vector<SavedVariable> inputs, turn;

    variable_list apply(variable_list&& incoming) override {
        const variable_list grads = plain_gradients(std::move(incoming));
        variable_list out(4);
        if (grads[0].defined() || grads[1].defined()) {
            variable_list in, rotation;
            {
                const std::lock_guard<std::mutex> lock(mutex_);
                for (const auto& v : inputs) in.push_back(v.unpack());
                for (const auto& v : turn) rotation.push_back(v.unpack());
            }
            at::NoGradGuard no_grad;
            out = call.backward(in, rotation, grads[0], grads[1]);
            for (size_t i = 0; i < out.size(); ++i)
                if (!task_should_compute_output(i)) out[i] = Tensor();
        }
        return once(std::move(out), "qk_norm");
    }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : inputs) v.reset_data();
        for (auto& v : turn) v.reset_data();
    }
    std::string name() const override { return "QkNormBackward"; }
};

py::object qk_norm(py::handle hq, py::handle hk, py::handle hqw, py::handle hkw, const std::string& norm, double eps,
                   py::handle hpositions, py::handle hfrequencies, py::handle haxes, bool interleaved) {
    const Tensor q = tensor_of(hq, "qk_norm: q"), k = tensor_of(hk, "qk_norm: k");
    check_type(q, "qk_norm: q");
    REQUIRE(q.dim() >= 3, "qk_norm: q must be (..., heads, D) with at least one dimension of tokens");
    REQUIRE(k.dim() == q.dim(), "qk_norm: k must have as many dimensions as q");
    const int64_t lead = q.dim() - 2;
    QkCall call;
    call.q_heads = q.size(-2);
    call.k_heads = k.size(-2);
    call.dim = q.size(-1);
    REQUIRE(call.q_heads >= 1 && call.k_heads >= 1 && call.dim >= 1, "qk_norm requires non-empty heads");
    REQUIRE(call.dim <= 256, "qk_norm: heads are limited to 256 channels, got ", std::to_string(call.dim));
    std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
    shape[lead] = call.k_heads;
    check_like(k, "qk_norm: k", q, shape);
    REQUIRE(k.scalar_type() == q.scalar_type(), "qk_norm: k must have q's dtype ", c10::toString(q.scalar_type()));
    call.type = q.scalar_type();
    call.tokens = q.size(lead - 1);
    for (int64_t d = 0; d + 1 < lead; ++d) call.batch *= q.size(d);
    REQUIRE(norm == "rms" || norm == "l2", "qk_norm: norm must be one of rms, l2");
    REQUIRE(std::isfinite(eps) && eps >= 0, "qk_norm: eps must be finite and not negative");
    call.eps = eps;
    call.flags = (norm == "l2" ? CUBUTTERFLY_B200_QK_LENGTH : 0) | (interleaved ? CUBUTTERFLY_B200_QK_INTERLEAVED : 0);
    Tensor qw = tensor_of(hqw, "qk_norm: q_weight", true), kw = tensor_of(hkw, "qk_norm: k_weight", true);
    auto weight = [&](Tensor& w, const char* what) {
        if (!w.defined()) return;
        check_like(w, what, q, {call.dim});
        REQUIRE(w.scalar_type() == call.type || w.scalar_type() == at::kFloat, what, " does not support dtype ",
                c10::toString(w.scalar_type()));
        w = w.contiguous();
    };
    weight(qw, "qk_norm: q_weight");
    weight(kw, "qk_norm: k_weight");
    Tensor positions = tensor_of(hpositions, "qk_norm: positions", true),
           frequencies = tensor_of(hfrequencies, "qk_norm: frequencies", true), axes = tensor_of(haxes, "qk_norm: axes", true);
    REQUIRE(positions.defined() == frequencies.defined(), "qk_norm: positions and frequencies go together");
    REQUIRE(positions.defined() || !axes.defined(), "qk_norm: axes need positions");
    if (positions.defined()) {
        for (const Tensor* t : {&positions, &frequencies, &axes})
            REQUIRE(!t->defined() || t->device() == q.device(),
                    "qk_norm: positions, frequencies and axes must be on q's device ", q.device().str());
        REQUIRE(frequencies.dim() == 1 && frequencies.numel() >= 1 && 2 * frequencies.numel() <= call.dim,
                "qk_norm: frequencies must hold one value for each rotated pair of a head's ", std::to_string(call.dim),
                " channels, got ", text(frequencies.sizes()));
        REQUIRE(frequencies.scalar_type() == at::kFloat, "qk_norm: frequencies does not support dtype ",
                c10::toString(frequencies.scalar_type()));
        REQUIRE(!any_requires_grad({&frequencies}), "qk_norm has no gradient in its frequencies");
        const bool wide = positions.scalar_type() == at::kLong;
        REQUIRE(wide || positions.scalar_type() == at::kInt, "qk_norm: positions does not support dtype ",
                c10::toString(positions.scalar_type()));
        if (wide) call.flags |= CUBUTTERFLY_B200_QK_POSITIONS64;
        auto at = positions.sizes();
        call.axis_count = 1;
        if (axes.defined()) {
            REQUIRE(axes.scalar_type() == at::kInt, "qk_norm: axes does not support dtype ", c10::toString(axes.scalar_type()));
            REQUIRE(axes.sizes() == frequencies.sizes(), "qk_norm: axes must have shape ", text(frequencies.sizes()), ", got ",
                    text(axes.sizes()));
            REQUIRE(positions.dim() >= 2 && positions.size(0) >= 1, "qk_norm: with axes, positions must be (axes, tokens ...)");
            call.axis_count = positions.size(0);
            at = at.slice(1);
            axes = axes.contiguous();
        }
        const auto all = q.sizes().slice(0, lead);
        REQUIRE(!at.empty() && at.size() <= all.size() && at == all.slice(all.size() - at.size()),
                "qk_norm: positions of shape ", text(positions.sizes()), " must match the leading dimensions ", text(all),
                " of q, or the last of them");
        call.rotary = 2 * frequencies.numel();
        call.period = 1;
        for (const int64_t n : at) call.period *= n;
        positions = positions.contiguous();
        frequencies = frequencies.contiguous();
    }
    const bool differentiable = any_requires_grad({&q, &k, &qw, &kw});
    variable_list in{q, k, qw, kw}, turn{positions, frequencies, axes};
    std::shared_ptr<QkNormBackward> node;
    if (differentiable) {
        node = std::shared_ptr<QkNormBackward>(new QkNormBackward(), torch::autograd::deleteNode);
        node->call = call;
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, qw, kw));
        for (const auto& t : in) node->inputs.push_back(saved(t));
        for (const auto& t : turn) node->turn.push_back(saved(t));
    }
    Tensor oq, ok;
    {
        at::NoGradGuard no_grad;
        call.forward(in, turn, &oq, &ok);
    }
    if (differentiable) {
        torch::autograd::set_history(oq, node);
        torch::autograd::set_history(ok, node);
    }
    return py::make_tuple(oq, ok);
}

}  // namespace

PYBIND11_MODULE(_block_ops, m) {
    m.def("bind", &bind);
    m.def("block_norm", &block_norm);
    m.def("gated_scan", &gated_scan);
    m.def("gated_scan_step", &gated_scan_step);
    m.def("qk_norm", &qk_norm);
    m.def("gated_delta", &gated_delta);
    m.def("gated_delta_step", &gated_delta_step);
    // parts of the checks, for tests without a GPU
    m.def("gate_rows", &gate_rows_of);
    m.def("rows", [](const Tensor& t, int64_t dim) {
        Rows r = rows_of(t, dim);
        return std::make_tuple(r.t, r.stride);
    });
    m.def("tokens", [](const Tensor& t, int64_t dim) {
        Tokens k = tokens_of(t, dim);
        return std::make_tuple(k.t, k.batch, k.token);
    });
}
