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
    PyObject* fail = nullptr;  // called with a status: raises the frontend's error
} abi;

void bind(uintptr_t norm_forward, uintptr_t norm_backward, uintptr_t norm_workspace, uintptr_t scan_forward,
          uintptr_t scan_backward, uintptr_t scan_workspace, uintptr_t scan_step, py::object fail) {
    abi.norm_forward = reinterpret_cast<decltype(abi.norm_forward)>(norm_forward);
    abi.norm_backward = reinterpret_cast<decltype(abi.norm_backward)>(norm_backward);
    abi.norm_workspace = reinterpret_cast<decltype(abi.norm_workspace)>(norm_workspace);
    abi.scan_forward = reinterpret_cast<decltype(abi.scan_forward)>(scan_forward);
    abi.scan_backward = reinterpret_cast<decltype(abi.scan_backward)>(scan_backward);
    abi.scan_workspace = reinterpret_cast<decltype(abi.scan_workspace)>(scan_workspace);
    abi.scan_step = reinterpret_cast<decltype(abi.scan_step)>(scan_step);
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
    REQUIRE(t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch(), what,
            " must be a CUDA tensor with storage of its own, not a wrapper of others");
    REQUIRE(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), what,
            " carries a forward-mode tangent: the block operators have reverse-mode gradients only");
}

// A CUDA tensor out of an argument; None where `optional`.
Tensor tensor_of(py::handle h, const char* what, bool optional = false) {
    if (optional && h.is_none()) return {};
    REQUIRE(THPVariable_Check(h.ptr()), what, " must be a CUDA tensor");
    const Tensor& t = THPVariable_Unpack(h.ptr());
    check_plain(t, what);
    REQUIRE(t.is_cuda(), what, " must be a CUDA tensor");
    return t;
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

    variable_list apply(variable_list&& grads) override {
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

    variable_list apply(variable_list&& grads) override {
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
    const Tensor state = tensor_of(hstate, "gated_scan_step: state");
    const Tensor next = hnew.is_none() ? state : tensor_of(hnew, "gated_scan_step: new_state");
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

}  // namespace

PYBIND11_MODULE(_block_ops, m) {
    m.def("bind", &bind);
    m.def("block_norm", &block_norm);
    m.def("gated_scan", &gated_scan);
    m.def("gated_scan_step", &gated_scan_step);
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
