// Host side of the calls that a training step makes many times or over many tensors (geomae_amd._host, a Python extension):
// what they do per call -- walking hundreds of parameters, argument checks, an autograd node -- costs more in Python than the
// kernels behind it take (a step of 330 parameters: 190 us in Python, 17 here, 21 on the GPU).  All device work goes through the
// C ABI of libgeomae_hip, whose entry points bind() takes by address.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <algorithm>
#include "../../include/geomae_hip.h"

namespace {

struct Entries {
    decltype(&geomae_multi_adamw_step) multi_adamw_step = nullptr;
    decltype(&geomae_group_norm_workspace_bytes) group_norm_workspace_bytes = nullptr;
    decltype(&geomae_group_norm_forward) group_norm_forward = nullptr;
    decltype(&geomae_group_norm_backward) group_norm_backward = nullptr;
    decltype(&geomae_last_error) last_error = nullptr;
} lib;

struct LibraryError : std::runtime_error { using std::runtime_error::runtime_error; };
void check(int rc, const char* what) {
    if (rc != 0) throw LibraryError(std::string(what) + " failed (" + std::to_string(rc) + "): " + lib.last_error());
}
geomaeStream_t stream_of(c10::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

int dtype_code(c10::ScalarType t) {
    return t == at::kFloat ? GEOMAE_DTYPE_F32 : t == at::kBFloat16 ? GEOMAE_DTYPE_BF16 : t == at::kHalf ? GEOMAE_DTYPE_F16 : -1;
}

// ------------------------------------------------------------------------------------------------ AdamW over many tensors
// What stands between two steps: where and how the parameters lie that the device table was made for, and the table's address.
// (A parameter may be cut or cast where it lies: its address alone does not say that the table still fits.)
struct AdamwParam {
    const void* at;
    c10::ScalarType dtype;
    c10::SmallVector<int64_t, 5> sizes, strides;
    explicit AdamwParam(const at::Tensor& p)
        : at(p.const_data_ptr()), dtype(p.scalar_type()), sizes(p.sizes().begin(), p.sizes().end()), strides(p.strides().begin(), p.strides().end()) {}
    bool is(const at::Tensor& p) const {
        return p.const_data_ptr() == at && p.scalar_type() == dtype && p.sizes() == c10::IntArrayRef(sizes) && p.strides() == c10::IntArrayRef(strides);
    }
};
struct AdamwPlan {
    std::vector<AdamwParam> params;
    std::vector<int64_t> first_chunk;
    const GeomaeAdamwTensor* table;
    const int32_t* chunks;
    void* workspace;
    int64_t workspace_bytes;
    float* norm_word;
    int state_bits;
    uint32_t seed;
    bool captured;                                                     // a captured step has these addresses
    c10::SmallVector<geomaeStream_t, 2> streams;                       // that steps were enqueued on ...
    bool new_stream;                                                   // ... the last one for the first time
    std::vector<const void*> grads;
    std::vector<int32_t> hyper_of;
    std::vector<c10::TensorImpl*> changed;
};

bool same_layout(const at::Tensor& a, const at::Tensor& b) {         // (of the same sizes)
    if (a.strides() == b.strides()) return true;
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

double number(PyObject* group, const char* key) {
    PyObject* v = PyDict_GetItemString(group, key);
    if (!v) throw py::key_error(key);
    const double d = PyFloat_AsDouble(v);
    if (PyErr_Occurred()) throw py::error_already_set();
    return d;
}

GeomaeAdamwHyper hyper_of_group(PyObject* group, c10::Device device) {
    GeomaeAdamwHyper h;
    PyObject* lr = PyDict_GetItemString(group, "lr");
    if (!lr) throw py::key_error("lr");
    h.lr = 0.0;
    h.lr_ptr = nullptr;
    if (THPVariable_Check(lr)) {
        const at::Tensor& t = THPVariable_Unpack(lr);
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.numel() == 1 && t.device() == device,
                          "MultiTensorAdamW: a tensor lr must be one float32 value on the parameters' GPU");
        h.lr_ptr = t.const_data_ptr<float>();
    } else h.lr = number(group, "lr");
    PyObject* betas = PyDict_GetItemString(group, "betas");
    py::object seq = py::reinterpret_steal<py::object>(betas ? PySequence_Fast(betas, "betas must be a pair") : nullptr);
    if (!seq) {
        if (PyErr_Occurred()) throw py::error_already_set();
        throw py::key_error("betas");
    }
    TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(seq.ptr()) == 2, "MultiTensorAdamW: betas must be a pair");
    h.beta1 = PyFloat_AsDouble(PySequence_Fast_GET_ITEM(seq.ptr(), 0));
    h.beta2 = PyFloat_AsDouble(PySequence_Fast_GET_ITEM(seq.ptr(), 1));
    if (PyErr_Occurred()) throw py::error_already_set();
    h.eps = number(group, "eps");
    h.weight_decay = number(group, "weight_decay");
    TORCH_CHECK_VALUE(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0, "MultiTensorAdamW: betas must be in [0, 1), got (",
                      h.beta1, ", ", h.beta2, ")");
    TORCH_CHECK_VALUE(h.lr >= 0.0 && h.eps >= 0.0 && h.weight_decay >= 0.0, "MultiTensorAdamW: lr, eps and weight_decay must not be negative");
    return h;
}
bool same_hyper(const GeomaeAdamwHyper& a, const GeomaeAdamwHyper& b) {
    return a.lr == b.lr && a.lr_ptr == b.lr_ptr && a.beta1 == b.beta1 && a.beta2 == b.beta2 && a.eps == b.eps && a.weight_decay == b.weight_decay;
}

// true: the step is enqueued; false: a parameter is not where or what the table says (nothing was done)
bool adamw_step(AdamwPlan& plan, py::list groups, double max_norm, double grad_scale, const c10::optional<at::Tensor>& scale_tensor,
                bool skip_nonfinite) {
    const at::NoGradGuard no_grad;
    const size_t n = plan.params.size();
    plan.changed.clear();
    plan.new_stream = false;
    std::vector<GeomaeAdamwHyper> hypers;
    std::vector<at::Tensor> copies;
    c10::optional<c10::Device> device;
    size_t i = 0;
    for (py::handle g : groups) {
        TORCH_CHECK_TYPE(PyDict_Check(g.ptr()), "MultiTensorAdamW: a parameter group is not a dict");
        PyObject* list = PyDict_GetItemString(g.ptr(), "params");
        TORCH_CHECK_TYPE(list && PyList_Check(list), "MultiTensorAdamW: a parameter group's params are not a list");
        const Py_ssize_t count = PyList_GET_SIZE(list);
        int32_t k = -1;
        for (Py_ssize_t j = 0; j < count; ++j, ++i) {
            PyObject* o = PyList_GET_ITEM(list, j);
            TORCH_CHECK_TYPE(THPVariable_Check(o), "MultiTensorAdamW: a parameter is not a tensor");
            const at::Tensor& p = THPVariable_Unpack(o);
            if (i >= n || !plan.params[i].is(p)) return false;
            if (!device) device = p.device();
            if (k < 0) {
                const GeomaeAdamwHyper h = hyper_of_group(g.ptr(), *device);
                for (k = (int32_t)hypers.size() - 1; k >= 0 && !same_hyper(hypers[k], h);) --k;
                if (k < 0) {
                    k = (int32_t)hypers.size();
                    hypers.push_back(h);
                }
            }
            plan.hyper_of[i] = k;
            plan.grads[i] = nullptr;
            const at::Tensor& grad = p.grad();
            if (!grad.defined()) continue;
            TORCH_CHECK(grad.layout() == at::kStrided, "MultiTensorAdamW: sparse gradients are not supported");
            TORCH_CHECK(grad.scalar_type() == p.scalar_type() && grad.device() == p.device() && grad.sizes() == p.sizes(),
                        "MultiTensorAdamW: a gradient (", grad.scalar_type(), ", ", grad.sizes(), ", ", grad.device(),
                        ") does not match its parameter (", p.scalar_type(), ", ", p.sizes(), ", ", p.device(), ")");
            if (same_layout(grad, p)) plan.grads[i] = grad.const_data_ptr();
            else {                                                     // a copy in the parameter's own layout
                copies.push_back(at::empty_strided(p.sizes(), p.strides(), p.options()).copy_(grad));
                plan.grads[i] = copies.back().const_data_ptr();
            }
            if (plan.grads[i] && !p.is_inference()) plan.changed.push_back(p.unsafeGetTensorImpl());
        }
    }
    if (i != n) return false;
    if (n == 0 || hypers.empty()) return true;
    const float* scale_ptr = nullptr;
    if (scale_tensor) {
        TORCH_CHECK(scale_tensor->scalar_type() == at::kFloat && scale_tensor->numel() == 1 && scale_tensor->device() == *device,
                    "MultiTensorAdamW: a tensor grad_scale must be one float32 value on the parameters' GPU");
        scale_ptr = scale_tensor->const_data_ptr<float>();
    }
    const c10::OptionalDeviceGuard guard(device);
    const geomaeStream_t stream = stream_of(*device);
    check(lib.multi_adamw_step(plan.table, plan.chunks, plan.first_chunk.data(), (int32_t)n, plan.grads.data(), plan.hyper_of.data(), hypers.data(),
                               (int32_t)hypers.size(), plan.state_bits, max_norm, grad_scale, scale_ptr, skip_nonfinite, plan.seed,
                               max_norm > 0.0 || skip_nonfinite ? plan.norm_word : nullptr, plan.workspace, plan.workspace_bytes, stream),
          "geomae_multi_adamw_step");
    plan.new_stream = std::find(plan.streams.begin(), plan.streams.end(), stream) == plan.streams.end();
    if (plan.new_stream) plan.streams.push_back(stream);
    for (c10::TensorImpl* t : plan.changed) t->bump_version();         // the parameters changed, for autograd's saved tensors too
    plan.captured = plan.captured || c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
    return true;
}

// ------------------------------------------------------------------------------------------------ group norm + activation
bool channels_last(const at::Tensor& t) {                              // t.movedim(1, -1) contiguous
    if (t.numel() == 0) return true;
    int64_t want = 1;
    if (t.size(1) != 1 && t.stride(1) != want) return false;
    want *= t.size(1);
    for (int64_t d = t.dim() - 1; d >= 0; --d) {
        if (d == 1) continue;
        if (t.size(d) != 1 && t.stride(d) != want) return false;
        want *= t.size(d);
    }
    return true;
}
at::Tensor empty_channels_last(const at::Tensor& x) {
    c10::SmallVector<int64_t, 5> strides(x.dim());
    int64_t want = x.size(1);
    strides[1] = 1;
    for (int64_t d = x.dim() - 1; d >= 0; --d) {
        if (d == 1) continue;
        strides[d] = want;
        want *= x.size(d);
    }
    return at::empty_strided(x.sizes(), strides, x.options());
}

struct GroupNormShape {
    int32_t dtype, weight_dtype, n, c, groups;
    int64_t rows;
    GroupNormShape(const at::Tensor& x, const at::Tensor& weight, int64_t g)
        : dtype(dtype_code(x.scalar_type())), weight_dtype(weight.defined() ? dtype_code(weight.scalar_type()) : 0), n((int32_t)x.size(0)),
          c((int32_t)x.size(1)), groups((int32_t)g), rows(x.numel() ? x.numel() / x.size(0) / x.size(1) : 0) {}
    at::Tensor workspace(const at::Tensor& x, bool backward, int64_t& bytes) const {
        bytes = lib.group_norm_workspace_bytes(n, rows, c, groups, dtype, backward);
        if (bytes < 0) check((int)bytes, "geomae_group_norm_workspace_bytes");
        return at::empty({bytes}, x.options().dtype(at::kByte));
    }
};
const void* data(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_data(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

std::pair<at::Tensor, at::Tensor> group_norm_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, int64_t groups,
                                                     double eps, int64_t act) {
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor y = empty_channels_last(x);
    if (x.numel() == 0) return {y, at::Tensor()};
    const GroupNormShape s(x, weight, groups);
    int64_t bytes;
    const at::Tensor ws = s.workspace(x, false, bytes);
    at::Tensor stats = at::empty({s.n, s.groups, 2}, x.options().dtype(at::kDouble));
    check(lib.group_norm_forward(data(x), s.dtype, s.n, s.rows, s.c, s.groups, data(weight), data(bias), s.weight_dtype, eps, (int32_t)act,
                                 mutable_data(y), static_cast<double*>(mutable_data(stats)), mutable_data(ws), bytes, stream_of(x.device())),
          "geomae_group_norm_forward");
    return {y, stats};
}

// The gradient of a leaf that a graph of eager work on the default stream still holds is accumulated there: while another stream
// is captured, autograd would order the two streams, which a capture does not survive (it ends the process).
bool accumulates_on_default_stream(const at::Tensor& t) {
    if (!t.defined()) return false;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : c10::nullopt;
    return stream && stream->id() == 0;
}
void check_capture(const torch::autograd::variable_list& leaves) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const at::Tensor& t : leaves)
        TORCH_CHECK(!accumulates_on_default_stream(t), "group_norm_act: a backward pass cannot be captured while a graph of eager work on the "
                    "default stream holds the gradient of the same leaf: release its outputs first, or do that work on another stream");
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& weight_,
                              const c10::optional<at::Tensor>& bias_, int64_t groups, double eps, int64_t act) {
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Tensor weight = weight_.value_or(at::Tensor()), bias = bias_.value_or(at::Tensor());
        auto [y, stats] = group_norm_forward(x, weight, bias, groups, eps, act);
        ctx->save_for_backward({x, weight, bias, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
        const bool again = at::GradMode::is_enabled();                 // create_graph: the result must not pass for a constant
        torch::autograd::variable_list out(6);
        {
            at::AutoGradMode off(false);
            const c10::OptionalDeviceGuard guard(x.device());
            check_capture({x, weight, bias});
            // (needs_input_grad counts the defined tensors among the inputs)
            at::Tensor dweight = weight.defined() && ctx->needs_input_grad(1) ? at::empty_like(weight) : at::Tensor();
            at::Tensor dbias = bias.defined() && ctx->needs_input_grad(2) ? at::empty_like(bias) : at::Tensor();
            at::Tensor dx = empty_channels_last(x), dy = grads[0];
            if (x.numel() == 0) {
                if (dweight.defined()) dweight.zero_();
                if (dbias.defined()) dbias.zero_();
            } else {
                if (!channels_last(dy)) dy = empty_channels_last(dy).copy_(dy);
                const GroupNormShape s(x, weight, ctx->saved_data["groups"].toInt());
                int64_t bytes;
                const at::Tensor ws = s.workspace(x, true, bytes);
                check(lib.group_norm_backward(data(x), data(dy), s.dtype, s.n, s.rows, s.c, s.groups, data(weight), data(bias), s.weight_dtype,
                                              (int32_t)ctx->saved_data["act"].toInt(), static_cast<const double*>(data(stats)), mutable_data(dx),
                                              mutable_data(dweight), mutable_data(dbias), mutable_data(ws), bytes, stream_of(x.device())),
                      "geomae_group_norm_backward");
            }
            out[0] = dx;
            out[1] = dweight;
            out[2] = dbias;
        }
        if (again) {
            const auto error = std::make_shared<torch::autograd::DelayedError>("group_norm_act has no second derivative", 3);
            torch::autograd::variable_list three(out.begin(), out.begin() + 3);
            for (at::Tensor& t : three)
                if (t.defined()) t = t.detach().set_requires_grad(true);
            three = (*error)(std::move(three));
            for (int i = 0; i < 3; ++i) out[i] = three[i];
        }
        return out;
    }
};

at::Tensor group_norm_act(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight_, const c10::optional<at::Tensor>& bias_,
                          double eps, const c10::optional<std::string>& activation) {
    const at::Tensor weight = weight_.value_or(at::Tensor()), bias = bias_.value_or(at::Tensor());
    // (a kernel that neither sees would give a zero derivative, and a trace that returns memory nobody wrote)
    for (const at::Tensor& t : {x, weight, bias})
        TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "group_norm_act has no forward-mode derivative");
    TORCH_CHECK(!torch::jit::tracer::isTracing(), "group_norm_act cannot be traced by torch.jit.trace");
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (geomae_amd has no CPU path)");
    TORCH_CHECK(x.dim() >= 2, "x must be [N, C, *], got ", x.sizes());
    TORCH_CHECK(dtype_code(x.scalar_type()) >= 0, "x must be float32, bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK(channels_last(x), "x must be in channels-last memory (x.movedim(1, -1) contiguous)");
    int64_t act = GEOMAE_ACT_NONE;
    if (activation) {
        act = *activation == "relu" ? GEOMAE_ACT_RELU : *activation == "silu" ? GEOMAE_ACT_SILU : *activation == "gelu" ? GEOMAE_ACT_GELU : -1;
        TORCH_CHECK(act > 0, "activation must be None, 'relu', 'silu' or 'gelu', got '", *activation, "'");
    }
    const int64_t c = x.size(1);
    TORCH_CHECK(groups >= 1 && c % groups == 0, c, " channels do not divide into ", groups, " groups");
    TORCH_CHECK(x.size(0) <= INT32_MAX && c <= INT32_MAX && groups <= INT32_MAX, "x is too large: ", x.sizes());
    for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>(weight, "weight"), {bias, "bias"}}) {
        if (!t.defined()) continue;
        TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (geomae_amd has no CPU path)");
        TORCH_CHECK(t.dim() == 1 && t.size(0) == c && t.is_contiguous() && dtype_code(t.scalar_type()) >= 0 && t.device() == x.device(), name,
                    " must be contiguous [", c, "] float32, bfloat16 or float16 on ", x.device(), ", got ", t.sizes(), " ", t.scalar_type(), " on ",
                    t.device());
    }
    TORCH_CHECK(weight.defined() || !bias.defined(), "a bias needs a weight");
    TORCH_CHECK(!bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight and bias must have one dtype, got ", weight.scalar_type(),
                " and ", bias.scalar_type());
    TORCH_CHECK(eps >= 0.0, "eps must not be negative, got ", eps);
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad())))
        return GroupNormAct::apply(x, weight_, bias_, groups, eps, act);
    at::AutoDispatchBelowADInplaceOrView below;
    return group_norm_forward(x, weight, bias, groups, eps, act).first;
}

template <typename F> void take(const py::dict& d, const char* name, F& f) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    static py::object library_error;
    m.def("bind", [](py::dict entries, py::object error) {
        take(entries, "geomae_multi_adamw_step", lib.multi_adamw_step);
        take(entries, "geomae_group_norm_workspace_bytes", lib.group_norm_workspace_bytes);
        take(entries, "geomae_group_norm_forward", lib.group_norm_forward);
        take(entries, "geomae_group_norm_backward", lib.group_norm_backward);
        take(entries, "geomae_last_error", lib.last_error);
        library_error = std::move(error);
    });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LibraryError& e) {
            PyErr_SetString(library_error.ptr(), e.what());
        }
    });
    py::class_<AdamwPlan>(m, "AdamwPlan")
        .def(py::init([](const std::vector<at::Tensor>& params, std::vector<int64_t> first_chunk, uintptr_t table, uintptr_t chunks, uintptr_t workspace,
                         int64_t workspace_bytes, uintptr_t norm_word, int state_bits) {
            TORCH_CHECK(first_chunk.size() == params.size() + 1, "AdamwPlan: one first chunk per tensor and the end are wanted");
            AdamwPlan p;
            for (const at::Tensor& t : params) p.params.emplace_back(t);
            p.first_chunk = std::move(first_chunk);
            p.table = reinterpret_cast<const GeomaeAdamwTensor*>(table);
            p.chunks = reinterpret_cast<const int32_t*>(chunks);
            p.workspace = reinterpret_cast<void*>(workspace);
            p.workspace_bytes = workspace_bytes;
            p.norm_word = reinterpret_cast<float*>(norm_word);
            p.state_bits = state_bits;
            p.seed = 0;
            p.captured = p.new_stream = false;
            p.grads.resize(params.size());
            p.hyper_of.resize(params.size());
            return p;
        }))
        .def_readwrite("seed", &AdamwPlan::seed)
        .def_readonly("captured", &AdamwPlan::captured)
        .def_readonly("new_stream", &AdamwPlan::new_stream)
        .def("step", &adamw_step);
    m.def("group_norm_act", &group_norm_act);
    m.def("accumulates_on_default_stream", &accumulates_on_default_stream);
}
