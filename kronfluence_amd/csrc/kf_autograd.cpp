// kf_autograd.cpp -- the differentiable operators of kronfluence_amd/functional.py over the C ABI of libkronfluence_hip.so.
//
// The rest of the package reaches the library through ctypes; these operators are called once per layer and pass inside the USER's
// model, forward from Python and backward from autograd's device thread, where a Python backward waits for the interpreter and runs
// on a thread that has just been woken.  Measured on calls whose kernels take 15 us: forward and backward of a norm of 32 x 1001
// elements 120 us with the nodes in Python.  So the argument checks, allocations and nodes are C++; nothing here computes.
//
// Errors become KfError.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/kronfluence_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct KfFailure : std::runtime_error {
    using std::runtime_error::runtime_error;
};

// (messages are put together only when they are needed)
#define KF_REQUIRE(condition, message) \
    do { \
        if (!(condition)) throw KfFailure(std::string("invalid argument: ") + (message)); \
    } while (0)

void check(int status, const char* what) {
    if (status != KF_OK) throw KfFailure(std::string(what) + " failed: " + kf_status_string(status) + " (" + std::to_string(status) + ")");
}

void require_device(const Tensor& t, const char* name) {
    if (!t.is_cuda())
        throw KfFailure(std::string("`") + name + "` lives on " + t.device().str() + "; the operators run only on an MI355X (there is no CPU fallback).");
}

int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return KF_F32;
        case at::kBFloat16: return KF_BF16;
        case at::kHalf: return KF_F16;
        default: return -1;
    }
}

// the current stream of the tensor's device (a DeviceGuard at the callers makes that device the current one for the launch)
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool wants_graph(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The kernels' backward passes are not differentiable themselves: a graph of the gradients would silently lack these operators.
void first_derivatives_only() {
    if (at::GradMode::is_enabled()) throw KfFailure("invalid argument: kronfluence_amd.functional has first derivatives only (create_graph=True)");
}

// The kernels read memory and write into fresh tensors: a forward-mode tangent, a node of a trace, or what a wrapper (torch.func's
// transforms, a subclass with a dispatch of its own) stands for would be lost without a word.
void plain_tensors(std::initializer_list<const Tensor*> tensors) {
    constexpr c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                            c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor});
    for (const Tensor* t : tensors) {
        if (!t->defined()) continue;
        KF_REQUIRE(!t->key_set().has_any(wrappers),
                   "kronfluence_amd.functional takes plain tensors (no torch.func transform, no subclass with a dispatch of its own)");
        KF_REQUIRE(!t->_fw_grad(0).defined(), "kronfluence_amd.functional has no forward-mode derivatives (the tangent would be lost)");
    }
    KF_REQUIRE(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
               "kronfluence_amd.functional cannot be recorded in a trace");
}

Tensor given(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// ---- attention ----------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_WIDTH = 128, MAX_TOKEN_BYTES = int64_t{1} << 23;

struct AttentionCall {
    int64_t sequences, length, rows, heads, kv_heads, width;
    int dtype, causal;
    float scale;
    bool empty() const { return sequences == 0 || rows == 0; }
};

AttentionCall attention_call(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& offsets, bool causal, double scale) {
    const bool packed = offsets.defined();
    KF_REQUIRE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() && v.device() == q.device(),
               "q, k and v share one dtype and one device");
    KF_REQUIRE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat,
               std::string("attention takes bfloat16 or float32 tensors, not ") + c10::toString(q.scalar_type()));
    KF_REQUIRE(!(packed && lengths.defined()), "lengths (padded batch) and cu_seqlens (packed batch) exclude each other");
    const int64_t dims = q.dim();
    KF_REQUIRE(dims == (packed ? 3 : 4), "q is [tokens, heads, width] with cu_seqlens, [batch, length, heads, width] without");
    const auto shape = q.sizes(), kv_shape = k.sizes();
    KF_REQUIRE(static_cast<int64_t>(kv_shape.size()) == dims && v.sizes() == kv_shape && kv_shape.slice(0, dims - 2) == shape.slice(0, dims - 2) &&
                   kv_shape[dims - 1] == shape[dims - 1],
               "k and v have the shape of q, but for the number of heads");
    AttentionCall c;
    c.heads = shape[dims - 2];
    c.kv_heads = kv_shape[dims - 2];
    c.width = shape[dims - 1];
    KF_REQUIRE(c.kv_heads > 0 && c.heads > 0 && c.heads % c.kv_heads == 0, "the number of heads is a multiple of the number of key / value heads");
    KF_REQUIRE(c.width > 0 && c.width <= MAX_WIDTH, "head widths up to " + std::to_string(MAX_WIDTH));
    KF_REQUIRE(std::isfinite(scale) && scale > 0 && static_cast<float>(scale) > 0 && std::isfinite(static_cast<float>(scale)), "scale is positive and finite");
    for (const Tensor* t : {&lengths, &offsets})
        KF_REQUIRE(!t->defined() || (t->dim() == 1 && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->device() == q.device()),
                   std::string(t == &lengths ? "lengths" : "cu_seqlens") + " is a vector of int32 or int64 on the device of q");
    if (packed) {
        KF_REQUIRE(offsets.numel() >= 1, "cu_seqlens holds the first row of every sequence and the last row's end");
        c.sequences = offsets.numel() - 1;
        c.length = 0;
        c.rows = shape[0];
    } else {
        KF_REQUIRE(!lengths.defined() || lengths.numel() == shape[0], "lengths has one entry per row of the batch");
        c.sequences = shape[0];
        c.length = shape[1];
        c.rows = shape[0] * shape[1];
    }
    require_device(q, "q");
    c.dtype = type_code(q);
    c.causal = causal;
    c.scale = static_cast<float>(scale);
    return c;
}

// `t` itself if the kernels can read it in place (contiguous width, 16-byte aligned start and strides, rows that do not overlap), else
// a contiguous copy.  The head width is a whole number of 16-byte chunks.
Tensor heads_operand(const Tensor& t) {
    const int64_t size = static_cast<int64_t>(t.element_size()), dims = t.dim();
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) {
        if (t.is_contiguous() && t.stride(dims - 3) * size <= MAX_TOKEN_BYTES) return t;
        bool usable = t.stride(dims - 1) == 1 &&
                      (t.size(dims - 3) == 1 || (t.stride(dims - 3) >= t.size(dims - 1) && t.stride(dims - 3) * size <= MAX_TOKEN_BYTES));
        for (int64_t i = 0; i < dims - 1; ++i) usable = usable && (t.size(i) == 1 || t.stride(i) * size % 16 == 0);
        if (usable) return t;
    }
    return t.clone(at::MemoryFormat::Contiguous);
}

kf_heads_view view(const Tensor& t) {   // (an axis of one element may carry any stride)
    const int64_t dims = t.dim();
    return kf_heads_view{t.data_ptr(), dims == 4 && t.size(0) > 1 ? t.stride(0) : 0, t.size(dims - 3) > 1 ? t.stride(dims - 3) : t.size(dims - 1),
                         t.size(dims - 2) > 1 ? t.stride(dims - 2) : 0};
}

// lengths as the kernels read them: contiguous int32, which they clamp to the rows that exist
Tensor row_counts(const Tensor& t, int64_t most) {
    if (!t.defined()) return t;
    return (t.scalar_type() == at::kInt ? t : t.clamp(0, most).to(at::kInt)).contiguous();
}

// offsets as the kernels read them: int32, within the rows and ascending, whatever the caller's say
Tensor row_starts(const AttentionCall& c, const Tensor& offsets) {
    if (!offsets.defined()) return offsets;
    const Tensor given = offsets.contiguous(), starts = at::empty({c.sequences + 1}, offsets.options().dtype(at::kInt));
    check(kf_attention_starts(starts.data_ptr<int32_t>(), given.data_ptr(), given.scalar_type() == at::kLong ? KF_I64 : KF_I32, c.sequences, c.rows,
                              stream_of(given)),
          "kf_attention_starts");
    return starts;
}

// the order a packed batch is best worked on in, or an undefined tensor
Tensor work_order(const AttentionCall& c, const Tensor& starts) {
    const int64_t bytes = starts.defined() ? kf_attention_order_bytes(c.sequences, c.rows, c.heads) : 0;
    if (bytes == 0) return Tensor();
    Tensor order = at::empty({bytes / 4}, starts.options());
    check(kf_attention_order(order.data_ptr<int32_t>(), starts.data_ptr<int32_t>(), c.sequences, c.rows, c.causal, stream_of(starts)), "kf_attention_order");
    return order;
}

// `lengths` and `offsets` come back as the kernels read them, for the backward pass
Tensor attention_forward(const AttentionCall& c, Tensor q, Tensor k, Tensor v, Tensor& lengths, Tensor& offsets, Tensor* stats, Tensor* order_out) {
    Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    if (stats)
        *stats = at::empty({kf_attention_stats_bytes(c.dtype, c.length, c.rows, c.heads, c.width, offsets.defined()) / 4}, q.options().dtype(at::kFloat));
    if (c.empty()) return out.zero_();
    const c10::DeviceGuard guard(q.device());
    q = heads_operand(q); k = heads_operand(k); v = heads_operand(v);
    lengths = row_counts(lengths, c.length);
    offsets = row_starts(c, offsets);
    const Tensor order = work_order(c, offsets);
    if (order_out) *order_out = order;
    const kf_heads_view vo = view(out), vq = view(q), vk = view(k), vv = view(v);
    check(kf_attention_forward(&vo, stats ? stats->data_ptr<float>() : nullptr, &vq, &vk, &vv, c.dtype, c.sequences, c.length, c.rows, c.heads, c.kv_heads, c.width,
                               static_cast<const int32_t*>(pointer(lengths)), static_cast<const int32_t*>(pointer(offsets)),
                               static_cast<const int32_t*>(pointer(order)), c.causal, c.scale, stream_of(q)),
          "kf_attention_forward");
    return out;
}

variable_list attention_backward(const AttentionCall& c, Tensor grad, Tensor out, const Tensor& stats, Tensor q, Tensor k, Tensor v, const Tensor& lengths,
                                 const Tensor& offsets, const Tensor& order) {
    const auto plain = q.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor dq = at::empty(q.sizes(), plain), dk = at::empty(k.sizes(), plain), dv = at::empty(v.sizes(), plain);
    if (c.empty()) return {dq.zero_(), dk.zero_(), dv.zero_()};
    const c10::DeviceGuard guard(q.device());
    grad = heads_operand(grad); out = heads_operand(out); q = heads_operand(q); k = heads_operand(k); v = heads_operand(v);
    const int64_t bytes = kf_attention_backward_workspace_bytes(c.sequences, c.length, c.rows, c.heads, c.kv_heads, c.width, offsets.defined(), c.causal);
    const Tensor workspace = at::empty({bytes}, q.options().dtype(at::kByte));
    const kf_heads_view vdq = view(dq), vdk = view(dk), vdv = view(dv), vg = view(grad), vo = view(out), vq = view(q), vk = view(k), vv = view(v);
    check(kf_attention_backward(&vdq, &vdk, &vdv, &vg, &vo, stats.data_ptr<float>(), &vq, &vk, &vv, c.dtype, c.sequences, c.length, c.rows, c.heads, c.kv_heads,
                                c.width, static_cast<const int32_t*>(pointer(lengths)), static_cast<const int32_t*>(pointer(offsets)),
                                static_cast<const int32_t*>(pointer(order)), c.causal, c.scale, workspace.data_ptr(), bytes, stream_of(q)),
          "kf_attention_backward");
    return {dq, dk, dv};
}

struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& lengths_,
                          const std::optional<Tensor>& offsets_, bool causal, double scale) {
        Tensor lengths = given(lengths_), offsets = given(offsets_), stats, order;
        const Tensor out = attention_forward(attention_call(q, k, v, lengths, offsets, causal, scale), q, k, v, lengths, offsets, &stats, &order);
        ctx->save_for_backward({q, k, v, out, stats, lengths, offsets, order});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &lengths = saved[5], &offsets = saved[6];
        if (!grads[0].defined()) return variable_list(7);
        plain_tensors({&grads[0]});
        const AttentionCall c = attention_call(q, k, v, lengths, offsets, ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
        variable_list d = attention_backward(c, grads[0], saved[3], saved[4], q, k, v, lengths, offsets, saved[7]);
        d.resize(7);
        return d;
    }
};

Tensor attention(Tensor q, Tensor k, Tensor v, bool causal, const std::optional<double>& scale, const std::optional<Tensor>& lengths_,
                 const std::optional<Tensor>& offsets_) {
    Tensor lengths = given(lengths_), offsets = given(offsets_);
    plain_tensors({&q, &k, &v, &lengths, &offsets});
    const int64_t width = q.dim() > 0 ? q.size(-1) : 0;
    const double by = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(width, 1)));
    const AttentionCall c = attention_call(q, k, v, lengths, offsets, causal, by);
    const int64_t whole = 16 / static_cast<int64_t>(q.element_size()), pad = (whole - c.width % whole) % whole;
    if (pad) {   // zero columns change no product
        q = at::constant_pad_nd(q, {0, pad});
        k = at::constant_pad_nd(k, {0, pad});
        v = at::constant_pad_nd(v, {0, pad});
    }
    Tensor out;
    if (wants_graph({&q, &k, &v})) out = Attention::apply(q, k, v, lengths_, offsets_, causal, by);
    else out = attention_forward(pad ? attention_call(q, k, v, lengths, offsets, causal, by) : c, q, k, v, lengths, offsets, nullptr, nullptr);
    return pad ? out.narrow(-1, 0, c.width) : out;
}

// ---- norms --------------------------------------------------------------------------------------------------------------
struct NormCall {
    int64_t rows, width;
    int dtype, vector_dtype;
};

NormCall norm_call(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    KF_REQUIRE(x.dim() >= 1 && x.size(-1) > 0, "x has a last axis to normalise over");
    NormCall c{x.numel() / x.size(-1), x.size(-1), type_code(x), 0};
    KF_REQUIRE(c.dtype >= 0, std::string("norms take float32, bfloat16 or float16 tensors, not ") + c10::toString(x.scalar_type()));
    for (const Tensor* t : {&weight, &bias})
        KF_REQUIRE(!t->defined() || (t->dim() == 1 && t->numel() == c.width && t->device() == x.device()),
                   std::string(t == &weight ? "weight" : "bias") + " is a vector of x's width on x's device");
    const Tensor& vector = weight.defined() ? weight : bias;
    if (vector.defined()) c.vector_dtype = type_code(vector);
    KF_REQUIRE(c.vector_dtype >= 0 && (!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type()),
               "weight and bias share one of the dtypes float32, bfloat16 and float16");
    require_device(x, "x");
    return c;
}

// x with a contiguous last axis, in place where its strides allow it, and the stride of its rows
std::pair<Tensor, int64_t> norm_rows(const Tensor& x, int64_t width) {
    if (x.is_contiguous()) return {x, width};
    Tensor flat = x.reshape({-1, width});
    if (flat.stride(1) != 1 && width != 1) flat = flat.contiguous();
    return {flat, flat.stride(0)};
}

Tensor norm_forward(const Tensor& x, Tensor weight, Tensor bias, double eps, bool centred, at::ScalarType out_type, Tensor* stats) {
    const NormCall c = norm_call(x, weight, bias);
    Tensor out = at::empty(x.sizes(), x.options().dtype(out_type).memory_format(at::MemoryFormat::Contiguous));
    if (stats) *stats = at::empty({c.rows, 2}, x.options().dtype(at::kFloat));
    if (c.rows == 0) return out;
    const c10::DeviceGuard guard(x.device());
    const auto [rows, stride] = norm_rows(x, c.width);
    if (weight.defined()) weight = weight.contiguous();
    if (bias.defined()) bias = bias.contiguous();
    check(kf_norm_forward(out.data_ptr(), type_code(out), stats ? stats->data_ptr<float>() : nullptr, rows.data_ptr(), c.dtype, c.rows, c.width, stride,
                          pointer(weight), pointer(bias), c.vector_dtype, centred, static_cast<float>(eps), stream_of(x)),
          "kf_norm_forward");
    return out;
}

struct Norm : torch::autograd::Function<Norm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps,
                          bool centred, int64_t out_type) {
        const Tensor weight = given(weight_), bias = given(bias_);
        Tensor stats;
        const Tensor out = norm_forward(x, weight, bias, eps, centred, static_cast<at::ScalarType>(out_type), &stats);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["centred"] = centred;
        ctx->saved_data["bias"] = bias.defined() ? static_cast<int64_t>(bias.scalar_type()) : -1;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &stats = saved[2];
        Tensor weight = saved[1], grad = grads[0];
        variable_list d(6);
        if (!grad.defined()) return d;
        plain_tensors({&grad});
        const int64_t bias = ctx->saved_data["bias"].toInt();
        NormCall c = norm_call(x, weight, Tensor());
        const auto plain = x.options().memory_format(at::MemoryFormat::Contiguous);
        if (ctx->needs_input_grad(0)) d[0] = at::empty(x.sizes(), plain);
        if (weight.defined() && ctx->needs_input_grad(1)) d[1] = at::empty({c.width}, weight.options());
        if (bias >= 0 && ctx->needs_input_grad(weight.defined() ? 2 : 1)) d[2] = at::empty({c.width}, x.options().dtype(static_cast<at::ScalarType>(bias)));
        if (c.rows == 0) {
            for (Tensor& t : d)
                if (t.defined()) t.zero_();
            return d;
        }
        const c10::DeviceGuard guard(x.device());
        const auto [rows, stride] = norm_rows(x, c.width);
        grad = grad.contiguous();
        if (weight.defined()) weight = weight.contiguous();
        Tensor workspace;
        int64_t bytes = 0;
        if (d[1].defined() || d[2].defined()) {
            bytes = kf_norm_backward_workspace_bytes(c.rows, c.width);
            workspace = at::empty({bytes}, x.options().dtype(at::kByte));
            c.vector_dtype = type_code(d[1].defined() ? d[1] : d[2]);
        }
        check(kf_norm_backward(pointer(d[0]), pointer(d[1]), pointer(d[2]), grad.data_ptr(), type_code(grad), rows.data_ptr(), c.dtype,
                               stats.data_ptr<float>(), c.rows, c.width, stride, pointer(weight), c.vector_dtype, ctx->saved_data["centred"].toBool(),
                               pointer(workspace), bytes, stream_of(x)),
              "kf_norm_backward");
        return d;
    }
};

Tensor norm(const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps, bool centred, at::ScalarType out_type) {
    const Tensor weight = given(weight_), bias = given(bias_);
    plain_tensors({&x, &weight, &bias});
    KF_REQUIRE(out_type == at::kFloat || out_type == at::kBFloat16 || out_type == at::kHalf,
               std::string("norms return float32, bfloat16 or float16 tensors, not ") + c10::toString(out_type));
    KF_REQUIRE(std::isfinite(eps) && eps >= 0, "eps is finite and not negative");
    if (wants_graph({&x, &weight, &bias})) return Norm::apply(x, weight_, bias_, eps, centred, static_cast<int64_t>(out_type));
    return norm_forward(x, weight, bias, eps, centred, out_type, nullptr);
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    m.def("abi_version", &kf_abi_version);
    m.def("attention", &attention);
    m.def("norm", &norm);
    m.def("set_error_type", [](const py::object& type) {   // kronfluence_amd._native.KfError
        static PyObject* error = nullptr;
        error = type.inc_ref().ptr();
        py::register_exception_translator([](std::exception_ptr p) {
            try {
                if (p) std::rethrow_exception(p);
            } catch (const KfFailure& e) {
                PyErr_SetString(error, e.what());
            }
        });
    });
}
