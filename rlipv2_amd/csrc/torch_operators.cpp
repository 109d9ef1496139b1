// torch_operators.cpp -- the host side of the cross attention and gradient norm operators: tensors to the C ABI of
// include/rlipv2_attention.h and include/rlipv2_gradnorm.h, workspaces, the autograd node.
//
// In C++ because of what the same lines cost in Python: a training step of one query over 64 labels spent 137 us on the host (an
// autograd function that does nothing: 53 us), several times its kernels.  The backward pass runs in the autograd engine's own thread
// without the interpreter.  The argument checks are in Python (rlipv2_amd/attention.py, optim.py); the entry points of the kernel
// library are handed over by bind(), so that this module and ctypes use one loaded library.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <limits>

#include "../../include/rlipv2_attention.h"
#include "../../include/rlipv2_gradnorm.h"
#include "../../include/rlipv2_msda.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Entries {
    decltype(&cross_attention_forward) forward;
    decltype(&cross_attention_backward) backward;
    decltype(&cross_attention_workspace_bytes) workspace;
    decltype(&cross_attention_short_keys) short_keys;
    decltype(&grad_norm) norm;
    decltype(&grad_clip) clip;
    decltype(&grad_norm_workspace_bytes) norm_workspace;
    decltype(&msda_strerror) strerror;
} entry;

void *stream_of(const at::Device &device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

void check(int status, const char *name) { TORCH_CHECK(status == 0, name, ": ", entry.strerror(status)); }

// The tensor itself where the kernels can read it: elements of a head contiguous, rows 16-byte aligned and less than 64 MB apart (the
// stride of a dimension of one element is never used: any value); else a copy.  A copy even of what counts as contiguous: contiguous()
// would return the same memory.
Tensor operand(const Tensor &t)
{
    const int64_t unit = 16 / (int64_t)t.element_size();
    bool fits = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i)
        fits &= t.size(i) <= 1 || (t.stride(i) % unit == 0 && (i != 1 || t.stride(i) < ((int64_t)1 << 22) * unit));
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

void set_strides(int64_t (&to)[3], const Tensor &t)
{
    for (int i = 0; i < 3; ++i) to[i] = t.size(i) <= 1 ? 0 : t.stride(i);
}

const void *data(const Maybe &t) { return t && t->defined() ? t->const_data_ptr() : nullptr; }

cross_attention_args args_of(const Tensor &q, const Tensor &k, const Tensor &v, const Maybe &padding, const Maybe &lengths, const Maybe &keep,
                             double scale, double keep_scale)
{
    cross_attention_args a = {};
    a.dtype = q.scalar_type() == at::kFloat ? MSDA_F32 : MSDA_BF16;
    // (sizes beyond 32 bits become one that the C entry refuses)
    const auto size = [](int64_t n) { return n > std::numeric_limits<int32_t>::max() ? -1 : (int32_t)n; };
    a.B = size(q.size(0)); a.Lq = size(q.size(1)); a.heads = size(q.size(2)); a.D = size(q.size(3));
    a.Lk = size(k.size(1)); a.kv_heads = size(k.size(2));
    a.scale = (float)scale;
    a.keep_scale = (float)keep_scale;
    a.query = q.const_data_ptr(); a.key = k.const_data_ptr(); a.value = v.const_data_ptr();
    set_strides(a.query_stride, q);
    set_strides(a.key_stride, k);
    set_strides(a.value_stride, v);
    a.padding = data(padding);
    a.padding_stride = a.padding ? padding->stride(0) : 0;
    a.lengths = data(lengths);
    a.keep = data(keep);
    return a;
}

// (the workspace belongs to this call: the allocator hands its memory on in stream order, a captured graph keeps its own)
Tensor give_workspace(cross_attention_args &a, bool backward, const Tensor &like)
{
    a.workspace_bytes = entry.workspace(&a, backward);
    Tensor work;
    if (a.workspace_bytes) {
        work = at::empty({(int64_t)a.workspace_bytes}, like.options().dtype(at::kByte));
        a.workspace = work.data_ptr();
    }
    return work;
}

struct Forward { Tensor q, k, v, out, low, stats; };

// `training`: also what the backward pass reads (the rows' statistics, and what rounding took from the result where it is wanted)
Forward run_forward(const Tensor &query, const Tensor &key, const Tensor &value, const Maybe &padding, const Maybe &lengths,
                    const Maybe &keep, double scale, double keep_scale, bool training)
{
    Forward f;
    f.q = operand(query); f.k = operand(key); f.v = operand(value);
    f.out = at::empty(query.sizes(), query.options());
    cross_attention_args a = args_of(f.q, f.k, f.v, padding, lengths, keep, scale, keep_scale);
    if (training) {
        f.stats = at::empty({query.size(0), query.size(2), query.size(1)}, query.options().dtype(at::kFloat));
        if (a.dtype == MSDA_BF16 && !entry.short_keys(&a)) f.low = at::empty(query.sizes(), query.options());
    }
    if (f.out.numel() == 0) return f;
    const c10::DeviceGuard guard(query.device());
    a.out = f.out.data_ptr();
    a.out_low = f.low.defined() ? f.low.data_ptr() : nullptr;
    a.stats = training ? f.stats.data_ptr() : nullptr;
    const Tensor work = give_workspace(a, false, query);
    check(entry.forward(&a, stream_of(query.device())), "cross_attention_forward");
    return f;
}

struct CrossAttentionFunction : public torch::autograd::Function<CrossAttentionFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &query, const Tensor &key, const Tensor &value, const Maybe &padding,
                          const Maybe &lengths, const Maybe &keep, double scale, double keep_scale)
    {
        const Forward f = run_forward(query, key, value, padding, lengths, keep, scale, keep_scale, true);
        ctx->save_for_backward({f.q, f.k, f.v, padding.value_or(Tensor()), lengths.value_or(Tensor()), keep.value_or(Tensor()), f.out, f.low,
                                f.stats});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["keep_scale"] = keep_scale;
        return f.out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[6], &low = s[7], &stats = s[8];
        const bool again = at::GradMode::is_enabled();          // (create_graph: the result must not look differentiable)
        variable_list result(8);
        {
            const at::NoGradGuard no_grad;
            const c10::DeviceGuard guard(q.device());
            const bool states = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
            result[0] = at::empty(q.sizes(), q.options());
            if (states) {
                result[1] = at::empty(k.sizes(), k.options());
                result[2] = at::empty(v.sizes(), v.options());
            }
            if (result[0].numel() || (states && result[1].numel())) {
                const Tensor grad_out = operand(grads[0].scalar_type() == q.scalar_type() ? grads[0] : grads[0].to(q.scalar_type()));
                const Tensor delta = at::empty(stats.sizes(), stats.options());
                cross_attention_args a = args_of(q, k, v, s[3], s[4], s[5], ctx->saved_data["scale"].toDouble(),
                                                 ctx->saved_data["keep_scale"].toDouble());
                a.out = out.data_ptr();
                a.out_low = low.defined() ? low.data_ptr() : nullptr;
                a.stats = stats.data_ptr();
                a.grad_out = grad_out.const_data_ptr();
                set_strides(a.grad_out_stride, grad_out);
                a.grad_query = result[0].data_ptr();
                a.grad_key = states ? result[1].data_ptr() : nullptr;
                a.grad_value = states ? result[2].data_ptr() : nullptr;
                a.delta = delta.data_ptr();
                const Tensor work = give_workspace(a, true, q);
                check(entry.backward(&a, stream_of(q.device())), "cross_attention_backward");
            }
        }
        if (again) {
            variable_list some;
            for (const Tensor &t : result)
                if (t.defined()) some.push_back(t);
            const auto error = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)some.size());
            some = (*error)(std::move(some));
            size_t at = 0;
            for (Tensor &t : result)
                if (t.defined()) t = some[at++];
        }
        return result;
    }
};

Tensor cross_attention(const Tensor &query, const Tensor &key, const Tensor &value, const Maybe &padding, const Maybe &lengths,
                       const Maybe &keep, double scale, double keep_scale)
{
    // (the kernels write through raw pointers: a tangent would be lost without a word)
    for (const Tensor *t : {&query, &key, &value})
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "cross_attention: forward-mode derivatives are not implemented");
    if (at::GradMode::is_enabled() && (query.requires_grad() || key.requires_grad() || value.requires_grad()))
        return CrossAttentionFunction::apply(query, key, value, padding, lengths, keep, scale, keep_scale);
    return run_forward(query, key, value, padding, lengths, keep, scale, keep_scale, false).out;
}

// (norm, workspace): the lists are the addresses of host arrays
std::pair<Tensor, Tensor> call_grad_norm(uintptr_t src, uintptr_t types, uintptr_t numel, int n, int order, double scale, int device)
{
    const c10::Device where(c10::DeviceType::CUDA, (c10::DeviceIndex)device);
    const c10::DeviceGuard guard(where);
    const size_t bytes = entry.norm_workspace(n);
    Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(where));
    Tensor work = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(where));
    check(entry.norm(reinterpret_cast<const void *const *>(src), reinterpret_cast<const uint8_t *>(types), reinterpret_cast<const int64_t *>(numel),
                     n, order, scale, work.data_ptr(), bytes, norm.data_ptr<float>(), stream_of(where)), "grad_norm");
    return {norm, work};
}

void call_grad_clip(uintptr_t src, uintptr_t types, uintptr_t dst, uintptr_t dst_types, uintptr_t numel, int n, double max_norm, double scale,
                    const Tensor &work)
{
    const c10::DeviceGuard guard(work.device());
    check(entry.clip(reinterpret_cast<const void *const *>(src), reinterpret_cast<const uint8_t *>(types), reinterpret_cast<void *const *>(dst),
                     reinterpret_cast<const uint8_t *>(dst_types), reinterpret_cast<const int64_t *>(numel), n, max_norm, scale,
                     work.const_data_ptr(), stream_of(work.device())), "grad_clip");
}

void bind_entries(const std::vector<uintptr_t> &p)
{
    TORCH_CHECK(p.size() * sizeof(uintptr_t) == sizeof(Entries), "bind: ", sizeof(Entries) / sizeof(uintptr_t), " entry points");
    std::memcpy(static_cast<void *>(&entry), p.data(), sizeof(Entries));
}

}  // namespace

PYBIND11_MODULE(_operators, m)
{
    m.def("bind", &bind_entries);
    m.def("cross_attention", &cross_attention, py::call_guard<py::gil_scoped_release>());
    m.def("grad_norm", &call_grad_norm);
    m.def("grad_clip", &call_grad_clip);
}
