// Autograd nodes of the operators whose calls are short: layer_norm, embedding, linear_cross_entropy and balance_loss.
//
// A backward pass runs on a thread of torch's own, and what it costs beyond the kernels is that thread's start and the host
// code that both threads come back to with cold caches: with the nodes in Python, layer_norm of 4096 x 384 and its gradients
// took 117 us a pass of which the kernels are 21, and 66 so; SRHead's loss of 128 rows, 6656 words of 1000 143 and 85.  The
// operators' arguments are checked here, their kernels are called through the C ABI of libmuon_sr_amd.so on the tensors' device and
// its current stream, their scratch memory comes from torch's allocator.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/muon_sr_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject *library_error = nullptr;   // _lib.MuonSRLibraryError
PyObject *accumulator = nullptr;     // _lib.accumulator

void check(int rc, const char *name) {
    if (!rc) return;
    const char *const why = msr_last_error();
    const std::string text = std::string(name) + " failed with code " + std::to_string(rc) + ": " + (why ? why : "");
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(library_error ? library_error : PyExc_RuntimeError, text.c_str());
    python_error e;
    e.persist();
    throw e;
}

// fn(args..., stream) on t's device and its current stream
template <typename F, typename... Args>
void call(const Tensor &t, const char *name, F fn, Args... args) {
    const c10::DeviceGuard guard(t.device());
    check(fn(args..., (msr_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream()), name);
}

// A weight's accumulator, as a backward pass finds it, and what it is accumulated with.
struct Accumulator {
    Tensor acc;
    uint32_t seed;
    int32_t noise_mode;
    bool first;                          // the weight has none yet: acc's elements are undefined
    // (the weight as Python has it: the accumulator is its attribute)
    Accumulator(const Tensor &owner, const char *what) {
        pybind11::gil_scoped_acquire gil;
        PyObject *const r = PyObject_CallFunction(accumulator, "Ns", THPVariable_Wrap(owner), what);
        if (!r) fail();
        const auto t = pybind11::reinterpret_steal<pybind11::tuple>(r);
        acc = THPVariable_Unpack(pybind11::object(t[0]).ptr());
        seed = t[1].cast<uint32_t>();
        first = t[2].cast<bool>();
        noise_mode = t[3].cast<int32_t>();
    }
    // after the call that wrote it
    void keep(const Tensor &owner) const {
        if (!first) return;
        pybind11::gil_scoped_acquire gil;
        const auto to = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(owner)), value = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(acc));
        if (PyObject_SetAttrString(to.ptr(), "acc_grad", value.ptr())) fail();
    }
    [[noreturn]] static void fail() {    // with Python's error
        python_error e;
        e.persist();
        throw e;
    }
};

const void *in(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
template <typename T>
T *at_(const Tensor &t) { return static_cast<T *>(out(t)); }

Tensor empty(at::IntArrayRef shape, const Tensor &like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }
Tensor workspace(size_t bytes, const Tensor &like) { return bytes ? empty({(int64_t)bytes}, like, at::kByte) : Tensor(); }

bool elem_ok(const Tensor &t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
int32_t elem(const Tensor &t) { return t.scalar_type() == at::kFloat ? MSR_F32 : MSR_BF16; }
bool whole(const Tensor &t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

void one_gpu(const char *what, const Tensor &first, std::initializer_list<const Tensor *> others) {
    TORCH_CHECK_VALUE(first.is_cuda(), what, " requires tensors on a ROCm GPU (got device ", first.device(), ")");
    for (const Tensor *t : others) {
        if (!t->defined() || t->device() == first.device()) continue;
        TORCH_CHECK_VALUE(t->is_cuda(), what, " requires tensors on a ROCm GPU (got device ", t->device(), ")");
        TORCH_CHECK_VALUE(false, what, " needs every tensor on one GPU");
    }
}

// t [..., d] as rows of unit column stride, and their stride
struct Rows {
    Tensor t;
    int64_t n, ld;
};
Rows flat_rows(const Tensor &t, int64_t d) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
    Rows r{t.dim() == 2 ? t : t.reshape({n, d}), n, d};
    if (n <= 1) {
        r.t = r.t.contiguous();
        return r;
    }
    if ((d > 1 && r.t.stride(1) != 1) || r.t.stride(0) < d) r.t = r.t.contiguous();
    r.ld = r.t.stride(0);
    return r;
}
Tensor contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
// contiguous and 16-byte aligned, as saved tensors were made and their hooks may not give them back
Tensor aligned(const Tensor &t) {
    const Tensor c = t.contiguous();
    return (uintptr_t)c.const_data_ptr() % 16 ? c.clone() : c;
}

// The gradients of a backward pass that is itself recorded: a second derivative raises.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor &g : grads) {
        if (!g.defined()) continue;
        auto error = std::make_shared<torch::autograd::DelayedError>("muon_sr_amd: the operators' gradients have no derivative of their own", 1);
        g = (*error)({g.detach().requires_grad_(true)})[0];
    }
    return grads;
}

// ---------------------------------------------------------------------------

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    // (a tensor that is left out has to be an empty optional here, and then has no number among the inputs)
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &w_, const std::optional<Tensor> &b_, double eps) {
        const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor());
        const int64_t d = x.size(-1);
        const Rows r = flat_rows(x, d);
        const Tensor weight = contiguous(w), bias = contiguous(b), y = at::empty(x.sizes(), x.options().requires_grad(false)),
                     stats = empty({3, r.n}, x, at::kFloat);   // mean's two numbers, rstd
        const Tensor &vector = weight.defined() ? weight : bias;
        const int32_t welem = vector.defined() ? elem(vector) : MSR_F32;
        float *const mean = at_<float>(stats);
        call(x, "msr_layer_norm", msr_layer_norm, in(r.t), r.ld, in(weight), in(bias), (float)eps, r.n, d, out(y), mean, mean + 2 * r.n, elem(x), welem);
        ctx->save_for_backward({x, w, stats});
        ctx->saved_data["welem"] = (int64_t)welem;
        ctx->saved_data["weight"] = w.defined();
        ctx->saved_data["bias"] = b.defined();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();   // saved-tensor hooks may have changed their strides
        const Tensor &x = saved[0], w = contiguous(saved[1]), stats = saved[2].contiguous();
        const int64_t d = x.size(-1);
        const Rows rx = flat_rows(x, d), ry = flat_rows(grads[0], d);
        const int32_t welem = (int32_t)ctx->saved_data["welem"].toInt();
        const auto vector = welem == MSR_F32 ? at::kFloat : at::kBFloat16;
        const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
        const Tensor dx = ctx->needs_input_grad(0) ? at::empty(x.sizes(), x.options().requires_grad(false)) : Tensor(),
                     dw = has_w && ctx->needs_input_grad(1) ? empty({d}, x, vector) : Tensor(),
                     db = has_b && ctx->needs_input_grad(has_w ? 2 : 1) ? empty({d}, x, vector) : Tensor();
        size_t bytes = 0;
        if (dw.defined() || db.defined()) check(msr_layer_norm_workspace_bytes(rx.n, d, elem(x), &bytes), "msr_layer_norm_workspace_bytes");
        const Tensor ws = workspace(bytes, x);
        const float *const mean = static_cast<const float *>(in(stats));
        call(x, "msr_layer_norm_grad", msr_layer_norm_grad, in(ry.t), ry.ld, in(rx.t), rx.ld, in(w), mean, mean + 2 * rx.n, rx.n, d, out(dx), out(dw),
             out(db), elem(x), welem, out(ws), bytes);
        return once({dx, dw, db, Tensor()});
    }
};

Tensor layer_norm(const Tensor &x, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    one_gpu("layer_norm", x, {&w, &b});
    TORCH_CHECK_VALUE(elem_ok(x), "layer_norm: x must be bf16 or fp32, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "layer_norm needs rows with elements, got ", x.sizes());
    for (const Tensor *t : {&w, &b})
        TORCH_CHECK_VALUE(!t->defined() || (elem_ok(*t) && t->dim() == 1 && t->size(0) == x.size(-1) && (!w.defined() || t->scalar_type() == w.scalar_type())),
                          "layer_norm needs a weight and bias of ", x.size(-1), " elements of one type, bf16 or fp32");
    return LayerNorm::apply(x, weight, bias, eps);
}

// ---------------------------------------------------------------------------

// accumulate: the gradient goes to w.acc_grad
struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext *ctx, const Tensor &ids_, const Tensor &w, double scale, int64_t padding, bool accumulate) {
        const Tensor ids = ids_.contiguous();
        const int64_t vocab = w.size(0), d = w.size(1);
        auto shape = ids.sizes().vec();
        shape.push_back(d);
        const Tensor y = at::empty(shape, w.options().requires_grad(false));
        call(w, "msr_embedding", msr_embedding, in(ids), (int32_t)(ids.scalar_type() == at::kLong), ids.numel(), in(w), vocab, d, (float)scale, out(y), elem(w));
        ctx->save_for_backward({ids});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["vocab"] = vocab;
        // the tensor that holds acc_grad: saved-tensor hooks (activation checkpointing, offloading) unpack another one
        if (accumulate) ctx->saved_data["owner"] = w;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor ids = ctx->get_saved_variables()[0].contiguous(), &dy = grads[0];
        const int64_t vocab = ctx->saved_data["vocab"].toInt(), d = dy.size(-1), n = ids.numel();
        const Rows r = flat_rows(dy, d);
        const auto owner = ctx->saved_data.find("owner");
        size_t bytes = 0;
        check(msr_embedding_workspace_bytes(n, vocab, d, &bytes), "msr_embedding_workspace_bytes");
        if (owner != ctx->saved_data.end()) {
            const Tensor w = owner->second.toTensor();
            const Accumulator to(w, "SREmbedding");
            const Tensor ws = workspace(bytes, dy);
            call(dy, "msr_embedding_grad_sr_accum", msr_embedding_grad_sr_accum, in(ids), (int32_t)(ids.scalar_type() == at::kLong), n,
                 static_cast<const uint16_t *>(in(r.t)), r.ld, vocab, d, (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(),
                 at_<uint16_t>(to.acc), to.seed, (int32_t)to.first, to.noise_mode, (const uint16_t *)nullptr, out(ws), bytes);
            to.keep(w);
            return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        }
        const Tensor dw = empty({vocab, d}, dy, dy.scalar_type()), ws = workspace(bytes, dy);
        call(dy, "msr_embedding_grad", msr_embedding_grad, in(ids), (int32_t)(ids.scalar_type() == at::kLong), n, in(r.t), r.ld, vocab, d,
             (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), out(dw), elem(dw), out(ws), bytes);
        return once({Tensor(), dw, Tensor(), Tensor(), Tensor()});
    }
};

// The arguments of `what`; the padding word's number, or -1
int64_t check_embedding(const char *what, const Tensor &ids, const Tensor &w, std::optional<int64_t> padding) {
    one_gpu(what, w, {&ids});
    TORCH_CHECK_VALUE(elem_ok(w), what, ": weight must be bf16 or fp32, got ", w.scalar_type());
    TORCH_CHECK_VALUE(w.dim() == 2 && w.is_contiguous(), what, " needs a contiguous weight [vocab, d], got ", w.sizes());
    TORCH_CHECK_VALUE(whole(ids), what, " needs int32 or int64 ids, got ", ids.scalar_type());
    const int64_t vocab = w.size(0);
    TORCH_CHECK_VALUE(vocab > 0, what, " needs words, got ", w.sizes());
    if (!padding) return -1;
    TORCH_CHECK_VALUE(*padding >= -vocab && *padding < vocab, what, ": padding_idx ", *padding, " is outside the ", vocab, " words");
    return *padding < 0 ? *padding + vocab : *padding;
}
// accumulate: w is a bf16 leaf that wants a gradient
Tensor embedding(const Tensor &ids, const Tensor &w, std::optional<int64_t> padding, double scale, bool accumulate) {
    const int64_t pad = check_embedding("embedding", ids, w, padding);
    return Embedding::apply(ids, w, scale, pad, accumulate);
}

// ---------------------------------------------------------------------------

// accumulate: the weight's gradient goes to w.acc_grad
struct HeadLoss : torch::autograd::Function<HeadLoss> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &target_, int64_t ignore, int64_t reduction, bool accumulate) {
        const int64_t vocab = w.size(0), d = w.size(1);
        const Rows r = flat_rows(x, d);
        const Tensor target = target_.contiguous(), packed = empty({r.n, d}, x, at::kBFloat16), kept = empty({3 * r.n + 1}, x, at::kInt),
                     sums = empty({r.n, 2}, x, at::kFloat), loss = empty(reduction == MSR_LOSS_NONE ? target.sizes() : at::IntArrayRef(), x, at::kFloat);
        size_t bytes = 0, backward_bytes = 0;
        check(msr_head_workspace_bytes(r.n, vocab, d, &bytes, &backward_bytes), "msr_head_workspace_bytes");
        const Tensor ws = workspace(bytes, x);
        call(x, "msr_head_forward", msr_head_forward, static_cast<const uint16_t *>(in(r.t)), r.ld, static_cast<const uint16_t *>(in(w)), in(target),
             (int32_t)(target.scalar_type() == at::kLong), ignore, r.n, vocab, d, (int32_t)reduction, at_<uint16_t>(packed), at_<int32_t>(kept),
             at_<float>(sums), at_<float>(loss), out(ws), bytes);
        ctx->save_for_backward({packed, w, kept, sums});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["reduction"] = reduction;
        if (accumulate) ctx->saved_data["owner"] = w;   // (as in Embedding)
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();   // saved-tensor hooks may have changed their strides
        const Tensor packed = aligned(saved[0]), w = aligned(saved[1]), kept = saved[2].contiguous(), sums = aligned(saved[3]),
                     dloss = grads[0].contiguous();
        const int64_t n = packed.size(0), vocab = w.size(0), d = w.size(1), reduction = ctx->saved_data["reduction"].toInt();
        const Tensor dx = ctx->needs_input_grad(0) ? empty(ctx->saved_data["shape"].toIntVector(), packed, at::kBFloat16) : Tensor();
        const auto owner = ctx->saved_data.find("owner");
        size_t forward_bytes = 0, bytes = 0;
        check(msr_head_workspace_bytes(n, vocab, d, &forward_bytes, &bytes), "msr_head_workspace_bytes");
        if (owner != ctx->saved_data.end()) {
            const Tensor weight = owner->second.toTensor();
            const Accumulator to(weight, "SRHead");
            const Tensor ws = workspace(bytes, packed);
            call(packed, "msr_head_backward", msr_head_backward, static_cast<const uint16_t *>(in(packed)), static_cast<const uint16_t *>(in(w)),
                 static_cast<const int32_t *>(in(kept)), static_cast<const float *>(in(sums)), static_cast<const float *>(in(dloss)), n, vocab, d,
                 (int32_t)reduction, at_<uint16_t>(dx), at_<uint16_t>(to.acc), to.noise_mode, to.seed, (int32_t)to.first, (const uint16_t *)nullptr, out(ws), bytes);
            to.keep(weight);
            return once({dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
        }
        const Tensor dw = ctx->needs_input_grad(1) ? empty({vocab, d}, w, at::kBFloat16) : Tensor(), ws = workspace(bytes, packed);
        call(packed, "msr_head_backward", msr_head_backward, static_cast<const uint16_t *>(in(packed)), static_cast<const uint16_t *>(in(w)),
             static_cast<const int32_t *>(in(kept)), static_cast<const float *>(in(sums)), static_cast<const float *>(in(dloss)), n, vocab, d,
             (int32_t)reduction, at_<uint16_t>(dx), at_<uint16_t>(dw), -1, 0u, 0, (const uint16_t *)nullptr, out(ws), bytes);
        return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

int64_t check_head(const char *what, const Tensor &x, const Tensor &w, const Tensor &target, const std::string &reduction) {
    one_gpu(what, x, {&w, &target});
    const int64_t code = reduction == "none" ? MSR_LOSS_NONE : reduction == "sum" ? MSR_LOSS_SUM : reduction == "mean" ? MSR_LOSS_MEAN : -1;
    TORCH_CHECK_VALUE(code >= 0, what, ": reduction must be 'mean', 'none' or 'sum', got '", reduction, "'");
    TORCH_CHECK_VALUE(w.dim() == 2 && w.is_contiguous(), what, " needs a contiguous weight [vocab, d], got ", w.sizes());
    TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16, what, " needs bf16 x and weight, got ", x.scalar_type(), " and ", w.scalar_type());
    TORCH_CHECK_VALUE(whole(target), what, " needs int32 or int64 targets, got ", target.scalar_type());
    const int64_t d = w.size(1);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == d && target.sizes() == x.sizes().slice(0, x.dim() - 1), what, " needs x [..., ", d,
                      "] and a target for each row, got ", x.sizes(), " and ", target.sizes());
    TORCH_CHECK_VALUE(d % 8 == 0 && d > 0 && w.size(0) > 0, what, " needs words, and a width that is a multiple of 8, got ", w.sizes());
    return code;
}
// accumulate: w is a leaf that wants a gradient
Tensor linear_cross_entropy(const Tensor &x, const Tensor &w, const Tensor &target, int64_t ignore, const std::string &reduction, bool accumulate) {
    const int64_t code = check_head(accumulate ? "SRHead" : "linear_cross_entropy", x, w, target, reduction);
    return HeadLoss::apply(x, w, target, ignore, code, accumulate);
}

// ---------------------------------------------------------------------------

struct Balance : torch::autograd::Function<Balance> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &ids_, const std::optional<Tensor> &mask_) {
        const int64_t tokens = logits.size(0), experts = logits.size(1);
        const Rows r = flat_rows(logits, experts);
        const Tensor ids = ids_.contiguous(), mask = contiguous(mask_.value_or(Tensor())), loss = empty({}, logits, at::kFloat), counts = empty({experts}, logits, at::kInt),
                     kept = empty({2 * tokens + experts}, logits, at::kFloat);   // the tokens' statistics, then slopes
        size_t bytes = 0;
        check(msr_balance_workspace_bytes(tokens, (int32_t)experts, &bytes), "msr_balance_workspace_bytes");
        const Tensor ws = workspace(bytes, logits);
        call(logits, "msr_balance_loss", msr_balance_loss, in(r.t), r.ld, in(ids), (int32_t)(ids.scalar_type() == at::kLong),
             static_cast<const uint8_t *>(in(mask)), tokens, (int32_t)experts, (int32_t)ids.size(1), at_<float>(loss), at_<int32_t>(counts),
             at_<float>(kept), at_<float>(kept) + 2 * tokens, elem(logits), out(ws), bytes);
        ctx->save_for_backward({logits, mask, kept});
        ctx->mark_non_differentiable({counts});
        return {loss, counts};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();   // saved-tensor hooks may have changed their strides
        const Tensor &logits = saved[0], mask = contiguous(saved[1]), kept = saved[2].contiguous(), dloss = grads[0].contiguous();
        const int64_t tokens = logits.size(0), experts = logits.size(1);
        const Rows r = flat_rows(logits, experts);
        const Tensor d = empty({tokens, experts}, logits, logits.scalar_type());
        const float *const stats = static_cast<const float *>(in(kept));
        call(logits, "msr_balance_grad", msr_balance_grad, in(r.t), r.ld, static_cast<const uint8_t *>(in(mask)), stats, stats + 2 * tokens,
             static_cast<const float *>(in(dloss)), tokens, (int32_t)experts, out(d), elem(logits));
        return once({d, Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor> balance_loss(const Tensor &logits, const Tensor &ids, const std::optional<Tensor> &mask_) {
    const Tensor mask = mask_.value_or(Tensor());
    one_gpu("balance_loss", logits, {&ids, &mask});
    TORCH_CHECK_VALUE(elem_ok(logits), "balance_loss: logits must be bf16 or fp32, got ", logits.scalar_type());
    TORCH_CHECK_VALUE(whole(ids), "balance_loss needs int32 or int64 ids, got ", ids.scalar_type());
    TORCH_CHECK_VALUE(logits.dim() == 2 && ids.dim() == 2 && ids.size(0) == logits.size(0) && ids.size(1) >= 1 && logits.size(1) >= 1 && logits.size(1) <= MSR_EXPERTS_MAX,
                      "balance_loss needs logits [tokens, experts] with 1 to ", MSR_EXPERTS_MAX, " experts and ids [tokens, k], got ", logits.sizes(), " and ", ids.sizes());
    TORCH_CHECK_VALUE(!mask.defined() || (mask.scalar_type() == at::kBool && mask.dim() == 1 && mask.size(0) == logits.size(0)), "balance_loss needs a bool mask of ",
                      logits.size(0), " tokens");
    const variable_list r = Balance::apply(logits, ids, mask_);
    return {r[0], r[1]};
}

}  // namespace

PYBIND11_MODULE(_nodes, m) {
    m.def("set_python", [](pybind11::object error_type, pybind11::object accumulator_) {
        library_error = error_type.release().ptr();
        accumulator = accumulator_.release().ptr();
    });
    m.def("layer_norm", torch::wrap_pybind_function(layer_norm));
    m.def("check_embedding", torch::wrap_pybind_function([](const std::string &what, const Tensor &ids, const Tensor &w, std::optional<int64_t> padding) { return check_embedding(what.c_str(), ids, w, padding); }));
    m.def("embedding", torch::wrap_pybind_function(embedding));
    m.def("linear_cross_entropy", torch::wrap_pybind_function(linear_cross_entropy));
    m.def("balance_loss", torch::wrap_pybind_function(balance_loss));
}
