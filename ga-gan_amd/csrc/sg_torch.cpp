// PyTorch side of the operators whose smallest calls are shorter than the host's work around them (fully connected layer,
// table lookup, clipped optimizer step): argument checks, allocation, autograd and the calls of the C ABI, without the
// interpreter in between.  A training step of one small layer spends its time on the host: with the same steps written in
// Python, a forward and backward call of a 32 x 512 x 512 layer took 172 us of which the kernels need 18; so it takes 40 to 68, of
// which autograd's change of threads is 10 to 34 (by where its thread runs).  The entry points themselves are the library's
// (include/sg_ops.h), resolved from the same file that ga_gan_amd._lib binds.
#include <dlfcn.h>

#include <atomic>
#include <memory>
#include <tuple>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/extension.h>

#include "sg_ops.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&::sg_last_error) last_error;
    decltype(&::sg_linear) linear;
    decltype(&::sg_linear_workspace_bytes) linear_workspace_bytes;
    decltype(&::sg_linear_backward) linear_backward;
    decltype(&::sg_linear_backward_workspace_bytes) linear_backward_workspace_bytes;
    decltype(&::sg_embedding) embedding;
    decltype(&::sg_embedding_backward) embedding_backward;
    decltype(&::sg_embedding_backward_workspace_bytes) embedding_backward_workspace_bytes;
    decltype(&::sg_grad_norm) grad_norm;
    decltype(&::sg_grad_norm_workspace_bytes) grad_norm_workspace_bytes;
    decltype(&::sg_scale_grads) scale_grads;
    decltype(&::sg_adam_step_list) adam_step_list;
} api;

void bind(const std::string& path) {
    void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(handle != nullptr, "cannot load ", path, ": ", dlerror());
    auto resolve = [&](auto& fn, const char* name) {
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(handle, name));
        TORCH_CHECK(fn != nullptr, path, " does not export ", name, ": rebuild it");
    };
    resolve(api.last_error, "sg_last_error");
    resolve(api.linear, "sg_linear");
    resolve(api.linear_workspace_bytes, "sg_linear_workspace_bytes");
    resolve(api.linear_backward, "sg_linear_backward");
    resolve(api.linear_backward_workspace_bytes, "sg_linear_backward_workspace_bytes");
    resolve(api.embedding, "sg_embedding");
    resolve(api.embedding_backward, "sg_embedding_backward");
    resolve(api.embedding_backward_workspace_bytes, "sg_embedding_backward_workspace_bytes");
    resolve(api.grad_norm, "sg_grad_norm");
    resolve(api.grad_norm_workspace_bytes, "sg_grad_norm_workspace_bytes");
    resolve(api.scale_grads, "sg_scale_grads");
    resolve(api.adam_step_list, "sg_adam_step_list");
}

// ---- launching ----------------------------------------------------------------------------------------------------------

// While launches are being recorded: recorder(label, bytes, flops, call).  A launch may come from a backward pass's thread, which does
// not hold the interpreter's lock, while another thread ends the recording: a launch keeps the object it saw until it is done
// with it, and whoever holds it last gives it up under the lock.  (Never destroyed itself: the interpreter may be gone by then.)
std::shared_ptr<py::object>& recorder = *new std::shared_ptr<py::object>;

void record(const py::object& callback) {
    std::shared_ptr<py::object> next;
    if (!callback.is_none())
        next = std::shared_ptr<py::object>(new py::object(callback), [](py::object* last) {
            py::gil_scoped_acquire gil;
            delete last;
        });
    std::atomic_store(&recorder, next);
}

// call(stream) on ref's device and the stream torch is enqueueing on there
template <class Call> void launch(const char* what, const char* label, double bytes, double flops, const Tensor& ref, Call call) {
    const c10::DeviceGuard guard(ref.device());
    void* stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(ref.device().index()).stream();
    int rc = 0;
    if (const auto recording = std::atomic_load(&recorder)) {
        py::gil_scoped_acquire gil;
        (*recording)(label, bytes, flops, py::cpp_function([&] { rc = call(stream); }));
    } else {
        rc = call(stream);
    }
    TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", api.last_error());
}

double nbytes(std::initializer_list<const Tensor*> tensors) {
    double sum = 0;
    for (const Tensor* t : tensors)
        if (t->defined()) sum += (double)t->nbytes();
    return sum;
}

void* ptr(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }

int dtype_code(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return SG_F32;
        case at::kHalf: return SG_F16;
        case at::kBFloat16: return SG_BF16;
        default: TORCH_CHECK(false, what, ": unsupported dtype ", t.scalar_type());
    }
}

// Whether t carries a tangent (forward-mode differentiation).  The functions below have no forward-mode derivative: a tensor that
// carries one goes through Function::apply, which refuses it, whether or not gradients are wanted.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

Tensor or_undefined(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// (t or a dense copy, elements between its rows): unit stride within a row, rows that do not overlap and that lie less than the
// 2^23 bytes apart that the library's 32-bit offsets within a tile allow
std::pair<Tensor, int64_t> rows_of(const Tensor& t) {
    const int64_t rows = t.size(0), cols = t.size(1);
    if ((cols <= 1 || t.stride(1) == 1) && (rows <= 1 || (t.stride(0) >= std::max<int64_t>(cols, 1) && t.stride(0) < (1 << 23) / (int64_t)t.element_size() - 1)))
        return {t, rows > 1 ? t.stride(0) : std::max<int64_t>(cols, 1)};
    return {t.contiguous(), std::max<int64_t>(cols, 1)};
}

// ---- fully connected layer ------------------------------------------------------------------------------------------------

enum Act { kLinear = 1, kRelu, kLrelu, kTanh, kSigmoid, kElu, kSelu, kSoftplus, kSwish };

struct LinearConfig {
    int64_t act;
    double alpha, gain, w_gain, b_gain;
};

sg_linear_params linear_params(const Tensor& x, int64_t ldx, const Tensor& w, int64_t ldw, const Tensor& b, const Tensor& residual, int64_t ldr,
                               const LinearConfig& c) {
    sg_linear_params p{};
    p.x = ptr(x); p.w = ptr(w); p.b = ptr(b); p.residual = ptr(residual);
    p.dtype = dtype_code(x, "linear");
    p.act = (int32_t)c.act;
    p.alpha = (float)c.alpha; p.gain = (float)c.gain; p.w_gain = (float)c.w_gain; p.b_gain = (float)c.b_gain;
    p.m = x.size(0); p.n = w.size(0); p.k = x.size(1);
    p.ldx = ldx; p.ldw = ldw; p.ldr = ldr;
    return p;
}

Tensor linear_forward(const Tensor& x_, const Tensor& w_, const Tensor& b_, const Tensor& residual_, const LinearConfig& c, Tensor* z, Tensor* positive) {
    const auto [x, ldx] = rows_of(x_);
    const auto [w, ldw] = rows_of(w_);
    const Tensor b = b_.defined() ? b_.contiguous() : b_;
    Tensor residual;
    int64_t ldr = 0;
    if (residual_.defined()) std::tie(residual, ldr) = rows_of(residual_);
    Tensor y = at::empty({x.size(0), w.size(0)}, x.options());
    if (z) *z = at::empty({x.size(0), w.size(0)}, x.options().dtype(at::kFloat));
    if (positive) *positive = at::empty({x.size(0), w.size(0)}, x.options().dtype(at::kByte));
    if (y.numel() == 0) return y;
    const sg_linear_params p = linear_params(x, ldx, w, ldw, b, residual, ldr, c);
    const size_t need = api.linear_workspace_bytes(&p);
    const Tensor work = workspace(need, x);
    launch("sg_linear", "linear_gemm_kernel", nbytes({&x, &w, &residual, &y}), 2.0 * p.m * p.n * p.k, x, [&](void* stream) {
        return api.linear(&p, ptr(y), z ? (float*)ptr(*z) : nullptr, positive ? (uint8_t*)ptr(*positive) : nullptr, ptr(work), need, stream);
    });
    return y;
}

// The layer from the framework's operators (differentiable to any order), in float32 whatever the operands' type: a z rounded to 16
// bits would choose other slopes than the forward pass did.  on: for relu and lrelu, where the forward pass had the slope of the
// positive side.
Tensor linear_composite(const Tensor& x_, const Tensor& w_, const Tensor& b_, const Tensor& on, const LinearConfig& c) {
    auto wide = [](const Tensor& t) { return t.defined() ? t.to(at::kFloat) : t; };
    const Tensor x = wide(x_), w = wide(w_), b = wide(b_);
    Tensor z = at::matmul(x, (c.w_gain != 1 ? w * c.w_gain : w).t());
    if (b.defined()) z = z + (c.b_gain != 1 ? b * c.b_gain : b);
    switch (c.act) {
        case kRelu: z = at::where(on, z, at::zeros_like(z)); break;
        case kLrelu: z = at::where(on, z, z * c.alpha); break;
        case kTanh: z = at::tanh(z); break;
        case kSigmoid: z = at::sigmoid(z); break;
        case kElu: z = at::elu(z); break;
        case kSelu: z = at::selu(z); break;
        case kSoftplus: z = at::softplus(z); break;
        case kSwish: z = at::silu(z); break;
        default: break;
    }
    return c.gain != 1 ? z * c.gain : z;
}

// What the backward pass keeps besides x and w: nothing for linear; for relu and lrelu the output itself, whose sign is the
// pre-activation's, or - where a residual, a gain that may take positive values to zero (float16: any), or a negative slope
// hides it - a byte per element; for the others the pre-activation values in float32 (rounded to 16 bits they would cost the
// gradient more accuracy than its own rounding does).
struct LinearFunction : torch::autograd::Function<LinearFunction> {
    enum Kept { kNothing, kY, kPositive, kZ };

    // (an absent tensor has no edge in the graph: the edges of those after it move up)
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const optional<Tensor>& b_, const optional<Tensor>& residual_,
                          const LinearConfig& c) {
        const Tensor b = or_undefined(b_), residual = or_undefined(residual_);
        const bool slopes = c.act != kLinear && (x.requires_grad() || w.requires_grad() || (b.defined() && b.requires_grad()));
        const bool by_sign = c.act == kRelu || c.act == kLrelu;
        const bool from_y = by_sign && !residual.defined() && x.scalar_type() != at::kHalf && std::abs(c.gain) >= 1.0 / 256 && (c.act == kRelu || c.alpha >= 0);
        const Kept kept = !slopes ? kNothing : from_y ? kY : by_sign ? kPositive : kZ;
        Tensor aux;
        Tensor y = linear_forward(x, w, b, residual, c, kept == kZ ? &aux : nullptr, kept == kPositive ? &aux : nullptr);
        if (kept == kY) aux = y;
        ctx->save_for_backward({x, w, b, aux});
        ctx->saved_data["config"] = std::vector<double>{(double)c.act, c.alpha, c.gain, c.w_gain, c.b_gain, (double)kept, (double)residual.defined()};
        ctx->set_materialize_grads(false);
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(5);
        Tensor dy = grads[0];
        if (!dy.defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x_ = saved[0], &w_ = saved[1], &b = saved[2], &aux = saved[3];
        const auto v = ctx->saved_data["config"].toDoubleVector();
        if (v[6] != 0 && ctx->needs_input_grad(b.defined() ? 3 : 2)) out[3] = dy;
        const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), b.defined() && ctx->needs_input_grad(2)};
        if (!need[0] && !need[1] && !need[2]) return out;
        TORCH_CHECK(!dual(dy), "linear: the backward pass has no forward-mode derivative");
        const LinearConfig c{(int64_t)v[0], v[1], v[2], v[3], v[4]};
        const int kept = (int)v[5];
        if (at::GradMode::is_enabled()) {                        // a graph of its own is wanted: differentiate the operators' version
            const c10::impl::ExcludeDispatchKeyGuard in_its_types(c10::autocast_dispatch_keyset);      // (the caller's autocast would round its products)
            variable_list in{x_.view_as(x_), w_.view_as(w_), b.defined() ? b.view_as(b) : b}, wanted;
            for (int i = 0; i < 3; i++)
                if (need[i]) wanted.push_back(in[i]);
            const Tensor on = kept == kY ? (c.gain < 0 ? aux < 0 : aux > 0) : kept == kPositive ? aux != 0 : Tensor();
            const variable_list got = torch::autograd::grad({linear_composite(in[0], in[1], in[2], on, c)}, wanted, {dy.to(at::kFloat)}, true, true);
            for (int i = 0, k = 0; i < 3; i++)
                if (need[i]) out[i] = got[k++];
            return out;
        }
        dy = dy.contiguous();
        // A linear layer's products read dy where it lies.  From 2^29 terms on the library copies operands that are not whole packets
        // (it plans before it sees dy's address): a dy that starts between packets is copied here, or both products would fall to
        // small tiles.  Gradients of 8192 x 2048 -> 2048 in bfloat16 360 us without, 141 with the copy; 10000 x 512 -> 512 in float32
        // 122 and 107; 1024^3 41 and 48, bound by the host.
        if (c.act == kLinear && reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 != 0 && (double)dy.numel() * x_.size(1) >= (double)(1 << 29)) dy = dy.clone();
        const auto [x, ldx] = rows_of(x_);
        const auto [w, ldw] = rows_of(w_);
        if (need[0]) out[0] = at::empty(x.sizes(), x.options());
        if (need[1]) out[1] = at::empty(w.sizes(), x.options());
        if (need[2]) out[2] = at::empty({w.size(0)}, x.options());
        const sg_linear_params p = linear_params(x, ldx, w, ldw, Tensor(), Tensor(), 0, c);
        const size_t bytes = api.linear_backward_workspace_bytes(&p);
        const Tensor work = workspace(bytes, x);
        launch("sg_linear_backward", "linear_gemm_kernel", nbytes({&dy, &x, &w, &out[0], &out[1]}), 2.0 * (need[0] + need[1]) * p.m * p.n * p.k, x,
               [&](void* stream) {
                   return api.linear_backward(&p, ptr(dy), kept == kY ? ptr(aux) : nullptr, kept == kZ ? (float*)ptr(aux) : nullptr,
                                              kept == kPositive ? (uint8_t*)ptr(aux) : nullptr, ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(work), bytes, stream);
               });
        return out;
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const optional<Tensor>& b_, const optional<Tensor>& residual_, int64_t act, double alpha, double gain,
              double w_gain, double b_gain) {
    const Tensor b = or_undefined(b_), residual = or_undefined(residual_);
    TORCH_CHECK(x.is_cuda(), "linear: x must be a GPU tensor (this op runs on the GPU only)");
    dtype_code(x, "linear");
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1), "linear: x ", x.sizes(), " and w ", w.sizes(), " do not match");
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w.size(0);
    TORCH_CHECK(!b.defined() || (b.dim() == 1 && b.size(0) == w.size(0)), "linear: b ", b_.value_or(w).sizes(), " must have one entry per row of w ", w.sizes());
    TORCH_CHECK(!residual.defined() || residual.sizes() == at::IntArrayRef(shape), "linear: residual ", residual_.value_or(w).sizes(),
                " must have the shape of the output ", at::IntArrayRef(shape));
    for (const Tensor* t : {&w, &b, &residual})
        TORCH_CHECK(!t->defined() || (t->scalar_type() == x.scalar_type() && t->device() == x.device()),
                    "linear: w, b and residual must have the dtype and device of x");
    const LinearConfig c{act, alpha, gain, w_gain, b_gain};
    const bool flat = x.dim() == 2;
    int64_t m = 1;
    for (size_t i = 0; i + 1 < shape.size(); i++) m *= shape[i];
    const Tensor x2 = flat ? x : x.reshape({m, x.size(-1)}), r2 = flat || !residual.defined() ? residual : residual.reshape({m, w.size(0)});
    const bool graph = at::GradMode::is_enabled() &&
                       (x.requires_grad() || w.requires_grad() || (b.defined() && b.requires_grad()) || (residual.defined() && residual.requires_grad()));
    const bool refused = dual(x) || dual(w) || dual(b) || dual(residual);
    const Tensor y = graph || refused ? LinearFunction::apply(x2, w, b_, r2.defined() ? optional<Tensor>(r2) : c10::nullopt, c) : linear_forward(x2, w, b, r2, c, nullptr, nullptr);
    return flat ? y : y.reshape(shape);
}

// ---- table lookup -----------------------------------------------------------------------------------------------------------

sg_embedding_params embedding_params(const Tensor& index, const Tensor& table, const Tensor& bias, double w_gain, double b_gain) {
    sg_embedding_params p{};
    p.index = ptr(index); p.table = ptr(table); p.bias = ptr(bias);
    p.dtype = dtype_code(table, "embedding");
    p.index_bytes = (int32_t)index.element_size();
    p.tokens = index.numel(); p.v = table.size(0); p.f = table.size(1);
    p.stride_v = table.stride(0); p.stride_f = table.stride(1);
    p.w_gain = (float)w_gain; p.b_gain = (float)b_gain;
    return p;
}

Tensor lookup(const Tensor& index, const Tensor& table, const Tensor& b_, double w_gain, double b_gain) {
    Tensor y = at::empty({index.numel(), table.size(1)}, table.options());
    if (y.numel() == 0) return y;
    const Tensor b = b_.defined() ? b_.contiguous() : b_;
    const sg_embedding_params p = embedding_params(index, table, b, w_gain, b_gain);
    launch("sg_embedding", "embedding_kernel", 2 * nbytes({&y}), 0, table, [&](void* stream) { return api.embedding(&p, ptr(y), stream); });
    return y;
}

// The lookup and its gradient are each other's gradients.
struct EmbeddingGradFunction : torch::autograd::Function<EmbeddingGradFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& dy, const Tensor& index, int64_t v, int64_t f, bool by_columns, double w_gain,
                                 double b_gain, bool want_bias) {
        ctx->save_for_backward({index});
        ctx->saved_data["gains"] = std::vector<double>{w_gain, b_gain};
        ctx->set_materialize_grads(false);
        return run(dy.contiguous(), index, v, f, by_columns, w_gain, b_gain, want_bias);
    }
    static variable_list run(const Tensor& dy, const Tensor& index, int64_t v, int64_t f, bool by_columns, double w_gain, double b_gain, bool want_bias) {
        Tensor dtable = by_columns ? at::empty({f, v}, dy.options()).t() : at::empty({v, f}, dy.options()), dbias;
        if (want_bias) dbias = at::empty({f}, dy.options());
        if (dtable.numel()) {
            sg_embedding_params p = embedding_params(index, dtable, Tensor(), w_gain, b_gain);
            p.stride_v = by_columns ? 1 : f;                     // (strides of a one-row or one-column table are not torch's to give)
            p.stride_f = by_columns ? v : 1;
            const size_t need = api.embedding_backward_workspace_bytes(&p);
            const Tensor work = workspace(need, dy);
            launch("sg_embedding_backward", "embedding_grad_runs_kernel", nbytes({&dy, &dtable}), 0, dy,
                   [&](void* stream) { return api.embedding_backward(&p, ptr(dy), ptr(dbias), ptr(work), need, stream); });
        }
        return want_bias ? variable_list{dtable, dbias} : variable_list{dtable};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads);
};

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const optional<Tensor>& b, const Tensor& index, double w_gain, double b_gain) {
        ctx->save_for_backward({index});
        const bool by_columns = table.stride(1) != 1 && table.stride(0) == 1;
        ctx->saved_data["shape"] = std::vector<int64_t>{table.size(0), table.size(1), by_columns, b.has_value()};
        ctx->saved_data["gains"] = std::vector<double>{w_gain, b_gain};
        ctx->set_materialize_grads(false);
        return lookup(index, table, or_undefined(b), w_gain, b_gain);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const Tensor index = ctx->get_saved_variables()[0];
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const auto gains = ctx->saved_data["gains"].toDoubleVector();
        const bool want_bias = shape[3] != 0 && ctx->needs_input_grad(1);
        const variable_list got = at::GradMode::is_enabled() || dual(grads[0])
            ? EmbeddingGradFunction::apply(grads[0], index, shape[0], shape[1], shape[2] != 0, gains[0], gains[1], want_bias)
            : EmbeddingGradFunction::run(grads[0].contiguous(), index, shape[0], shape[1], shape[2] != 0, gains[0], gains[1], want_bias);
        if (ctx->needs_input_grad(0)) out[0] = got[0];
        if (want_bias) out[1] = got[1];
        return out;
    }
};

Tensor embedding(const Tensor& index, const Tensor& table, const optional<Tensor>& b_, double w_gain, double b_gain) {
    const Tensor b = or_undefined(b_);
    TORCH_CHECK(table.is_cuda(), "embedding: table must be a GPU tensor (this op runs on the GPU only)");
    dtype_code(table, "embedding");
    TORCH_CHECK(index.scalar_type() == at::kInt || index.scalar_type() == at::kLong, "embedding: indices must be int32 or int64, not ", index.scalar_type());
    TORCH_CHECK(table.dim() == 2 && table.size(0) >= 1, "embedding: table ", table.sizes(), " must be [V, F] with at least one row");
    TORCH_CHECK(index.device() == table.device() && (!b.defined() || (b.device() == table.device() && b.scalar_type() == table.scalar_type())),
                "embedding: index and b must be on the device of the table, b of its dtype");
    TORCH_CHECK(!b.defined() || (b.dim() == 1 && b.size(0) == table.size(1)), "embedding: b ", b_.value_or(table).sizes(),
                " must have one entry per column of the table ", table.sizes());
    const Tensor flat = index.reshape({-1}).contiguous();
    const bool graph = at::GradMode::is_enabled() && (table.requires_grad() || (b.defined() && b.requires_grad()));
    const Tensor y = graph || dual(table) || dual(b) ? EmbeddingFunction::apply(table, b_, flat, w_gain, b_gain) : lookup(flat, table, b, w_gain, b_gain);
    if (index.dim() == 1) return y;
    std::vector<int64_t> shape = index.sizes().vec();
    shape.push_back(table.size(1));
    return y.reshape(shape);
}

variable_list EmbeddingGradFunction::backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(8);
    const Tensor index = ctx->get_saved_variables()[0];
    const auto gains = ctx->saved_data["gains"].toDoubleVector();
    const Tensor ddbias = grads.size() > 1 ? grads[1] : Tensor();
    const Tensor from_bias = ddbias.defined() ? (ddbias * gains[1]).expand({index.numel(), ddbias.size(0)}) : Tensor();
    out[0] = from_bias;
    if (grads[0].defined()) {
        // (a token outside the table added to no row: its dy has no part in the rows' gradient, where a lookup would read NaN)
        const Tensor rows = embedding(index, grads[0], ddbias.defined() ? optional<Tensor>(ddbias) : c10::nullopt, gains[0], gains[1]);
        const Tensor inside = at::logical_and(index >= 0, index < grads[0].size(0)).unsqueeze(1);
        out[0] = at::where(inside, rows, from_bias.defined() ? from_bias : at::zeros_like(rows));
    }
    return out;
}

// ---- gradient norm, clipping, optimizer step ----------------------------------------------------------------------------------

// Host arrays of a list of gradients (kept alive while the library reads them).
struct GradList {
    std::vector<void*> pointers;
    std::vector<int64_t> numels;
    std::vector<int32_t> dtypes;
    sg_grad_list args;
    double bytes = 0;

    GradList(const std::vector<Tensor>& grads, const char* what) {
        for (const Tensor& g : grads) {
            dtypes.push_back(dtype_code(g, what));
            TORCH_CHECK(g.is_cuda() && g.device() == grads[0].device(), what, ": gradients must reside on one CUDA device");
            TORCH_CHECK(g.is_contiguous(), what, ": gradients must be dense");
            pointers.push_back(ptr(g));
            numels.push_back(g.numel());
            bytes += (double)g.nbytes();
        }
        args = {pointers.data(), numels.data(), dtypes.data(), (int32_t)grads.size()};
    }
};

void distinct(std::vector<void*> pointers, const char* what) {
    std::sort(pointers.begin(), pointers.end());
    for (size_t i = 1; i < pointers.size(); i++)
        TORCH_CHECK(pointers[i] == nullptr || pointers[i] != pointers[i - 1], what, ": a tensor appears twice");
}

// float32 [2]: the norm, and min(1, max_norm / (norm + eps))
Tensor norm_and_scale(const GradList& list, const Tensor& first, double grad_limit, double max_norm, double eps) {
    const size_t need = api.grad_norm_workspace_bytes(&list.args);
    const Tensor out = at::empty({2}, first.options().dtype(at::kFloat));
    const Tensor work = workspace(need, first);
    launch("sg_grad_norm", "grad_norm_kernel", list.bytes, 0, out, [&](void* stream) {
        return api.grad_norm(&list.args, (float)grad_limit, (float)max_norm, (float)eps, (float*)ptr(out), ptr(work), need, stream);
    });
    return out;
}

Tensor grad_norm(const std::vector<Tensor>& grads, double grad_limit, double max_norm, double eps) {
    const GradList list(grads, "grad_norm");
    return norm_and_scale(list, grads.at(0), grad_limit, max_norm, eps);
}

Tensor clip_grads(const std::vector<Tensor>& grads, double max_norm, double eps) {
    const GradList list(grads, "clip_grad_norm_");
    distinct(list.pointers, "clip_grad_norm_");
    const Tensor out = norm_and_scale(list, grads.at(0), 0, max_norm, eps);
    launch("sg_scale_grads", "grad_scale_kernel", 2 * list.bytes, 0, out,
           [&](void* stream) { return api.scale_grads(&list.args, (const float*)ptr(out) + 1, stream); });
    for (const Tensor& g : grads) g.unsafeGetTensorImpl()->bump_version();
    return out.select(0, 0);
}

// One group of an optimizer's tensors, checked, as the library takes it (the vectors are what args points into).
struct AdamGroup {
    std::vector<void*> pointers;
    std::vector<int64_t> numels;
    std::vector<int32_t> counts;
    sg_adam_list args{};
    double bytes = 0;

    AdamGroup(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& exp_avgs, const std::vector<Tensor>& exp_avg_sqs,
              const std::vector<int64_t>& steps, double lr, double beta1, double beta2, double eps, double grad_limit) {
        const size_t count = params.size();
        TORCH_CHECK(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count && steps.size() == count,
                    "adam_step: lists differ in length");
        const std::vector<Tensor>* lists[4] = {&params, &grads, &exp_avgs, &exp_avg_sqs};
        static const char* const names[4] = {"param", "grad", "exp_avg", "exp_avg_sq"};
        pointers.resize(4 * count);
        numels.resize(count);
        counts.resize(count);
        for (size_t i = 0; i < count; i++) {
            const c10::Device device = params[i].device();
            numels[i] = params[i].numel();
            counts[i] = (int32_t)std::min<int64_t>(steps[i], INT32_MAX);
            bytes += 32.0 * numels[i];
            for (int k = 0; k < 4; k++) {
                const Tensor& t = (*lists[k])[i];
                TORCH_CHECK(t.is_cuda() && t.device() == device, names[k], " must reside on CUDA device ", device);
                TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous(), names[k], " must be a dense float32 tensor");
                TORCH_CHECK(t.sizes() == params[i].sizes(), "adam_step: ", names[k], " ", t.sizes(), " does not match its parameter ", params[i].sizes());
                pointers[k * count + i] = ptr(t);
            }
            TORCH_CHECK(steps[i] >= 1, "adam_step: tensor ", i, ": step ", steps[i]);
        }
        args.lr = (float)lr; args.beta1 = (float)beta1; args.beta2 = (float)beta2; args.eps = (float)eps; args.grad_limit = (float)grad_limit;
        TORCH_CHECK(args.beta1 >= 0 && args.beta1 < 1 && args.beta2 >= 0 && args.beta2 < 1 && args.eps >= 0 && args.grad_limit > 0,
                    "adam_step: betas must lie in [0, 1), eps >= 0, grad_limit > 0");
        float* const* base = reinterpret_cast<float* const*>(pointers.data());
        args.param = base; args.grad = base + count; args.exp_avg = base + 2 * count; args.exp_avg_sq = base + 3 * count;
        args.numel = numels.data(); args.step = counts.data();
        args.count = (int32_t)count;
    }
    AdamGroup(const AdamGroup&) = delete;
};

using AdamArgs = std::tuple<std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, std::vector<int64_t>, double, double, double, double, double>;

std::vector<std::unique_ptr<AdamGroup>> checked(const std::vector<AdamArgs>& groups) {
    std::vector<std::unique_ptr<AdamGroup>> found;
    for (const AdamArgs& g : groups)
        found.push_back(std::apply([](const auto&... a) { return std::make_unique<AdamGroup>(a...); }, g));
    return found;
}

// Whether a step of these groups would be refused: raises what it would raise, and launches nothing.
void adam_check(const std::vector<AdamArgs>& groups) { checked(groups); }

// One step of all groups (each: params, grads, exp_avgs, exp_avg_sqs, steps, lr, beta1, beta2, eps, grad_limit), clipped by the norm of all
// their sanitised gradients, which it returns.  Everything is checked before anything is launched.
Tensor adam_step_clipped(const std::vector<AdamArgs>& groups, double max_norm, double norm_eps) {
    const auto found = checked(groups);
    std::vector<Tensor> grads;
    std::vector<void*> pointers;
    for (size_t i = 0; i < groups.size(); i++) {
        const auto& of_group = std::get<1>(groups[i]);
        grads.insert(grads.end(), of_group.begin(), of_group.end());
        pointers.insert(pointers.end(), found[i]->pointers.begin(), found[i]->pointers.end());
        TORCH_CHECK(found[i]->args.grad_limit == found[0]->args.grad_limit, "adam_step: groups that are clipped together must share grad_limit");
    }
    TORCH_CHECK(!grads.empty(), "adam_step: no tensors");
    distinct(pointers, "adam_step");
    const GradList list(grads, "adam_step");
    const Tensor out = norm_and_scale(list, grads[0], found[0]->args.grad_limit, max_norm, norm_eps);
    for (size_t i = 0; i < groups.size(); i++) {
        AdamGroup& group = *found[i];
        if (group.args.count == 0) continue;
        group.args.grad_scale = (const float*)ptr(out) + 1;
        launch("sg_adam_step_list", "adam_kernel", group.bytes, 0, grads[0], [&](void* stream) { return api.adam_step_list(&group.args, stream); });
        for (const auto* tensors : {&std::get<0>(groups[i]), &std::get<1>(groups[i]), &std::get<2>(groups[i]), &std::get<3>(groups[i])})
            for (const Tensor& t : *tensors) t.unsafeGetTensorImpl()->bump_version();
    }
    return out.select(0, 0);
}

}  // namespace

PYBIND11_MODULE(_sg_torch, m) {
    m.def("bind", &bind);
    m.def("record", &record);
    m.def("linear", &linear);
    m.def("embedding", &embedding);
    m.def("grad_norm", &grad_norm);
    m.def("clip_grads", &clip_grads);
    m.def("adam_check", &adam_check);
    m.def("adam_step_clipped", &adam_step_clipped);
}
