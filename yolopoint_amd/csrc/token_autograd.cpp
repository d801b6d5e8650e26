// The host side of the token operators (yolopoint_amd/utils/token_ops.py): argument checks, buffers, launches through the C ABI and the autograd nodes.
// In C++ because these operators take microseconds: autograd runs a backward pass on a thread of its own, where every Python statement waits for cold
// caches and the interpreter's lock (a layer norm's forward + backward on 64 x 256 cost the host 166 us as a Python autograd function).
// The entry points come as addresses from the ctypes binding (init), so that this module serves whichever build of the library is loaded.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <cstdarg>
#include <optional>
#include "../../include/yolopoint_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

// ---------------------------------------------------------------------------------------------------------------- errors, entry points
struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };     // becomes yolopoint_amd._hip.YpError in Python

[[noreturn]] void fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
void fail(const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    throw Refused(text);
}

struct Entry {
    decltype(&yp_last_error) last_error;
    decltype(&yp_layer_norm_fwd) norm_fwd;
    decltype(&yp_layer_norm_bwd) norm_bwd;
    decltype(&yp_layer_norm_bwd_workspace_bytes) norm_workspace;
    decltype(&yp_layer_norm_max_width) norm_max_width;
    decltype(&yp_dropout) dropout;
    decltype(&yp_rotary) rotary;
} lib{};
PyObject* yp_error = nullptr;

void check(int rc) {
    if (rc != 0) fail("libyolopoint_hip error %d: %s", rc, lib.last_error());
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int type_code(at::ScalarType t) { return t == at::kHalf ? YP_F16 : t == at::kBFloat16 ? YP_BF16 : t == at::kFloat ? YP_F32 : -1; }

std::string shape_of(const Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

// A tracer sees the buffers that a call allocates and not the kernels that fill them: what it recorded would return memory as it was found.  (Other
// dispatch modes -- counters, checkpointing -- run the call as it is and may stay.)
void check_untraced(const char* what) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    bool traced = torch::jit::tracer::isTracing();
    if (!traced && Modes::any_modes_set())
        for (int i = 0; i < (int)c10::impl::TorchDispatchModeKey::NUM_MODE_KEYS; ++i) traced |= Modes::get_mode((c10::impl::TorchDispatchModeKey)i).has_value();
    if (traced) fail("%s: cannot be traced (torch.jit.trace, make_fx, fake tensors): its kernels are launched, not dispatched", what);
}

// A tensor with elements has memory: the entry points take a missing address for an operand that was not given, so tensors without storage of their own
// (sharded parameters and other wrappers, fake tensors) must not reach them.  (Tensors that torch knows to be zero are written out where they are read.)
bool has_memory(const Tensor& t) {
    if (t.numel() == 0 || t._is_zerotensor()) return true;
    if (!t.has_storage()) return false;
    try {
        return t.const_data_ptr() != nullptr;
    } catch (const c10::Error&) {
        return false;
    }
}
void check_memory(const char* what, const Tensor& t) {
    if (!has_memory(t)) fail("%s: a tensor of shape %s holds no memory of its own (a wrapper: pass what it wraps)", what, shape_of(t).c_str());
}

void check_tensor(const char* what, const Tensor& x) {
    check_untraced(what);
    if (!x.defined() || !x.is_cuda()) fail("%s: a tensor on the GPU is needed (there is no CPU path)", what);
    if (x.layout() != at::kStrided || type_code(x.scalar_type()) < 0) fail("%s: a dense tensor of float16, bfloat16 or float32, not %s", what, toString(x.scalar_type()));
    check_memory(what, x);
    if (x._fw_grad(0).defined()) fail("%s: forward-mode differentiation is not offered", what);
}
void check_beside(const char* what, const Tensor& x, const MaybeTensor& o) {
    if (o && (o->device() != x.device() || o->layout() != at::kStrided)) fail("%s: all tensors dense and on %s", what, x.device().str().c_str());
    if (o) check_memory(what, *o);
    if (o && o->is_floating_point() && o->_fw_grad(0).defined()) fail("%s: forward-mode differentiation is not offered", what);
}

bool wants(const MaybeTensor& t) { return t && t->requires_grad(); }
Tensor given(const MaybeTensor& t) { return t ? *t : Tensor(); }

// the address of an operand: null for one that was not given, and for no other that has elements
void* address(const Tensor& t) {
    if (!t.defined() || t.numel() == 0) return nullptr;
    void* p = t.has_storage() ? t.data_ptr() : nullptr;
    if (p == nullptr) fail("a token operator was given a tensor of shape %s without memory", shape_of(t).c_str());
    return p;
}

// gradients of gradients are refused when they are asked for, as by once_differentiable
variable_list once(variable_list&& grads) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    auto error = std::make_shared<torch::autograd::DelayedError>("a token operator's gradient is differentiable once", (int64_t)grads.size());
    variable_list as_inputs;
    for (auto& g : grads) as_inputs.push_back(g.defined() ? g.detach().requires_grad_() : g);
    return (*error)(std::move(as_inputs));
}

// ---------------------------------------------------------------------------------------------------------------- rows
// t with its values in memory: a copy of a view that is negated when it is read (the imaginary part of a conjugate is), and of one that is known to be zero
Tensor plain(const Tensor& t) { return t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg(); }

// t as it lies if it is dense, else a dense copy
Tensor dense(const Tensor& t) { return t.defined() ? plain(t).contiguous() : t; }

// x with rows of one distance where they lie, anything else through a dense copy
struct Rows { Tensor t; int64_t stride; };
Rows rows_of(const Tensor& t) {
    const Tensor x = plain(t);
    const int64_t D = x.size(-1);
    if (x.is_contiguous()) return {x, D};
    if (D == 1 || x.stride(-1) == 1) {
        int64_t step = -1, size = 1;
        bool one = true;
        for (int64_t i = x.dim() - 2; i >= 0 && one; --i) {
            if (x.size(i) == 1) continue;
            if (step < 0) step = x.stride(i);
            else if (x.stride(i) != step * size) one = false;
            size *= x.size(i);
        }
        if (one) return {x, step < 0 ? D : step};
    }
    return {x.contiguous(), D};
}

// ---------------------------------------------------------------------------------------------------------------- layer norm
struct Dropping {
    double p = 0.0;
    uint64_t seed = 0, offset = 0;
    bool any() const { return p * 65536.0 + 0.5 >= 1.0; }  // (the applied rate, in steps of 2^-16)
};

void check_norm(const char* what, const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps) {
    const int widest = lib.norm_max_width(type_code(x.scalar_type()));
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > widest) fail("%s: the last dimension has 1 to %d features, not %s", what, widest, shape_of(x).c_str());
    for (const MaybeTensor* t : {&w, &b}) {
        if (!*t) continue;
        check_beside(what, x, *t);
        if ((*t)->dim() != 1 || (*t)->size(0) != x.size(-1) || ((*t)->scalar_type() != at::kFloat && (*t)->scalar_type() != x.scalar_type()))
            fail("%s: weight and bias [%lld] in float32 or the tokens' type, not %s in %s", what, (long long)x.size(-1), shape_of(**t).c_str(), toString((*t)->scalar_type()));
    }
    if (w && b && w->scalar_type() != b->scalar_type()) fail("%s: weight and bias of one type", what);
    if (!(eps >= 0.0)) fail("%s: eps %g", what, eps);
}

void check_drop(const char* what, const Tensor& x, double p, const MaybeTensor& rng) {
    if (!(p >= 0.0 && p <= 1.0)) fail("%s: a rate of 0 to 1, not %g", what, p);
    if (rng && (rng->scalar_type() != at::kLong || rng->dim() != 1 || rng->size(0) != 2 || !rng->is_contiguous() || rng->is_neg() || rng->device() != x.device() || !has_memory(*rng)))
        fail("%s: rng as a tensor is int64 [seed, offset] on %s", what, x.device().str().c_str());
}

at::ScalarType weight_type(const Tensor& w, const Tensor& b) { return w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat; }

struct NormResult { Tensor y, z, stats; };                 // stats: fp32 [rows, 3], mean | 1 / deviation | what the mean's nearest fp32 number leaves

NormResult norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, double eps, const Dropping& drop, const Tensor& rng, bool keep) {
    const int64_t D = x.size(-1), rows = x.numel() / D;
    const Rows xr = rows_of(x);
    const Tensor w = dense(weight), b = dense(bias);
    NormResult r;
    r.y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    YpLayerNormDesc d{};
    Rows rr;
    if (residual.defined()) {
        rr = rows_of(residual);
        r.z = at::empty(x.sizes(), r.y.options());
        d.res = address(rr.t);
        d.res_stride = rr.stride;
        d.z = r.z.data_ptr();
    }
    if (keep) {
        r.stats = at::empty({rows, 3}, x.options().dtype(at::kFloat));
        d.stats = (float*)address(r.stats);
    }
    d.x = address(xr.t);
    d.x_stride = xr.stride;
    d.y = r.y.data_ptr();
    d.weight = address(w);
    d.bias = address(b);
    d.rows = rows;
    d.D = (int32_t)D;
    d.eps = (float)eps;
    d.dtype = type_code(x.scalar_type());
    d.wdtype = type_code(weight_type(w, b));
    d.p = drop.p;
    d.seed = drop.seed;
    d.offset = drop.offset;
    d.rng = (const int64_t*)address(rng);
    check(lib.norm_fwd(&d, stream_of(x)));
    return r;
}

Tensor drop_launch(const Tensor& x, const Tensor& residual, const Dropping& drop, const Tensor& rng) {
    const Tensor xc = dense(x), rc = dense(residual);
    Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    check(lib.dropout(address(xc), address(rc), y.data_ptr(), x.numel(), type_code(x.scalar_type()), drop.p, drop.seed, drop.offset, (const int64_t*)address(rng), stream_of(x)));
    return y;
}

struct NormBackward : Node {
    SavedVariable z, weight, stats, rng;                   // z: what was normalised (the input itself without a residual)
    Dropping drop;
    at::ScalarType wtype = at::kFloat;
    bool fused = false;

    std::string name() const override { return fused ? "DropoutAddLayerNormBackward" : "LayerNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        z.reset_data();
        weight.reset_data();
        stats.reset_data();
        rng.reset_data();
    }
    // gradients of (x, weight, bias), or of (x, residual, weight, bias)
    variable_list apply(variable_list&& in) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const int n = fused ? 4 : 3;
        variable_list out(n);
        check_untraced(fused ? "dropout_add_layer_norm's gradient" : "layer_norm's gradient");
        Tensor dy = in[0], dz = fused ? in[1] : Tensor();
        if (!dy.defined() && !dz.defined()) return out;
        const Tensor z_ = z.unpack(shared_from_this()), w_ = weight.unpack(), stats_ = stats.unpack(), rng_ = rng.unpack();
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(z_.device());
            const bool drops = drop.any(), need_x = task_should_compute_output(0), need_res = fused && task_should_compute_output(1);
            const bool need_w = task_should_compute_output(n - 2), need_b = task_should_compute_output(n - 1);
            const auto options = z_.options().memory_format(at::MemoryFormat::Contiguous);
            if (!dy.defined()) {                           // y was not used: the gradient of z goes on to its parts
                if (need_res) out[1] = dz;
                if (need_x) out[0] = drops ? drop_launch(dz, Tensor(), drop, rng_) : dz;
                if (need_w) out[n - 2] = at::zeros({z_.size(-1)}, options.dtype(wtype));
                if (need_b) out[n - 1] = at::zeros({z_.size(-1)}, options.dtype(wtype));
                return once(std::move(out));
            }
            const int64_t D = z_.size(-1), rows = z_.numel() / D;
            const Rows zr = rows_of(z_), dyr = rows_of(dy);
            Rows dzr;
            const Tensor w = dense(w_);
            Tensor dres, dx, dw, db, ws;
            YpLayerNormDesc d{};
            // (the branch's gradient is another tensor than the residual's only where elements were dropped; rows that no one asked for are not written)
            const bool rows_wanted = need_res || need_x;
            if (rows_wanted) { dres = at::empty(z_.sizes(), options); d.dres = address(dres); }
            if (need_x && drops) { dx = at::empty(z_.sizes(), options); d.dx = address(dx); }
            if (need_w) dw = at::empty({D}, options.dtype(wtype));
            if (need_b) db = at::empty({D}, options.dtype(wtype));
            if (!rows_wanted) dz = Tensor();
            if (dw.defined() || db.defined()) {            // (a workspace of its own in every call: streams and captured graphs share none)
                d.workspace_bytes = lib.norm_workspace(rows, (int)D, type_code(z_.scalar_type()));
                ws = at::empty({(int64_t)d.workspace_bytes}, options.dtype(at::kByte));
                d.workspace = ws.data_ptr();
            }
            if (dz.defined()) { dzr = rows_of(dz); d.dz = address(dzr.t); d.dz_stride = dzr.stride; }
            d.x = address(zr.t);
            d.x_stride = zr.stride;
            d.dy = address(dyr.t);
            d.dy_stride = dyr.stride;
            d.stats = (float*)address(stats_);
            d.weight = address(w);
            d.dweight = address(dw);
            d.dbias = address(db);
            d.rows = rows;
            d.D = (int32_t)D;
            d.dtype = type_code(z_.scalar_type());
            d.wdtype = type_code(wtype);
            if (dx.defined()) {
                d.p = drop.p;
                d.seed = drop.seed;
                d.offset = drop.offset;
                d.rng = (const int64_t*)address(rng_);
            }
            check(lib.norm_bwd(&d, stream_of(z_)));
            if (need_x) out[0] = drops ? dx : dres;
            if (need_res) out[1] = dres;
            out[n - 2] = dw;
            out[n - 1] = db;
        }
        return once(std::move(out));
    }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
    check_tensor("layer_norm", x);
    check_norm("layer_norm", x, weight, bias, eps);
    const c10::DeviceGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || wants(weight) || wants(bias));
    const Tensor w = given(weight), b = given(bias);
    NormResult r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = norm_forward(x, Tensor(), w, b, eps, Dropping(), Tensor(), grad);
    }
    if (grad) {
        std::shared_ptr<NormBackward> node(new NormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
        node->z = SavedVariable(x, false);
        node->weight = SavedVariable(w, false);
        node->stats = SavedVariable(r.stats, false);
        node->wtype = weight_type(w, b);
        torch::autograd::set_history(r.y, node);
    }
    return r.y;
}

std::tuple<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, const MaybeTensor& bias, double p, uint64_t seed,
                                                  uint64_t offset, const MaybeTensor& rng, double eps) {
    const char* what = "dropout_add_layer_norm";
    check_tensor(what, x);
    check_beside(what, x, residual);
    if (!residual || residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type()) fail("%s: residual of x's shape and type", what);
    check_norm(what, x, weight, bias, eps);
    check_drop(what, x, p, rng);
    const c10::DeviceGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || residual->requires_grad() || wants(weight) || wants(bias));
    const Tensor w = given(weight), b = given(bias), state = given(rng);
    const Dropping drop{p, seed, offset};
    NormResult r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = norm_forward(x, *residual, w, b, eps, drop, state, grad);
    }
    if (grad) {
        std::shared_ptr<NormBackward> node(new NormBackward(), torch::autograd::deleteNode);
        node->fused = true;
        node->set_next_edges(torch::autograd::collect_next_edges(x, *residual, w, b));
        node->drop = drop;
        node->wtype = weight_type(w, b);
        torch::autograd::set_history(r.y, node);
        torch::autograd::set_history(r.z, node);
        node->z = SavedVariable(r.z, true);
        node->weight = SavedVariable(w, false);
        node->stats = SavedVariable(r.stats, false);
        if (drop.any()) node->rng = SavedVariable(state, false);     // (a state that is not read may move on)
    }
    return {r.y, r.z};
}

// ---------------------------------------------------------------------------------------------------------------- dropout
struct DropoutBackward : Node {
    SavedVariable rng;
    Dropping drop;

    std::string name() const override { return "DropoutBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        rng.reset_data();
    }
    variable_list apply(variable_list&& in) override {     // gradients of (x, residual)
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(2);
        check_untraced("dropout's gradient");
        const Tensor dy = in[0];
        if (!dy.defined()) return out;
        const Tensor rng_ = rng.unpack();
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(dy.device());
            if (task_should_compute_output(0)) out[0] = drop_launch(dy, Tensor(), drop, rng_);
            if (task_should_compute_output(1)) out[1] = dy;
        }
        return once(std::move(out));
    }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const MaybeTensor& rng, const MaybeTensor& residual) {
    check_tensor("dropout", x);
    check_beside("dropout", x, residual);
    if (residual && (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type())) fail("dropout: residual of x's shape and type");
    check_drop("dropout", x, p, rng);
    const c10::DeviceGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || wants(residual));
    const Tensor r = given(residual), state = given(rng);
    const Dropping drop{p, seed, offset};
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = drop_launch(x, r, drop, state);
    }
    if (grad) {
        std::shared_ptr<DropoutBackward> node(new DropoutBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, r));
        node->drop = drop;
        if (drop.any()) node->rng = SavedVariable(state, false);
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------------------------------------------------------- rotary positions
struct Turn {
    int64_t start = 0;
    bool interleaved = false, heads_first = false;
    int axes = 1;
    double scale = 1.0;
};

int64_t batch_of(const Tensor& x) { return x.size(0); }
int64_t tokens_of(const Tensor& x, bool heads_first) { return x.size(heads_first ? 2 : 1); }
int64_t heads_of(const Tensor& x, bool heads_first) { return x.size(heads_first ? 1 : 2); }
void strides_of(const Tensor& x, bool heads_first, int64_t (&s)[3]) {
    s[0] = x.stride(0);
    s[1] = x.stride(heads_first ? 2 : 1);
    s[2] = x.stride(heads_first ? 1 : 2);
}

void turn_launch(const Tensor& q, const Tensor& k, const Tensor& q_out, const Tensor& k_out, const Tensor& positions, const Tensor& inv_freq, const Turn& how, bool inverse) {
    YpRotaryDesc d{};
    const bool hf = how.heads_first;
    d.q = address(q);
    d.q_out = q_out.data_ptr();
    strides_of(q, hf, d.q_stride);
    strides_of(q_out, hf, d.q_out_stride);
    d.B = (int32_t)batch_of(q);
    d.T = (int32_t)tokens_of(q, hf);
    d.Hq = (int32_t)heads_of(q, hf);
    if (k.defined()) {
        d.k = address(k);
        d.k_out = k_out.data_ptr();
        strides_of(k, hf, d.k_stride);
        strides_of(k_out, hf, d.k_out_stride);
        d.Hk = (int32_t)heads_of(k, hf);
    }
    d.D = (int32_t)q.size(3);
    d.R = 2 * (int32_t)inv_freq.numel();
    d.inv_freq = (const double*)address(inv_freq);
    if (positions.defined()) {
        const int64_t n = positions.dim() - (how.axes == 2 ? 1 : 0);        // [T] or [B, T], behind it the axes
        d.positions = address(positions);
        d.position_type = positions.scalar_type() == at::kLong ? YP_POS_I64 : positions.scalar_type() == at::kInt ? YP_POS_I32 : YP_POS_F32;
        d.position_stride[0] = n == 2 && positions.size(0) != 1 ? positions.stride(0) : 0;
        d.position_stride[1] = positions.stride(n - 1);
        d.position_stride[2] = how.axes == 2 ? positions.stride(n) : 0;
    }
    d.start = how.start;
    d.dtype = type_code(q.scalar_type());
    d.axes = how.axes;
    d.interleaved = how.interleaved;
    d.inverse = inverse;
    d.scale = (float)how.scale;
    check(lib.rotary(&d, stream_of(q)));
}

Tensor feature_dense(const Tensor& x) { return x.defined() && x.stride(3) == 1 && !x.is_neg() && !x._is_zerotensor() ? x : dense(x); }

std::pair<Tensor, Tensor> turned(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq, const Turn& how, bool inverse) {
    const Tensor qd = feature_dense(q), kd = feature_dense(k);
    Tensor q_out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous)), k_out;
    if (k.defined()) k_out = at::empty(k.sizes(), q_out.options());
    turn_launch(qd, kd, q_out, k_out, positions, inv_freq, how, inverse);
    return {q_out, k_out};
}

struct RotaryBackward : Node {
    SavedVariable positions, inv_freq;
    Turn how;
    bool has_k = false;

    std::string name() const override { return "RotaryBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        positions.reset_data();
        inv_freq.reset_data();
    }
    variable_list apply(variable_list&& in) override {     // gradients of (q, k)
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(2);
        check_untraced("rotary's gradient");
        const Tensor dq = task_should_compute_output(0) ? in[0] : Tensor(), dk = has_k && task_should_compute_output(1) ? in[1] : Tensor();
        const Tensor first = dq.defined() ? dq : dk, second = dq.defined() ? dk : Tensor();
        if (!first.defined()) return out;
        const Tensor positions_ = positions.unpack(), inv_freq_ = inv_freq.unpack();
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(first.device());
            auto [a, b] = turned(first, second, positions_, inv_freq_, how, true);
            if (dq.defined()) { out[0] = a; out[1] = b; }
            else out[1] = a;
        }
        return once(std::move(out));
    }
};

// no element twice: every stride reaches past what the smaller ones cover
bool apart(const Tensor& t) {
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t covered = 1;
    for (auto& d : dims) {
        if (d.first < covered) return false;
        covered += (d.second - 1) * d.first;
    }
    return true;
}

// q and k share no element: their memory does not meet, or they are parts of one tensor that stand beside each other in every batch entry, token or head.
// Of their dimensions some are walked by both with the same strides; what one step of those spans holds the one's remaining dimensions and behind them
// the other's.  Every choice of common dimensions is tried.
bool separate(const Tensor& q, const Tensor& k) {
    if (q.numel() == 0 || k.numel() == 0) return true;
    const char *a = (const char*)q.data_ptr(), *b = (const char*)k.data_ptr();
    const Tensor &low = a <= b ? q : k, &high = a <= b ? k : q;
    const int64_t size = q.element_size(), bytes = a <= b ? b - a : a - b;
    auto reach = [](const Tensor& t, int common) {
        int64_t n = 1;
        for (int i = 0; i < 4; ++i)
            if (!(common >> i & 1)) n += (t.size(i) - 1) * t.stride(i);
        return n;
    };
    if (reach(low, 0) * size <= bytes) return true;
    if (bytes % size) return false;
    for (int common = 1; common < 8; ++common) {            // (never the features: a run of them is the smallest part)
        std::vector<std::pair<int64_t, int64_t>> steps;
        bool fits = reach(low, common) <= bytes / size;
        for (int i = 0; i < 3; ++i) {
            if (!(common >> i & 1) || std::max(q.size(i), k.size(i)) == 1) continue;
            fits = fits && q.stride(i) == k.stride(i);
            steps.emplace_back(q.stride(i), std::max(q.size(i), k.size(i)));
        }
        std::sort(steps.begin(), steps.end());
        int64_t covered = bytes / size + reach(high, common);
        for (auto& st : steps) {
            fits = fits && st.first >= covered;
            covered += (st.second - 1) * st.first;
        }
        if (fits) return true;
    }
    return false;
}

std::tuple<Tensor, MaybeTensor> rotary(const Tensor& q, const MaybeTensor& k, const MaybeTensor& positions, int64_t start, const Tensor& inv_freq, bool interleaved, bool heads_first,
                                       double scale, bool inplace) {
    check_tensor("rotary", q);
    check_beside("rotary", q, k);
    check_beside("rotary", q, positions);
    check_beside("rotary", q, inv_freq);
    if (q.dim() != 4 || q.size(3) < 2 || q.size(3) > 1024) fail("rotary: q of four dimensions, heads of 2 to 1024 features, not %s", shape_of(q).c_str());
    if (inv_freq.scalar_type() != at::kDouble || inv_freq.dim() != 1 || !inv_freq.is_contiguous() || inv_freq.numel() < 1 || 2 * inv_freq.numel() > q.size(3))
        fail("rotary: inv_freq is float64 [R / 2] with R <= the head's features");
    if (inv_freq.requires_grad() || inv_freq.is_neg()) fail("rotary: inv_freq is a plain table and has no gradient");
    const int64_t B = batch_of(q), T = tokens_of(q, heads_first);
    const int64_t most = (int64_t)1 << 31;
    if (B >= most || T >= most || (T && B >= (most + T - 1) / T) || heads_of(q, heads_first) >= most / 2) fail("rotary: fewer than 2^31 tokens a call");
    if (k && (k->dim() != 4 || k->scalar_type() != q.scalar_type() || k->size(3) != q.size(3) || batch_of(*k) != B || tokens_of(*k, heads_first) != T || heads_of(*k, heads_first) >= most / 2))
        fail("rotary: k of q's type, batch, tokens and head size");
    Turn how;
    how.start = start;
    how.interleaved = interleaved;
    how.heads_first = heads_first;
    how.scale = scale;
    if (positions) {
        const auto t = positions->scalar_type();
        if (t != at::kLong && t != at::kInt && t != at::kFloat) fail("rotary: positions in int32, int64 or float32");
        if (positions->requires_grad()) fail("rotary: positions have no gradient");
        auto is = [&](std::initializer_list<int64_t> s) { return positions->sizes() == at::IntArrayRef(s); };
        if (!is({T}) && !is({1, T}) && !is({B, T})) {
            how.axes = 2;
            if (!is({T, 2}) && !is({1, T, 2}) && !is({B, T, 2}))
                fail("rotary: positions [T], [B, T], [T, 2] or [B, T, 2] with B = %lld, T = %lld, not %s", (long long)B, (long long)T, shape_of(*positions).c_str());
            if (inv_freq.numel() % 2) fail("rotary: two axes need an even number of pairs");
        }
    }
    const c10::DeviceGuard guard(q.device());
    const Tensor k_ = given(k), positions_ = positions ? plain(*positions) : Tensor();
    const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || wants(k));
    if (inplace) {
        if (grad) fail("rotary: no gradients in place");
        if (q.stride(3) != 1 || q.is_neg() || q._is_zerotensor() || (k && (k->stride(3) != 1 || k->is_neg() || k->_is_zerotensor()))) fail("rotary: dense features in place");
        if (q.numel() + (k ? k->numel() : 0) == 0) return {q, k};
        if (!apart(q) || (k && (!apart(*k) || !separate(q, *k)))) fail("rotary: q and k hold each element once in place");
        q.unsafeGetTensorImpl()->bump_version();            // (refuses an inference tensor outside inference mode)
        if (k) k_.unsafeGetTensorImpl()->bump_version();
        turn_launch(q, k_, q, k_, positions_, inv_freq, how, false);
        return {q, k};
    }
    std::pair<Tensor, Tensor> out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = turned(q, k_, positions_, inv_freq, how, false);
    }
    if (grad) {
        std::shared_ptr<RotaryBackward> node(new RotaryBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(q, k_));
        node->how = how;
        node->has_k = k.has_value();
        node->positions = SavedVariable(positions_, false);
        node->inv_freq = SavedVariable(inv_freq, false);
        torch::autograd::set_history(out.first, node);
        if (k) torch::autograd::set_history(out.second, node);
    }
    return {out.first, k ? MaybeTensor(out.second) : MaybeTensor()};
}

void init(const std::vector<uintptr_t>& entries, py::object error) {
    TORCH_CHECK(entries.size() == 7, "seven entry points");
    lib = Entry{(decltype(Entry::last_error))entries[0], (decltype(Entry::norm_fwd))entries[1], (decltype(Entry::norm_bwd))entries[2], (decltype(Entry::norm_workspace))entries[3],
                (decltype(Entry::norm_max_width))entries[4], (decltype(Entry::dropout))entries[5], (decltype(Entry::rotary))entries[6]};
    yp_error = error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(_token_autograd, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused& e) {
            PyErr_SetString(yp_error ? yp_error : PyExc_RuntimeError, e.what());
        }
    });
    typedef py::call_guard<py::gil_scoped_release> Free;
    m.def("init", &init);
    m.def("layer_norm", &layer_norm, Free());
    m.def("dropout_add_layer_norm", &dropout_add_layer_norm, Free());
    m.def("dropout", &dropout, Free());
    m.def("rotary", &rotary, Free());
}
