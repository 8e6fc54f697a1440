// The differentiable operators' way from torch to the C ABI: allocation, autograd nodes and launches in C++.
//
// These operators run inside training steps, where a Python autograd function costs more than the kernels of a small call:
// the engine's worker thread has to take the interpreter lock and interpret the backward pass on another core.  Measured on
// a B200's host for a layer norm of 154 x 1152, forward and backward: 120 us a step with Python functions (23 forward, about
// 45 the engine itself), 74 with these (torch's own layer norm: 76).  The arguments' checks are here for the same reason:
// they took a third of a small call in Python.
//
// The library's functions are bound by address, so that this module calls the very library that ctypes loaded.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../../include/nunchaku_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Library {
    decltype(&nb_layer_norm) layer_norm;
    decltype(&nb_layer_norm_backward) layer_norm_backward;
    decltype(&nb_layer_norm_workspace_bytes) layer_norm_workspace_bytes;
    decltype(&nb_rotary_ladder_init) rotary_ladder_init;
    decltype(&nb_rotary_axes) rotary_axes;
    decltype(&nb_rotary_table) rotary_table;
    decltype(&nb_lora_forward) lora_forward;
    decltype(&nb_lora_backward) lora_backward;
    decltype(&nb_lora_workspace_bytes) lora_workspace_bytes;
    decltype(&nb_lora_h_bytes) lora_h_bytes;
    decltype(&nb_strerror) strerror;
    decltype(&nb_last_error_detail) last_error_detail;
    decltype(&nb_last_cuda_error) last_cuda_error;
    decltype(&nb_last_cuda_error_string) last_cuda_error_string;
} lib;

// (device index) -> address of its status word, after the device's self-test; called once per device
PyObject* first_use = nullptr;

void bind(const std::map<std::string, uintptr_t>& at, py::function on_first_use) {
    first_use = on_first_use.release().ptr();
#define NB_BIND(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at("nb_" #name))
    NB_BIND(layer_norm); NB_BIND(layer_norm_backward); NB_BIND(layer_norm_workspace_bytes);
    NB_BIND(rotary_ladder_init); NB_BIND(rotary_axes); NB_BIND(rotary_table);
    NB_BIND(lora_forward); NB_BIND(lora_backward); NB_BIND(lora_workspace_bytes); NB_BIND(lora_h_bytes);
    NB_BIND(strerror); NB_BIND(last_error_detail); NB_BIND(last_cuda_error); NB_BIND(last_cuda_error_string);
#undef NB_BIND
}

// the exceptions of _lib.check()
void check(int status, const char* what) {
    if (status == NB_OK) return;
    std::string message = std::string(what) + ": " + lib.strerror(status);
    const std::string detail = lib.last_error_detail();
    if (!detail.empty()) message += " (" + detail + ")";
    if (status == NB_ERR_LAUNCH) {
        message += std::string(": ") + lib.last_cuda_error_string();
        lib.last_cuda_error();
    }
    TORCH_CHECK_VALUE(status != NB_ERR_INVALID, message);
    TORCH_CHECK_NOT_IMPLEMENTED(status != NB_ERR_UNSUPPORTED, message);
    TORCH_CHECK(false, message);
}

int64_t status_of(int device) {
    static std::array<int64_t, 64> known = {};
    TORCH_CHECK(device >= 0 && device < (int)known.size(), "device index ", device);
    if (!known[device]) {  // (the caller is Python: it holds the interpreter lock)
        known[device] = py::reinterpret_borrow<py::function>(first_use)(device).cast<int64_t>();
    }
    return known[device];
}
// All given tensors live on one CUDA device; its status word.
template <typename... Rest>
int64_t require_cuda(const Tensor& first, const Rest&... rest) {
    const auto one = [&](const Tensor& t) {
        if (!t.defined()) return;
        TORCH_CHECK(t.is_cuda(), "nunchaku_rocm_b200 kernels need CUDA tensors (there is no CPU path)");
        TORCH_CHECK_VALUE(t.get_device() == first.get_device(), "tensors on different devices");
    };
    one(first);
    (one(rest), ...);
    return status_of(first.get_device());
}
// An uninitialised contiguous tensor beside `like`, without the dispatcher.
Tensor empty_of(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor empty_of(at::IntArrayRef sizes, const Tensor& like) { return empty_of(sizes, like.scalar_type(), like); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool defined(const OptTensor& t) { return t.has_value() && t->defined(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && wants_grad(*t); }
// A tensor with a tangent (forward-mode differentiation) would lose it here without a word.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename... Tensors>
void refuse_tangents(const char* what, const Tensors&... tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(tensors) || ...), what, " has no forward-mode derivative");
}
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

int dtype_of(const Tensor& t) {
    return t.scalar_type() == at::kBFloat16 ? NB_DTYPE_BF16 : t.scalar_type() == at::kHalf ? NB_DTYPE_FP16 : NB_DTYPE_FP32;
}

// Whether the rows of `t (..., C)` are evenly strided: every outer dimension steps over whole runs of the ones inside it.
bool even_rows(const Tensor& t, int64_t* stride) {
    *stride = t.size(-1);
    if (t.is_contiguous()) return true;
    if (t.stride(-1) != 1) return false;
    int64_t run = 1;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (run == 1) *stride = t.stride(d);
        else if (t.stride(d) != run * *stride) return false;
        run *= t.size(d);
    }
    return true;
}
// `t` and the stride between its rows: a copy only where the rows are not evenly strided (and, with `aligned`, not on
// 16-byte boundaries)
Tensor strided_rows(const Tensor& t, int64_t* stride, bool aligned) {
    const int64_t c = t.size(-1);
    Tensor r = t;
    if (!even_rows(t, stride)) {
        r = t.contiguous();
        *stride = c;
    }
    if (aligned && ((*stride % 8) != 0 || (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15))) {
        r = r.clone(at::MemoryFormat::Contiguous);
        *stride = c;
    }
    return r;
}

// Gradients that have no graph of their own: differentiating them again raises (as Python's once_differentiable does).
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list held;
    for (auto& g : grads) {
        if (!g.defined()) continue;
        held.push_back(g.detach());
        held.back().set_requires_grad(true);
    }
    if (held.empty()) return grads;
    const int n = (int)held.size();
    variable_list out =
        (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that can be differentiated once", n))(std::move(held));
    size_t k = 0;
    for (auto& g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}

// ---------------------------------------------------------------------------------------------------------- layer norm
nb_layer_norm_args ln_args(const Tensor& x, int64_t stride, const Tensor& weight, const Tensor& bias, double eps, double add) {
    nb_layer_norm_args a = {};
    const Tensor& first = weight.defined() ? weight : bias;
    const bool grouped = first.defined() && first.dim() == 2;
    a.dim = (int32_t)x.size(-1);
    a.groups = grouped ? (int32_t)x.size(0) : 1;
    const int64_t rows = x.numel() / a.dim / a.groups;
    TORCH_CHECK(rows <= (1 << 30), "layer_norm: more than 2^30 rows");
    a.rows = (int32_t)rows;
    a.dtype = dtype_of(x);
    a.x = x.const_data_ptr();
    a.stride_x = stride;
    if (weight.defined()) a.w = weight.const_data_ptr();
    if (bias.defined()) a.b = bias.const_data_ptr();
    if (first.defined()) {
        a.w_fp32 = first.scalar_type() == at::kFloat;
        a.stride_w = grouped ? first.stride(0) : 0;
    }
    a.eps = (float)eps;
    a.weight_add = (float)add;
    return a;
}
bool known_type(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat; }
Tensor ln_weight(const char* name, const Tensor& w, const Tensor& x) {
    const int64_t dim = x.size(-1);
    TORCH_CHECK_VALUE(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, name, " must be ", x.scalar_type(), " or Float, got ",
                      w.scalar_type());
    const bool one = w.dim() == 1 && w.size(0) == dim, each = w.dim() == 2 && x.dim() == 3 && w.size(0) == x.size(0) && w.size(1) == dim;
    TORCH_CHECK_VALUE(one || each, name, " must be (", dim, ",), or (B, ", dim, ") for x (B, T, ", dim, "); got ", w.sizes(), " for ", x.sizes());
    return w.stride(-1) == 1 ? w : w.contiguous();
}
// The checks of the arguments; weight and bias with one stride and unit inner stride.
void ln_prepare(const Tensor& x, Tensor& weight, Tensor& bias, double add) {
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "layer_norm needs at least one channel, got x ", x.sizes());
    TORCH_CHECK_NOT_IMPLEMENTED(x.size(-1) <= NB_LAYER_NORM_MAX_DIM, "layer_norm takes up to ", NB_LAYER_NORM_MAX_DIM, " channels, got ", x.size(-1));
    TORCH_CHECK_VALUE(known_type(x), "layer_norm takes bfloat16, float16 and float32, got ", x.scalar_type());
    const bool grouped = (weight.defined() && weight.dim() == 2) || (bias.defined() && bias.dim() == 2);
    TORCH_CHECK(!grouped || x.size(0) <= 65535 || x.numel() == 0, "layer_norm: more than 65535 samples with a row of weights each");
    TORCH_CHECK_VALUE(weight.defined() || add == 0, "weight_add without a weight");
    if (weight.defined()) weight = ln_weight("weight", weight, x);
    if (!bias.defined()) return;
    bias = ln_weight("bias", bias, x);
    if (!weight.defined()) return;
    TORCH_CHECK_VALUE(bias.scalar_type() == weight.scalar_type() && bias.dim() == weight.dim(), "weight and bias must have one shape and one dtype");
    if (bias.dim() == 2 && bias.stride(0) != weight.stride(0)) {
        weight = weight.contiguous();
        bias = bias.contiguous();
    }
}
// y and / or the rows' (mean, rstd) into the given tensors
void ln_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, double add, const Tensor& y, const Tensor& stats) {
    if (x.numel() == 0) return;
    const c10::cuda::CUDAGuard guard(x.device());
    int64_t stride;
    const Tensor rows = strided_rows(x, &stride, false);
    nb_layer_norm_args a = ln_args(rows, stride, weight, bias, eps, add);
    if (y.defined()) a.y = y.data_ptr();
    if (stats.defined()) {
        a.mean = stats.data_ptr<float>();
        a.rstd = a.mean + stats.numel() / 2;
    }
    check(lib.layer_norm(&a, stream_of(x)), "layer_norm");
}
variable_list ln_backward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& stats, const Tensor& dy, double eps, double add,
                          bool need_x, bool need_w, bool need_b) {
    variable_list out(3);
    const c10::cuda::CUDAGuard guard(x.device());
    const bool empty = x.numel() == 0;
    if (need_x) out[0] = empty_of(x.sizes(), x);
    if (need_w) out[1] = empty ? at::zeros(weight.sizes(), weight.options()) : empty_of(weight.sizes(), weight);
    if (need_b) out[2] = empty ? at::zeros(bias.sizes(), bias.options()) : empty_of(bias.sizes(), bias);
    if (empty) return out;
    int64_t stride_x, stride_dy;
    const Tensor rows = strided_rows(x, &stride_x, false), grad = strided_rows(dy, &stride_dy, false);
    nb_layer_norm_args a = ln_args(rows, stride_x, weight, bias, eps, add);
    a.mean = stats.data_ptr<float>();
    a.rstd = a.mean + stats.numel() / 2;
    a.dy = grad.const_data_ptr();
    a.stride_dy = stride_dy;
    if (need_x) a.dx = out[0].data_ptr();
    if (need_w) a.dw = out[1].data_ptr();
    if (need_b) a.db = out[2].data_ptr();
    Tensor ws;
    if (need_w || need_b) {
        a.workspace_bytes = lib.layer_norm_workspace_bytes(a.groups, a.rows, a.dim, a.dtype);
        ws = empty_of({a.workspace_bytes}, at::kByte, x);
        a.workspace = ws.data_ptr();
    }
    check(lib.layer_norm_backward(&a, stream_of(x)), "layer_norm backward");
    return out;
}
Tensor new_stats(const Tensor& x) { return empty_of({2, x.numel() / x.size(-1)}, at::kFloat, x); }

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, double add) {
        const Tensor y = empty_of(x.sizes(), x), stats = new_stats(x), w = or_none(weight), b = or_none(bias);
        ln_forward(x, w, b, eps, add, y, stats);
        ctx->save_for_backward({x, w, b, stats});
        ctx->saved_data["consts"] = std::vector<double>{eps, add};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto consts = ctx->saved_data["consts"].toDoubleVector();
        const bool need_w = saved[1].defined() && ctx->needs_input_grad(1), need_b = saved[2].defined() && ctx->needs_input_grad(saved[1].defined() ? 2 : 1);
        variable_list g = once(ln_backward(saved[0], saved[1], saved[2], saved[3], grads[0], consts[0], consts[1], ctx->needs_input_grad(0), need_w, need_b));
        return {g[0], g[1], g[2], Tensor(), Tensor()};
    }
};
Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, double add) {
    Tensor w = or_none(weight), b = or_none(bias);
    ln_prepare(x, w, b, add);
    refuse_tangents("layer_norm", x, w, b);
    require_cuda(x, w, b);
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) return LayerNorm::apply(x, or_none(w), or_none(b), eps, add);
    const Tensor y = empty_of(x.sizes(), x);
    ln_forward(x, w, b, eps, add, y, Tensor());
    return y;
}
// without autograd: y and / or the statistics, and the gradients from these
void layer_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, double add, const OptTensor& y, const OptTensor& stats) {
    Tensor w = or_none(weight), b = or_none(bias);
    ln_prepare(x, w, b, add);
    ln_forward(x, w, b, eps, add, or_none(y), or_none(stats));
}
std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const Tensor& stats,
                                                                const Tensor& dy, double eps, double add, bool need_x, bool need_w, bool need_b) {
    Tensor w = or_none(weight), b = or_none(bias);
    ln_prepare(x, w, b, add);
    const auto g = ln_backward(x, w, b, stats, dy, eps, add, need_x, need_w, need_b);
    return {or_none(g[0]), or_none(g[1]), or_none(g[2])};
}

// -------------------------------------------------------------------------------------------------------------- rotary
struct Ladder : torch::CustomClassHolder {
    nb_rotary_ladder l = {};
    Ladder(const std::vector<int32_t>& axes, double theta) { check(lib.rotary_ladder_init(&l, axes.data(), (int32_t)axes.size(), theta), "rotary ladder"); }
    int pairs() const { return l.pair_end[l.n_axes - 1]; }
};
using LadderPtr = c10::intrusive_ptr<Ladder>;

constexpr int64_t kMaxRows = 0x7fffffff;

int ids_type(const Tensor& ids) {
    switch (ids.scalar_type()) {
        case at::kFloat: return NB_IDS_F32;
        case at::kInt: return NB_IDS_I32;
        case at::kLong: return NB_IDS_I64;
        case at::kDouble: return NB_IDS_F64;
        default: TORCH_CHECK_VALUE(false, "ids must be float32, float64, int32 or int64, got ", ids.scalar_type());
    }
}
void check_ids(const char* what, const Tensor& ids, int64_t axes, int64_t batch, int64_t rows) {
    ids_type(ids);
    const int64_t d = ids.dim();
    TORCH_CHECK_VALUE((d == 2 || (d == 3 && ids.size(0) == batch)) && ids.size(d - 2) == rows && ids.size(d - 1) == axes, "ids must be (", rows, ", ", axes,
                      ") or (", batch, ", ", rows, ", ", axes, "), got ", ids.sizes());
    TORCH_CHECK_VALUE(!(ids.requires_grad() && at::GradMode::is_enabled()), what, " has no gradient for ids");
}
// (q', k'): one launch over the heads of both; k may be undefined
variable_list rotate(const Tensor& q_in, const Tensor& k_in, const Tensor& ids, const Ladder& ladder, bool half, bool inverse) {
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = q_in.stride(3) == 1 ? q_in : q_in.contiguous();
    const Tensor k = !k_in.defined() || k_in.stride(3) == 1 ? k_in : k_in.contiguous();
    variable_list out = {empty_of(q.sizes(), q), k.defined() ? empty_of(k.sizes(), k) : Tensor()};
    nb_rotary_args a = {};
    a.q = q.const_data_ptr();
    a.q_out = out[0].data_ptr();
    a.ids = ids.const_data_ptr();
    a.B = (int32_t)q.size(0); a.S = (int32_t)q.size(1); a.H = (int32_t)q.size(2); a.D = (int32_t)q.size(3);
    a.stride_qb = q.stride(0); a.stride_qs = q.stride(1); a.stride_qh = q.stride(2);
    if (k.defined()) {
        a.k = k.const_data_ptr();
        a.k_out = out[1].data_ptr();
        a.Hk = (int32_t)k.size(2);
        a.stride_kb = k.stride(0); a.stride_ks = k.stride(1); a.stride_kh = k.stride(2);
    }
    const bool batched = ids.dim() == 3;
    a.stride_ib = batched ? ids.stride(0) : 0;
    a.stride_is = ids.stride(batched);
    a.stride_ia = ids.stride(batched + 1);
    a.dtype = dtype_of(q);
    a.ids_type = ids_type(ids);
    a.half = half;
    a.inverse = inverse;
    check(lib.rotary_axes(&a, &ladder.l, stream_of(q)), "rotary_axes");
    return out;
}
struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& ids, const LadderPtr& ladder, bool half, bool inverse) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({ids});
        ctx->saved_data["ladder"] = c10::IValue::make_capsule(ladder);
        ctx->saved_data["half"] = half;
        ctx->saved_data["inverse"] = inverse;
        ctx->saved_data["k"] = defined(k);
        variable_list out = rotate(q, or_none(k), ids, *ladder, half, inverse);
        if (!defined(k)) out.pop_back();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto capsule = ctx->saved_data["ladder"].toCapsule();
        const Ladder& ladder = *static_cast<const Ladder*>(capsule.get());
        const bool half = ctx->saved_data["half"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
        const Tensor dq = ctx->needs_input_grad(0) ? grads[0] : Tensor();
        const Tensor dk = ctx->saved_data["k"].toBool() && ctx->needs_input_grad(1) ? grads[1] : Tensor();
        variable_list g(2);
        if (dq.defined()) g = rotate(dq, dk, saved[0], ladder, half, !inverse);
        else if (dk.defined()) g[1] = rotate(dk, Tensor(), saved[0], ladder, half, !inverse)[0];
        g = once(std::move(g));
        return {g[0], g[1], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
// q', or (q', k')
py::object rotary_axes(const Tensor& q, const OptTensor& k, const Tensor& ids, const LadderPtr& ladder, bool half, bool inverse) {
    TORCH_CHECK_VALUE(known_type(q), "rotary_axes takes bfloat16, float16 and float32, got ", q.scalar_type());
    TORCH_CHECK_VALUE(q.dim() == 4, "q must be (B, S, H, D), got ", q.sizes());
    if (defined(k))
        TORCH_CHECK_VALUE(k->dim() == 4 && k->scalar_type() == q.scalar_type() && k->size(0) == q.size(0) && k->size(1) == q.size(1) && k->size(3) == q.size(3),
                          "k must be (B, S, Hk, D) beside q, got ", k->sizes(), " ", k->scalar_type(), " for ", q.sizes(), " ", q.scalar_type());
    check_ids("rotary_axes", ids, ladder->l.n_axes, q.size(0), q.size(1));
    // (as the C entry, whose sizes have 32 bits)
    TORCH_CHECK(q.size(0) <= kMaxRows && q.size(1) <= kMaxRows && q.size(2) <= kMaxRows && q.size(3) <= kMaxRows && (!defined(k) || k->size(2) <= kMaxRows),
                "rotary_axes: more than 2^31 rows or 2^26 channels per row");
    TORCH_CHECK_VALUE(2 * ladder->pairs() <= q.size(3), "the axes have ", 2 * ladder->pairs(), " channels, more than a head (", q.size(3), ")");
    TORCH_CHECK_VALUE(q.size(2) > 0 && (!defined(k) || k->size(2) > 0), "no heads");
    refuse_tangents("rotary_axes", q, k, ids);
    require_cuda(q, or_none(k), ids);
    const bool graph = at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k));
    const variable_list out = graph ? Rotary::apply(q, k, ids, ladder, half, inverse) : rotate(q, or_none(k), ids, *ladder, half, inverse);
    return defined(k) ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}
Tensor rotary_table(const Tensor& ids, const LadderPtr& ladder) {
    TORCH_CHECK_VALUE(ids.dim() == 2 || ids.dim() == 3, "ids must be (S, axes) or (B, S, axes), got ", ids.sizes());
    check_ids("rotary_table", ids, ladder->l.n_axes, ids.size(0), ids.size(-2));
    TORCH_CHECK(ids.size(0) <= kMaxRows && ids.size(-2) <= kMaxRows, "rotary_table: more than 2^31 rows");
    refuse_tangents("rotary_table", ids);
    require_cuda(ids);
    const c10::cuda::CUDAGuard guard(ids.device());
    const bool batched = ids.dim() == 3;
    auto shape = ids.sizes().vec();
    shape.back() = ladder->pairs();
    shape.push_back(1);
    shape.push_back(2);
    const Tensor out = empty_of(shape, at::kFloat, ids);
    check(lib.rotary_table(ids.const_data_ptr(), ids_type(ids), batched ? (int32_t)ids.size(0) : 1, (int32_t)ids.size(batched), batched ? ids.stride(0) : 0,
                           ids.stride(batched), ids.stride(batched + 1), out.data_ptr<float>(), &ladder->l, stream_of(out)),
          "rotary_table");
    return out;
}

// ------------------------------------------------------------------------------------------------------------ adapters
nb_lora_args lora_args(int64_t rows, const Tensor& down, const Tensor& up, const Tensor& offsets, const Tensor& adapters, const Tensor& scale, int64_t impl,
                       int64_t status) {
    nb_lora_args a = {};
    TORCH_CHECK(rows <= (1 << 30), "lora_batched: more than 2^30 rows");
    a.T = (int32_t)rows;
    a.A = (int32_t)down.size(0); a.R = (int32_t)down.size(1); a.K = (int32_t)down.size(2); a.N = (int32_t)up.size(1);
    a.requests = (int32_t)adapters.size(0);
    a.dtype = dtype_of(down);
    a.down = down.const_data_ptr();
    a.up = up.const_data_ptr();
    a.offsets = offsets.const_data_ptr<int32_t>();
    a.adapters = adapters.const_data_ptr<int32_t>();
    if (scale.defined()) a.scale = scale.const_data_ptr<float>();
    a.impl = (int32_t)impl;
    a.status = reinterpret_cast<void*>(status);
    return a;
}
// out, and scale x down^T as the backward pass reads it
Tensor run_lora(const Tensor& x, const Tensor& base, const Tensor& down, const Tensor& up, const Tensor& offsets, const Tensor& adapters, const Tensor& scale,
                const Tensor& out, int64_t impl, int64_t status) {
    const int64_t rows = x.numel() / down.size(2);
    if (rows == 0) return empty_of({0}, at::kByte, x);
    const c10::cuda::CUDAGuard guard(x.device());
    nb_lora_args a = lora_args(rows, down, up, offsets, adapters, scale, impl, status);
    const Tensor h = empty_of({lib.lora_h_bytes(&a)}, at::kByte, x);
    const Tensor xr = strided_rows(x, &a.stride_x, true);
    a.x = xr.const_data_ptr();
    Tensor br;
    if (base.defined()) {
        br = strided_rows(base, &a.stride_base, true);
        a.base = br.const_data_ptr();
    }
    const Tensor to = strided_rows(out, &a.stride_out, false);
    a.out = to.data_ptr();
    a.h = h.data_ptr();
    check(lib.lora_forward(&a, stream_of(x)), "lora_batched");
    return h;
}
Tensor new_out(const Tensor& x, const Tensor& up) {
    auto shape = x.sizes().vec();
    shape.back() = up.size(1);
    return empty_of(shape, x);
}
struct Lora : torch::autograd::Function<Lora> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& down, const Tensor& up, const OptTensor& base, const Tensor& offsets,
                          const Tensor& adapters, const OptTensor& scale, int64_t impl, int64_t status) {
        const Tensor out = new_out(x, up), s = or_none(scale);
        const Tensor h = run_lora(x, or_none(base), down, up, offsets, adapters, s, out, impl, status);
        // x only for down's gradient, h only for up's
        ctx->save_for_backward({down.requires_grad() ? x : Tensor(), down, up, up.requires_grad() ? h : Tensor(), offsets, adapters, s});
        auto consts = x.sizes().vec();
        consts.push_back(impl);
        consts.push_back(status);
        consts.push_back(defined(base));
        ctx->saved_data["consts"] = consts;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        auto shape = ctx->saved_data["consts"].toIntVector();
        const bool has_base = shape.back();
        shape.pop_back();
        const int64_t status = shape.back();
        shape.pop_back();
        const int64_t impl = shape.back();
        shape.pop_back();
        const Tensor &x = saved[0], &down = saved[1], &up = saved[2], &h = saved[3], &dy = grads[0];
        const bool need_x = ctx->needs_input_grad(0), need_down = ctx->needs_input_grad(1), need_up = ctx->needs_input_grad(2);
        const c10::cuda::CUDAGuard guard(down.device());
        const int64_t rows = dy.numel() / up.size(1);
        Tensor dx, ddown, dup, ws, xr, dyr;
        if (need_x) dx = empty_of(shape, down);
        if (need_down) ddown = rows ? empty_of(down.sizes(), down) : at::zeros(down.sizes(), down.options());
        if (need_up) dup = rows ? empty_of(up.sizes(), up) : at::zeros(up.sizes(), up.options());
        if (rows && (need_x || need_down || need_up)) {
            nb_lora_args a = lora_args(rows, down, up, saved[4], saved[5], saved[6], impl, status);
            dyr = strided_rows(dy, &a.stride_dy, true);
            a.dy = dyr.const_data_ptr();
            if (need_x) a.dx = dx.data_ptr();
            if (need_down) {
                xr = strided_rows(x, &a.stride_x, true);
                a.x = xr.const_data_ptr();
                a.ddown = ddown.data_ptr();
            }
            if (need_up) {
                a.h = h.data_ptr();
                a.dup = dup.data_ptr();
            }
            // the workspace and g in one allocation (each costs the worker thread some microseconds)
            a.workspace_bytes = need_down || need_up ? lib.lora_workspace_bytes(&a) : 0;
            const int64_t at_g = (a.workspace_bytes + 255) / 256 * 256;
            ws = empty_of({at_g + (need_x || need_down ? lib.lora_h_bytes(&a) : 0)}, at::kByte, down);
            if (a.workspace_bytes) a.workspace = ws.data_ptr();
            if (need_x || need_down) a.g = ws.data_ptr<uint8_t>() + at_g;
            check(lib.lora_backward(&a, stream_of(down)), "lora_batched backward");
        }
        variable_list r = once({dx, ddown, dup});
        return {r[0], r[1], r[2], has_base && ctx->needs_input_grad(3) ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
// Whether the kernels can write `t (..., C)` in place: rows evenly strided and apart, each on a 16-byte boundary.
bool writable_rows(const Tensor& t) {
    int64_t stride;
    return even_rows(t, &stride) && stride % 8 == 0 && (stride >= t.size(-1) || t.numel() <= t.size(-1)) &&
           (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
}
Tensor lora_batched(const Tensor& x, const Tensor& down_, const Tensor& up_, const Tensor& offsets_, const Tensor& adapters_, const OptTensor& base,
                    const OptTensor& scale_, const OptTensor& out, int64_t impl) {
    const auto type = x.scalar_type();
    const auto other = [&](const Tensor& t) { return t.defined() && t.scalar_type() != type; };
    TORCH_CHECK_VALUE((type == at::kBFloat16 || type == at::kHalf) && !other(down_) && !other(up_) && !other(or_none(base)) && !other(or_none(out)),
                      "x, base, down, up and out must share one dtype, bfloat16 or float16");
    TORCH_CHECK_VALUE(down_.dim() == 3 && up_.dim() == 3 && down_.size(0) == up_.size(0) && down_.size(1) == up_.size(2) && down_.size(0) > 0,
                      "down must be (A, R, K) and up (A, N, R); got ", down_.sizes(), " and ", up_.sizes());
    const int64_t A = down_.size(0), R = down_.size(1), K = down_.size(2), N = up_.size(1);
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) == K, "x must be (..., ", K, "), got ", x.sizes());
    const auto fits = [&](const OptTensor& t) {
        return !defined(t) || (t->dim() == x.dim() && t->size(-1) == N && t->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1));
    };
    TORCH_CHECK_VALUE(fits(base), "base must be (..., ", N, ") beside x ", x.sizes(), ", got ", base->sizes());
    TORCH_CHECK_VALUE(fits(out), "out must be (..., ", N, ") beside x ", x.sizes(), ", got ", out->sizes());
    TORCH_CHECK_NOT_IMPLEMENTED(R > 0 && R % 16 == 0 && R <= NB_LORA_MAX_RANK && K > 0 && K % 8 == 0 && N > 0 && N % 8 == 0, "rank ", R,
                                " must be a multiple of 16 up to ", NB_LORA_MAX_RANK, ", K=", K, " and N=", N, " multiples of 8");
    TORCH_CHECK_VALUE(offsets_.scalar_type() == at::kInt && adapters_.scalar_type() == at::kInt && offsets_.dim() == 1 && adapters_.dim() == 1,
                      "offsets and adapters must be 1-D int32 tensors");
    TORCH_CHECK_VALUE(offsets_.size(0) == adapters_.size(0) + 1, adapters_.size(0), " adapters need ", adapters_.size(0) + 1, " offsets, got ",
                      offsets_.size(0));
    TORCH_CHECK_VALUE(!defined(scale_) || (scale_->scalar_type() == at::kFloat && scale_->dim() == 1 && scale_->size(0) == A), "scale must be (", A,
                      ",) float32");
    // (as the C entry, whose sizes have 32 bits)
    TORCH_CHECK(A <= 65535 && adapters_.size(0) <= 65535 && K <= (1 << 24) && N <= (1 << 24), "lora_batched: more than 65535 adapters or requests, or 2^24 columns");
    const bool grad = at::GradMode::is_enabled();
    TORCH_CHECK_VALUE(!grad || !wants_grad(scale_), "lora_batched has no gradient for scale");
    TORCH_CHECK_VALUE(!defined(out) || writable_rows(*out), "out must have evenly strided rows on 16-byte boundaries that do not overlap");
    refuse_tangents("lora_batched", x, down_, up_, base, scale_, out);
    const int64_t status = require_cuda(x, down_, up_, offsets_, adapters_, or_none(base), or_none(scale_), or_none(out));
    const bool graph = grad && (wants_grad(x) || wants_grad(down_) || wants_grad(up_) || wants_grad(base));
    TORCH_CHECK_VALUE(!defined(out) || !(graph || (grad && wants_grad(out))), "out cannot be given where a gradient is asked for");
    const Tensor down = down_.contiguous(), up = up_.contiguous(), offsets = offsets_.contiguous(), adapters = adapters_.contiguous();
    const OptTensor scale = defined(scale_) ? OptTensor(scale_->contiguous()) : std::nullopt;
    if (graph) return Lora::apply(x, down, up, base, offsets, adapters, scale, impl, status);
    const Tensor to = defined(out) ? *out : new_out(x, up);
    run_lora(x, or_none(base), down, up, offsets, adapters, or_none(scale), to, impl, status);
    if (defined(out) && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version();  // a graph that saved it must notice
    return to;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    m.def("bind", &bind);
    m.def("has_tangent", py::overload_cast<const Tensor&>(&has_tangent));
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_forward", &layer_norm_forward);
    m.def("layer_norm_backward", &layer_norm_backward);
    py::class_<Ladder, LadderPtr>(m, "Ladder")
        .def(py::init([](const std::vector<int32_t>& axes, double theta) { return c10::make_intrusive<Ladder>(axes, theta); }))
        .def_property_readonly("n_axes", [](const Ladder& l) { return l.l.n_axes; })
        .def_property_readonly("pairs", &Ladder::pairs);
    m.def("rotary_axes", &rotary_axes);
    m.def("rotary_table", &rotary_table);
    m.def("lora_batched", &lora_batched);
}
