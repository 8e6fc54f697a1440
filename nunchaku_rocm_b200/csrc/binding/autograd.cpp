// The differentiable operators' way from torch to the C ABI: allocation, autograd nodes and launches in C++.
//
// These operators run inside training steps, where a Python autograd function costs more than the kernels of a small call:
// the engine's worker thread has to take the interpreter lock and interpret the backward pass on another core.  Measured on
// a B200's host for a layer norm of 154 x 1152, forward and backward: 120 us a step with Python functions (23 forward, about
// 45 the engine itself), 82 with these (torch's own layer norm: 72).  The arguments' checks stay in Python
// (ops/elementwise.py, ops/rotary.py, ops/lora.py): what arrives here is valid.
//
// The library's functions are bound by address, so that this module calls the very library that ctypes loaded.
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
    decltype(&nb_strerror) strerror;
    decltype(&nb_last_error_detail) last_error_detail;
    decltype(&nb_last_cuda_error) last_cuda_error;
    decltype(&nb_last_cuda_error_string) last_cuda_error_string;
} lib;

void bind(const std::map<std::string, uintptr_t>& at) {
#define NB_BIND(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at("nb_" #name))
    NB_BIND(layer_norm); NB_BIND(layer_norm_backward); NB_BIND(layer_norm_workspace_bytes);
    NB_BIND(rotary_ladder_init); NB_BIND(rotary_axes); NB_BIND(rotary_table);
    NB_BIND(lora_forward); NB_BIND(lora_backward); NB_BIND(lora_workspace_bytes);
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

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool defined(const OptTensor& t) { return t.has_value() && t->defined(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && wants_grad(*t); }
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

int dtype_of(const Tensor& t) {
    return t.scalar_type() == at::kBFloat16 ? NB_DTYPE_BF16 : t.scalar_type() == at::kHalf ? NB_DTYPE_FP16 : NB_DTYPE_FP32;
}

// `t (..., C)` and the stride between its rows: a copy only where the rows are not evenly strided (and, with `aligned`, not
// on 16-byte boundaries)
Tensor strided_rows(const Tensor& t, int64_t* stride, bool aligned) {
    const int64_t c = t.size(-1);
    Tensor r = t;
    *stride = c;
    if (!t.is_contiguous()) {
        // rows are evenly strided when every outer dimension steps over whole runs of the ones inside it
        bool even = t.stride(-1) == 1;
        int64_t step = 0, run = 1;
        for (int64_t d = t.dim() - 2; even && d >= 0; --d) {
            if (t.size(d) == 1) continue;
            if (run == 1) step = t.stride(d);
            else even = t.stride(d) == run * step;
            run *= t.size(d);
        }
        if (even) *stride = run == 1 ? c : step;
        else r = t.contiguous();
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
    if (need_x) out[0] = at::empty(x.sizes(), x.options());
    if (need_w) out[1] = empty ? at::zeros(weight.sizes(), weight.options()) : at::empty(weight.sizes(), weight.options());
    if (need_b) out[2] = empty ? at::zeros(bias.sizes(), bias.options()) : at::empty(bias.sizes(), bias.options());
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
        ws = at::empty({a.workspace_bytes}, x.options().dtype(at::kByte));
        a.workspace = ws.data_ptr();
    }
    check(lib.layer_norm_backward(&a, stream_of(x)), "layer_norm backward");
    return out;
}
Tensor new_stats(const Tensor& x) { return at::empty({2, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat)); }

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, double add) {
        const Tensor y = at::empty(x.sizes(), x.options()), stats = new_stats(x), w = or_none(weight), b = or_none(bias);
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
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias))) return LayerNorm::apply(x, weight, bias, eps, add);
    const Tensor y = at::empty(x.sizes(), x.options());
    ln_forward(x, or_none(weight), or_none(bias), eps, add, y, Tensor());
    return y;
}
void layer_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, double add, const OptTensor& y, const OptTensor& stats) {
    ln_forward(x, or_none(weight), or_none(bias), eps, add, or_none(y), or_none(stats));
}
std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const Tensor& stats,
                                                                const Tensor& dy, double eps, double add, bool need_x, bool need_w, bool need_b) {
    const auto g = ln_backward(x, or_none(weight), or_none(bias), stats, dy, eps, add, need_x, need_w, need_b);
    return {or_none(g[0]), or_none(g[1]), or_none(g[2])};
}

// -------------------------------------------------------------------------------------------------------------- rotary
struct Ladder : torch::CustomClassHolder {
    nb_rotary_ladder l = {};
    Ladder(const std::vector<int32_t>& axes, double theta) { check(lib.rotary_ladder_init(&l, axes.data(), (int32_t)axes.size(), theta), "rotary ladder"); }
    int pairs() const { return l.pair_end[l.n_axes - 1]; }
};
using LadderPtr = c10::intrusive_ptr<Ladder>;

int ids_type(const Tensor& ids) {
    switch (ids.scalar_type()) {
        case at::kFloat: return NB_IDS_F32;
        case at::kInt: return NB_IDS_I32;
        case at::kLong: return NB_IDS_I64;
        default: return NB_IDS_F64;
    }
}
// (q', k'): one launch over the heads of both; k may be undefined
variable_list rotate(const Tensor& q_in, const Tensor& k_in, const Tensor& ids, const Ladder& ladder, bool half, bool inverse) {
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = q_in.stride(3) == 1 ? q_in : q_in.contiguous();
    const Tensor k = !k_in.defined() || k_in.stride(3) == 1 ? k_in : k_in.contiguous();
    variable_list out = {at::empty(q.sizes(), q.options()), k.defined() ? at::empty(k.sizes(), k.options()) : Tensor()};
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
variable_list rotary_axes(const Tensor& q, const OptTensor& k, const Tensor& ids, const LadderPtr& ladder, bool half, bool inverse) {
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k))) return Rotary::apply(q, k, ids, ladder, half, inverse);
    variable_list out = rotate(q, or_none(k), ids, *ladder, half, inverse);
    if (!defined(k)) out.pop_back();
    return out;
}
Tensor rotary_table(const Tensor& ids, const LadderPtr& ladder) {
    const c10::cuda::CUDAGuard guard(ids.device());
    const bool batched = ids.dim() == 3;
    auto shape = ids.sizes().vec();
    shape.back() = ladder->pairs();
    shape.push_back(1);
    shape.push_back(2);
    const Tensor out = at::empty(shape, ids.options().dtype(at::kFloat));
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
// out, and the two 16-bit parts of scale x down^T
Tensor run_lora(const Tensor& x, const Tensor& base, const Tensor& down, const Tensor& up, const Tensor& offsets, const Tensor& adapters, const Tensor& scale,
                const Tensor& out, int64_t impl, int64_t status) {
    const int64_t rows = x.numel() / down.size(2);
    const Tensor h = at::empty({2, rows, down.size(1)}, x.options());
    if (rows == 0) return h;
    const c10::cuda::CUDAGuard guard(x.device());
    nb_lora_args a = lora_args(rows, down, up, offsets, adapters, scale, impl, status);
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
    return at::empty(shape, x.options());
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
        if (need_x) dx = at::empty(shape, down.options());
        if (need_down) ddown = rows ? at::empty(down.sizes(), down.options()) : at::zeros(down.sizes(), down.options());
        if (need_up) dup = rows ? at::empty(up.sizes(), up.options()) : at::zeros(up.sizes(), up.options());
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
            ws = at::empty({at_g + (need_x || need_down ? 4 * rows * down.size(1) : 0)}, down.options().dtype(at::kByte));
            if (a.workspace_bytes) a.workspace = ws.data_ptr();
            if (need_x || need_down) a.g = ws.data_ptr<uint8_t>() + at_g;
            check(lib.lora_backward(&a, stream_of(down)), "lora_batched backward");
        }
        variable_list r = once({dx, ddown, dup});
        return {r[0], r[1], r[2], has_base && ctx->needs_input_grad(3) ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
Tensor lora_batched(const Tensor& x, const Tensor& down, const Tensor& up, const Tensor& offsets, const Tensor& adapters, const OptTensor& base,
                    const OptTensor& scale, const OptTensor& out, int64_t impl, int64_t status) {
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(down) || wants_grad(up) || wants_grad(base)))
        return Lora::apply(x, down, up, base, offsets, adapters, scale, impl, status);
    const Tensor to = defined(out) ? *out : new_out(x, up);
    run_lora(x, or_none(base), down, up, offsets, adapters, or_none(scale), to, impl, status);
    if (defined(out) && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version();  // a graph that saved it must notice
    return to;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    m.def("bind", &bind);
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
