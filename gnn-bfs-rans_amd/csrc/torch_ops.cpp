// The row operators (mignn.attention) as PyTorch calls with gradients: this
// module (mignn/_ops.so) owns memory and the autograd graph, the arithmetic is
// libmignn's C ABI.  In C++ because a call of a probe's size is a few
// microseconds of work: a Python autograd function costs 60 us more a training
// step, most of it in the engine's thread, and the arguments' checks 1.5 us a
// call.
#include <torch/extension.h>

#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <array>
#include <cmath>
#include <cstring>
#include <stdexcept>
#include <string>

#include "../../include/mignn.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

// The library's entry points, by the addresses that the loader resolved (the
// library is the one that mignn._lib loaded)
struct Library {
    decltype(&mignn_last_error) last_error;
    decltype(&mignn_rms_norm) rms_norm;
    decltype(&mignn_rms_norm_backward_scratch_bytes) rms_norm_backward_scratch_bytes;
    decltype(&mignn_rms_norm_backward) rms_norm_backward;
    decltype(&mignn_rotary) rotary;
    decltype(&mignn_cross_attn_forward) cross_attn_forward;
    decltype(&mignn_cross_attn_backward) cross_attn_backward;
} lib;

void bind(const std::vector<uint64_t>& at) {
    if (at.size() * sizeof(uint64_t) != sizeof(lib)) throw std::invalid_argument("mignn: entry points");
    std::memcpy(&lib, at.data(), sizeof(lib));
}

void check(int rc, const char* what) {
    if (rc == 0) return;
    throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(rc) +
                             "): " + lib.last_error());
}

void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// A plan's or an axes' table may have been made on another stream than the one
// that reads it: its memory is not given away before this stream is done
void reads(const Tensor& t) {
    if (t.is_cuda())
        c10::hip::HIPCachingAllocator::recordStream(t.storage().data_ptr(),
                                                    c10::hip::getCurrentHIPStream(t.device().index()));
}
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
int row_type(const Tensor& t) {
    return is_f32(t) ? MIGNN_ROW_F32 : t.scalar_type() == at::kBFloat16 ? MIGNN_ROW_BF16 : MIGNN_ROW_F16;
}
Tensor copied(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool needs_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ---------------------------------------------------------------------------
// Refusals

[[noreturn]] void not_implemented(const std::string& message) {
    PyErr_SetString(PyExc_NotImplementedError, message.c_str());
    throw py::error_already_set();
}
// Dual tensors (forward-mode derivatives): their tangents would be dropped
void no_tangents(const char* what, std::initializer_list<std::pair<const char*, const Tensor*>> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const auto& [name, t] : inputs)
        if (t->defined() && t->_fw_grad(0).defined())
            not_implemented(std::string(what) + ": " + name + " carries a tangent (no forward-mode derivatives)");
}

std::string shape(at::IntArrayRef sizes) {
    std::string s = "(";
    for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
    return s + (sizes.size() == 1 ? ",)" : ")");
}
std::string shape(const Tensor& t) { return shape(t.sizes()); }
std::string dtype(const Tensor& t) { return py::str(py::cast(t).attr("dtype")); }
std::string number(double v) { return py::str(py::float_(v)); }
bool is_row(const Tensor& t) {
    return is_f32(t) || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
}
void check_rows(const char* what, const Tensor& t) {
    if (!is_row(t))
        throw py::type_error(std::string(what) + ": rows must be float32, bfloat16 or float16, got " + dtype(t));
}
void on_device(const char* what, const Tensor& ref, std::initializer_list<std::pair<const char*, const Tensor*>> others) {
    if (!ref.is_cuda()) throw std::runtime_error(std::string("mignn ") + what + " runs on ROCm devices only (no CPU path)");
    for (const auto& [name, t] : others)
        if (t->defined() && t->device() != ref.device())
            throw std::runtime_error(std::string("mignn ") + what + ": " + name + " is on " + t->device().str() +
                                     ", not on " + ref.device().str());
}

// What saved-tensor hooks gave back for a saved tensor: the kernels read it by
// the gradient's device and the forward's type and shape
const Tensor& returned(const char* what, const char* name, const Tensor& t, const Tensor& grad, bool type_ok,
                       at::IntArrayRef sizes) {
    if (t.device() != grad.device() || !type_ok || t.sizes() != sizes)
        throw std::runtime_error(std::string(what) + " backward: saved " + name + " came back as " +
                                 c10::toString(t.scalar_type()) + " " + shape(t) + " on " + t.device().str() +
                                 " (expected " + shape(sizes) + ", the type that was saved, on " +
                                 grad.device().str() + ")");
    return t;
}

// Gradients that autograd cannot differentiate again: under create_graph they
// refuse it when asked.
variable_list first_order(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list real;
    for (Tensor& g : grads)
        if (g.defined()) real.push_back(g.detach().requires_grad_(true));
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "mignn row operators: gradients are first order only", static_cast<int>(real.size()));
    variable_list wrapped = (*error)(std::move(real));
    size_t k = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = wrapped[k++];
    return grads;
}

// Rows with contiguous columns that do not overlap (a copy if need be)
Tensor matrix(const Tensor& t) {
    if (!t.defined() || ((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))))
        return t;
    return copied(t);
}
int64_t row_stride(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }

// ---------------------------------------------------------------------------
// Root-mean-square norm

std::pair<Tensor, Tensor> norm_forward(const Tensor& x_, const Tensor& w_, const Tensor& r_, double eps) {
    c10::DeviceGuard guard(x_.device());
    const Tensor x = matrix(x_), r = matrix(r_), w = w_.contiguous();
    const int64_t n = x.size(0), h = x.size(1);
    Tensor y = at::empty({n, h}, x.options());
    Tensor s = r.defined() ? at::empty({n, h}, x.options()) : Tensor();
    check(lib.rms_norm(ptr(x), row_stride(x), ptr(r), row_stride(r), ptr(w), is_f32(w), n, static_cast<int>(h),
                       static_cast<float>(eps), row_type(x), out(y), h, out(s), h, stream(x)),
          "mignn_rms_norm");
    return {y, s};
}

struct RMSNorm : torch::autograd::Function<RMSNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& r,
                                 double eps) {
        auto [y, s] = norm_forward(x, w, value(r), eps);
        ctx->set_materialize_grads(false);
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["residual"] = s.defined();
        // fp32 rows: the stored s is the s that was normed; 16-bit rows: it is
        // rounded, so the gradient adds x and the residual again
        if (s.defined() && is_f32(x)) ctx->save_for_backward({s, w, Tensor()});
        else ctx->save_for_backward({x, w, value(r)});
        if (s.defined()) return {y, s};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const bool residual = ctx->saved_data["residual"].toBool();
        const bool want_w = ctx->needs_input_grad(1);
        const Tensor dy = matrix(grads[0]), ds = residual ? matrix(grads[1]) : Tensor();
        Tensor dx, dw;
        if (!dy.defined()) {
            dx = ds;
            if (want_w) dw = at::zeros_like(saved[1]);
        } else {
            const int64_t n = dy.size(0), h = dy.size(1);
            auto like_dy = [&](const Tensor& t) { return t.scalar_type() == dy.scalar_type(); };
            for (int i : {0, 2})
                if (saved[i].defined())
                    returned("rms_norm", "rows", saved[i], dy, like_dy(saved[i]), dy.sizes());
            returned("rms_norm", "weight", saved[1], dy, is_f32(saved[1]) || like_dy(saved[1]), {h});
            const Tensor x = matrix(saved[0]), w = saved[1].contiguous(), r = matrix(saved[2]);
            c10::DeviceGuard guard(dy.device());
            dx = at::empty({n, h}, x.options());
            Tensor scratch;
            size_t bytes = 0;
            if (want_w) {
                dw = at::empty(w.sizes(), w.options());
                bytes = lib.rms_norm_backward_scratch_bytes(n, static_cast<int>(h), row_type(x));
                if (bytes > 0) scratch = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
            }
            check(lib.rms_norm_backward(ptr(x), row_stride(x), ptr(r), row_stride(r), ptr(w), is_f32(w), n,
                                        static_cast<int>(h), static_cast<float>(ctx->saved_data["eps"].toDouble()),
                                        row_type(x), ptr(dy), row_stride(dy), ptr(ds), row_stride(ds), out(dx), h,
                                        out(dw), out(scratch), bytes, stream(x)),
                  "mignn_rms_norm_backward");
        }
        return first_order({dx, dw, residual ? dx : Tensor(), Tensor()});
    }
};

py::object rms_norm(const Tensor& x, const Tensor& w, const OptTensor& r, double eps) {
    if (x.dim() != 2) throw py::value_error("rms_norm: x must be [N, H], got " + shape(x));
    check_rows("rms_norm", x);
    const int64_t h = x.size(1);
    if (h < 1 || h > MIGNN_RMS_NORM_MAX_H)
        throw py::value_error("rms_norm: width " + std::to_string(h) + " is not in 1.." +
                              std::to_string(MIGNN_RMS_NORM_MAX_H));
    if (w.dim() != 1 || w.size(0) != h)
        throw py::value_error("rms_norm: weight must be [" + std::to_string(h) + "], got " + shape(w));
    if (!is_f32(w) && w.scalar_type() != x.scalar_type())
        throw py::type_error("rms_norm: weight must be float32 or " + dtype(x) + ", got " + dtype(w));
    if (r.has_value() && (r->sizes() != x.sizes() || r->scalar_type() != x.scalar_type()))
        throw py::value_error("rms_norm: residual must be " + shape(x) + " " + dtype(x) + ", got " + shape(*r) + " " +
                              dtype(*r));
    if (!(eps >= 0.0)) throw py::value_error("rms_norm: eps must not be negative, got " + number(eps));
    const Tensor res = value(r);
    no_tangents("rms_norm", {{"x", &x}, {"weight", &w}, {"residual", &res}});
    on_device("rms_norm", x, {{"weight", &w}, {"residual", &res}});
    if (needs_grad({&x, &w}) || (r.has_value() && needs_grad({&*r}))) {
        variable_list o = RMSNorm::apply(x, w, r, eps);
        if (o.size() == 1) return py::cast(o[0]);
        return py::make_tuple(o[0], o[1]);
    }
    auto [y, s] = norm_forward(x, w, value(r), eps);
    if (!s.defined()) return py::cast(y);
    return py::make_tuple(y, s);
}

// ---------------------------------------------------------------------------
// Rotary positions

// [rows, heads, d] with contiguous columns; align: bytes that the pointer and
// the strides are multiples of, the strides then also within the kernels'
// 32-bit offsets (a copy if need be)
Tensor heads_of(const Tensor& t, int64_t align = 1) {
    if (t.size(2) > 1 && t.stride(2) != 1) return copied(t);
    if (align > 1) {
        const int64_t es = t.element_size(), a = t.stride(0), b = t.stride(1);
        if ((reinterpret_cast<int64_t>(t.const_data_ptr()) | a * es | b * es) % align ||
            std::max(a, b) > MIGNN_CROSS_MAX_STRIDE)
            return copied(t);
    }
    return t;
}

Tensor turn(const Tensor& x_, const Tensor& pos_, const Tensor& freq, const Tensor& axis, bool interleaved,
            bool inverse) {
    c10::DeviceGuard guard(x_.device());
    const Tensor x = heads_of(x_);
    const Tensor pos = pos_.size(1) > 1 && pos_.stride(1) != 1 ? pos_.contiguous() : pos_;
    const int pos_type = is_f32(pos) ? MIGNN_POS_F32 : pos.scalar_type() == at::kDouble ? MIGNN_POS_F64
                         : pos.scalar_type() == at::kInt ? MIGNN_POS_I32 : MIGNN_POS_I64;
    const int64_t n = x.size(0), heads = x.size(1), d = x.size(2);
    Tensor y = at::empty({n, heads, d}, x.options());
    reads(freq), reads(axis);
    check(lib.rotary(ptr(x), x.stride(0), x.stride(1), n, static_cast<int>(heads), static_cast<int>(d), ptr(pos),
                     pos_type, pos.stride(0), static_cast<const double*>(ptr(freq)),
                     static_cast<const int32_t*>(ptr(axis)), static_cast<int>(freq.numel()), interleaved, inverse,
                     row_type(x), out(y), heads * d, d, stream(x)),
          "mignn_rotary");
    return y;
}

struct Rotary : torch::autograd::Function<Rotary> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& pos, const Tensor& freq,
                          const Tensor& axis, bool interleaved) {
        ctx->save_for_backward({pos});
        // the axes' tables: out of the hooks' reach
        ctx->saved_data["freq"] = freq;
        ctx->saved_data["axis"] = axis;
        ctx->saved_data["axes"] = pos.size(1);
        ctx->saved_data["pos_type"] = static_cast<int64_t>(pos.scalar_type());
        ctx->saved_data["interleaved"] = interleaved;
        return turn(x, pos, freq, axis, interleaved, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor pos = ctx->get_saved_variables()[0];
        returned("rotary", "pos", pos, grads[0],
                 static_cast<int64_t>(pos.scalar_type()) == ctx->saved_data["pos_type"].toInt(),
                 {grads[0].size(0), ctx->saved_data["axes"].toInt()});
        return first_order({turn(grads[0], pos, ctx->saved_data["freq"].toTensor(),
                                 ctx->saved_data["axis"].toTensor(), ctx->saved_data["interleaved"].toBool(), true),
                            Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor rotary(const Tensor& x, const Tensor& pos, const Tensor& freq, const Tensor& axis, int64_t axes,
              bool interleaved) {
    if (x.dim() != 3) throw py::value_error("rotary: x must be [N, heads, d], got " + shape(x));
    check_rows("rotary", x);
    if (pos.dim() != 2 || pos.size(0) != x.size(0) || pos.size(1) != axes)
        throw py::value_error("rotary: pos must be [" + std::to_string(x.size(0)) + ", " + std::to_string(axes) +
                              "], got " + shape(pos));
    const auto pt = pos.scalar_type();
    if (pt != at::kFloat && pt != at::kDouble && pt != at::kInt && pt != at::kLong)
        throw py::type_error("rotary: pos must be float32, float64, int32 or int64, got " + dtype(pos));
    if (2 * freq.numel() > x.size(2))
        throw py::value_error("rotary: " + std::to_string(freq.numel()) + " pairs do not fit heads of width " +
                              std::to_string(x.size(2)));
    if (needs_grad({&pos})) not_implemented("rotary: positions get no gradient (pass pos.detach())");
    no_tangents("rotary", {{"x", &x}, {"pos", &pos}});
    on_device("rotary", x, {{"pos", &pos}, {"axes", &freq}});
    if (needs_grad({&x})) return Rotary::apply(x, pos, freq, axis, interleaved);
    return turn(x, pos, freq, axis, interleaved, false);
}

// ---------------------------------------------------------------------------
// Cross attention

// A plan's call moved from its lists at `from` to the same bytes at `to`
mignn_cross_call moved(mignn_cross_call c, const void* from, const void* to) {
    const uintptr_t by = reinterpret_cast<uintptr_t>(to) - reinterpret_cast<uintptr_t>(from);
    for (mignn_cross_pass& p : c.pass) {
        p.items = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p.items) + by);
        p.joins = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p.joins) + by);
    }
    return c;
}

// a plan's call, with the tensors of one use filled in
mignn_cross_call call_of(const mignn_cross_call& plan, const Tensor& q, const Tensor& k, const Tensor& v,
                         const Tensor& mask, double scale, const Tensor& scratch) {
    mignn_cross_call c = plan;
    c.q = ptr(q), c.k = ptr(k), c.v = ptr(v);
    c.key_mask = static_cast<const uint8_t*>(ptr(mask));
    c.ldq = q.stride(0), c.ldqh = q.stride(1);
    c.ldk = k.stride(0), c.ldkh = k.stride(1);
    c.ldv = v.stride(0), c.ldvh = v.stride(1);
    c.scale = static_cast<float>(scale);
    c.scratch = out(scratch);
    c.scratch_bytes = scratch.defined() ? scratch.numel() : 0;
    return c;
}

Tensor scratch_for(int64_t bytes, const Tensor& t) {
    return bytes > 0 ? at::empty({bytes}, t.options().dtype(at::kByte)) : Tensor();
}

struct CrossOut {
    Tensor out, out32, lse;
};

CrossOut cross_forward(const mignn_cross_call& plan, const Tensor& q_, const Tensor& k_, const Tensor& v_,
                       const Tensor& mask, const Tensor& lists, double scale, bool train) {
    c10::DeviceGuard guard(q_.device());
    reads(lists);
    const Tensor q = heads_of(q_, 16), k = heads_of(k_, 16), v = heads_of(v_, 16);
    CrossOut o;
    o.out = at::empty(q.sizes(), q.options());
    if (train) {
        o.lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
        if (!is_f32(q)) o.out32 = at::empty(q.sizes(), q.options().dtype(at::kFloat));
    }
    const Tensor scratch = scratch_for(plan.pass[MIGNN_CROSS_FORWARD].part_bytes, q);
    const mignn_cross_call c = call_of(plan, q, k, v, mask, scale, scratch);
    check(lib.cross_attn_forward(&c, out(o.out), static_cast<float*>(out(o.out32)),
                                 static_cast<float*>(out(o.lse)), stream(q)),
          "mignn_cross_attn_forward");
    if (!o.out32.defined()) o.out32 = o.out;
    return o;
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const OptTensor& mask, const Tensor& lists, uint64_t plan, double scale) {
        const auto& c = *reinterpret_cast<const mignn_cross_call*>(plan);
        const CrossOut o = cross_forward(c, q, k, v, value(mask), lists, scale, true);
        // out32 (the fp32 output): <do, o> from the rounded output would leave
        // the rounding of o in every dS
        ctx->save_for_backward({q, k, v, value(mask), o.out32, o.lse});
        // The plan may be gone by the backward, and saved tensors may come back as
        // others (saved-tensor hooks, checkpointing): the lists are held here,
        // out of the hooks' reach, and the call holds distances into them
        const mignn_cross_call placed = moved(c, ptr(lists), nullptr);
        ctx->saved_data["lists"] = lists;
        ctx->saved_data["plan"] = std::string(reinterpret_cast<const char*>(&placed), sizeof(placed));
        ctx->saved_data["scale"] = scale;
        return o.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        mignn_cross_call plan;
        std::memcpy(&plan, ctx->saved_data["plan"].toStringRef().data(), sizeof(plan));
        const Tensor lists = ctx->saved_data["lists"].toTensor();
        plan = moved(plan, nullptr, ptr(lists));
        const Tensor& g = grads[0];
        auto rows = [&](int i, const char* name, at::IntArrayRef sizes) {
            const bool type_ok = saved[i].scalar_type() == g.scalar_type();
            return heads_of(returned("cross_attention", name, saved[i], g, type_ok, sizes), 16);
        };
        auto flat = [&](int i, const char* name, at::ScalarType type, at::IntArrayRef sizes) {
            const bool type_ok = saved[i].scalar_type() == type;
            return returned("cross_attention", name, saved[i], g, type_ok, sizes).contiguous();
        };
        const std::array<int64_t, 3> key_rows{plan.n_keys, plan.kv_heads, plan.d};
        c10::DeviceGuard guard(g.device());
        const Tensor q = rows(0, "q", g.sizes()), k = rows(1, "k", key_rows), v = rows(2, "v", key_rows);
        const Tensor mask = saved[3].defined() ? flat(3, "key_mask", at::kBool, {plan.n_keys}) : Tensor();
        const Tensor out32 = flat(4, "output", at::kFloat, g.sizes());
        const Tensor lse = flat(5, "statistics", at::kFloat, {g.size(0), g.size(1)});
        const Tensor dout = heads_of(g, 16);
        reads(lists);
        Tensor dq = at::empty(q.sizes(), q.options()), dk, dv;
        const bool keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
        if (keys) {
            dk = at::empty(k.sizes(), k.options());
            dv = at::empty(v.sizes(), v.options());
        }
        const Tensor delta = at::empty(lse.sizes(), lse.options());
        const Tensor scratch = scratch_for(std::max(plan.pass[MIGNN_CROSS_DQ].part_bytes,
                                                    plan.pass[MIGNN_CROSS_DKV].part_bytes), q);
        const mignn_cross_call c = call_of(plan, q, k, v, mask, ctx->saved_data["scale"].toDouble(), scratch);
        check(lib.cross_attn_backward(&c, ptr(dout), dout.stride(0), dout.stride(1),
                                      static_cast<const float*>(ptr(out32)), static_cast<const float*>(ptr(lse)),
                                      static_cast<float*>(out(delta)), out(dq), out(dk), out(dv), stream(q)),
              "mignn_cross_attn_backward");
        if (!ctx->needs_input_grad(0)) dq = Tensor();
        if (!ctx->needs_input_grad(1)) dk = Tensor();
        if (!ctx->needs_input_grad(2)) dv = Tensor();
        return first_order({dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_mask,
                       const c10::optional<double>& scale_, const Tensor& lists, uint64_t plan, int64_t queries,
                       bool train) {
    const auto& c = *reinterpret_cast<const mignn_cross_call*>(plan);
    const std::array<int64_t, 3> want_q{queries, c.heads, c.d}, want_k{c.n_keys, c.kv_heads, c.d};
    const auto type = c.dtype == MIGNN_ROW_F32 ? at::kFloat : c.dtype == MIGNN_ROW_BF16 ? at::kBFloat16 : at::kHalf;
    auto check_like = [&](const char* name, const Tensor& t, const std::array<int64_t, 3>& want) {
        if (t.sizes() != at::IntArrayRef(want))
            throw py::value_error(std::string("cross_attention: the plan's ") + name + " is " + shape(want) +
                                  ", got " + shape(t));
        if (t.scalar_type() != type)
            throw py::type_error(std::string("cross_attention: the plan's rows are ") +
                                 dtype(at::empty({0}, type)) + ", " + name + " is " + dtype(t));
    };
    check_like("q", q, want_q), check_like("k", k, want_k), check_like("v", v, want_k);
    Tensor mask = value(key_mask);
    if (mask.defined() && (mask.scalar_type() != at::kBool || mask.dim() != 1 || mask.size(0) != c.n_keys))
        throw py::value_error("cross_attention: key_mask must be bool [" + std::to_string(c.n_keys) + "], got " +
                              dtype(mask) + " " + shape(mask));
    const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt(static_cast<double>(c.d));
    if (!(scale > 0.0 && scale < 1e30))
        throw py::value_error("cross_attention: scale must be positive and finite, got " + number(scale));
    no_tangents("cross_attention", {{"q", &q}, {"k", &k}, {"v", &v}});
    on_device("cross_attention", q, {{"k", &k}, {"v", &v}, {"key_mask", &mask}, {"plan", &lists}});
    if (mask.defined()) mask = mask.contiguous();
    const bool grad = needs_grad({&q, &k, &v});
    if (grad && !train) throw py::value_error("cross_attention: gradients need a plan built with train=True");
    if (grad)
        return CrossAttention::apply(q, k, v, mask.defined() ? OptTensor(mask) : OptTensor(), lists, plan,
                                     scale);
    return cross_forward(c, q, k, v, mask, lists, scale, false).out;
}

// The addresses of a plan's lists (each pass's items and joins), as a backward
// forms them that finds the lists at `at`
std::vector<uint64_t> plan_places(uint64_t plan, const Tensor& lists, const Tensor& at) {
    const mignn_cross_call c = moved(
        moved(*reinterpret_cast<const mignn_cross_call*>(plan), ptr(lists), nullptr), nullptr, ptr(at));
    std::vector<uint64_t> places;
    for (const mignn_cross_pass& p : c.pass)
        for (const void* a : {p.items, p.joins}) places.push_back(reinterpret_cast<uint64_t>(a));
    return places;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "row operators over libmignn (mignn.attention)";
    m.def("bind", &bind);
    m.def("rms_norm", &rms_norm);
    m.def("rotary", &rotary);
    m.def("cross_attention", &cross_attention);
    m.def("plan_places", &plan_places);
}
