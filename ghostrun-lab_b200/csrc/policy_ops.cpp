// PyTorch binding of the policy operators (norm.py, heads.py): argument checks, output and work tensors, the current stream
// and the autograd nodes, around the C-ABI entry points of librlenv_b200.so. In C++ because the host's time is what a small
// call costs: layer norm of 4,096 x 512 with its gradients takes 150 us through ctypes and a Python autograd function, 101 us
// this way, against 13 us on the GPU. The library is not linked: bind() is given its functions' addresses, so that the one
// library that the process has loaded is the one that runs.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>
#include <limits>
#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "../../include/rlenv_api.h"   // the entry points' types

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct Library {
    decltype(&rl_norm_fwd) norm_fwd = nullptr;
    decltype(&rl_norm_bwd_work_bytes) norm_bwd_work_bytes = nullptr;
    decltype(&rl_norm_bwd) norm_bwd = nullptr;
    decltype(&rl_norm_error) norm_error = nullptr;
    decltype(&rl_moves_sample) moves_sample = nullptr;
    decltype(&rl_sample) sample = nullptr;
    decltype(&rl_moves_logp) moves_logp = nullptr;
    decltype(&rl_moves_logp_bwd_work_bytes) moves_logp_bwd_work_bytes = nullptr;
    decltype(&rl_moves_logp_bwd) moves_logp_bwd = nullptr;
    decltype(&rl_heads_error) heads_error = nullptr;
};

// The functions that calls use: all ten at once, since a backward may run while another library is bound. An older table
// stays, a call may be in it.
std::atomic<const Library*> bound{nullptr};

const Library& library() {
    const Library* lib = bound.load(std::memory_order_acquire);
    TORCH_CHECK(lib, "policy_ops_b200 has no library yet: policy_ops.load() gives it one");
    return *lib;
}

template <class F>
void take(const py::dict& addresses, const char* name, F& f) {
    f = reinterpret_cast<F>(py::cast<uintptr_t>(addresses[name]));
}

void bind(const py::dict& at) {
    auto lib = std::make_unique<Library>();
    take(at, "rl_norm_fwd", lib->norm_fwd);
    take(at, "rl_norm_bwd_work_bytes", lib->norm_bwd_work_bytes);
    take(at, "rl_norm_bwd", lib->norm_bwd);
    take(at, "rl_norm_error", lib->norm_error);
    take(at, "rl_moves_sample", lib->moves_sample);
    take(at, "rl_sample", lib->sample);
    take(at, "rl_moves_logp", lib->moves_logp);
    take(at, "rl_moves_logp_bwd_work_bytes", lib->moves_logp_bwd_work_bytes);
    take(at, "rl_moves_logp_bwd", lib->moves_logp_bwd);
    take(at, "rl_heads_error", lib->heads_error);
    bound.store(lib.release(), std::memory_order_release);
}

// The library's number of a type; -1: none of its three.
int type_of(at::ScalarType t) {
    return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}
int type_of(const Tensor& t) { return type_of(t.scalar_type()); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

const void* at_or_null(const MaybeTensor& t) { return t ? t->const_data_ptr() : nullptr; }
void* out_or_null(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

Tensor make(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
    const at::AutoDispatchBelowADInplaceOrView below;   // a new tensor has no history to keep
    return at::empty(shape, like.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
}

// t as [rows, width] with adjacent columns (a view where its strides allow one).
Tensor rows_of(const Tensor& t, int64_t width) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
    return width == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

// Forward-mode derivatives are not there: an input that carries one is refused, where the result would be without it.
void no_tangent(const char* what, const Tensor& t) {
    TORCH_CHECK(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), what,
                ": an input has a forward-mode derivative, which this operator does not carry");
}
void no_tangent(const char* what, const MaybeTensor& t) {
    if (t) no_tangent(what, *t);
}

// What a gradient that has no graph of its own is given where the caller keeps one (create_graph): the error comes when a
// second derivative is asked for.
variable_list without_graph(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (auto& g : grads)
        if (g.defined()) some.push_back(g.detach().requires_grad_(true));
    if (some.empty()) return grads;
    auto node = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + ": the gradients have no derivatives of their own", static_cast<int64_t>(some.size()));
    some = (*node)(std::move(some));
    size_t n = 0;
    for (auto& g : grads)
        if (g.defined()) g = some[n++];
    return grads;
}

// ------------------------------------------------------------------ layer norm

struct Normed {
    Tensor y, sum, rows, stats;   // sum: undefined without a residual; rows: what was normalised; stats: undefined unless wanted
};

Normed norm_forward(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, const MaybeTensor& residual,
                    at::ScalarType out_type, bool want_stats) {
    const Library& lib = library();
    const int64_t width = x.size(-1);
    const Tensor x2 = rows_of(x, width), r2 = residual ? rows_of(*residual, width) : Tensor();
    const MaybeTensor w = weight ? MaybeTensor(weight->contiguous()) : std::nullopt;
    const MaybeTensor b = bias ? MaybeTensor(bias->contiguous()) : std::nullopt;
    Normed n;
    const int64_t rows = x2.size(0);
    n.y = make(x.sizes(), out_type, x);
    if (residual) n.sum = make(x.sizes(), x.scalar_type(), x);
    if (want_stats) n.stats = make({rows, 2}, at::kFloat, x);
    const int rc = lib.norm_fwd(x2.const_data_ptr(), residual ? r2.const_data_ptr() : nullptr, at_or_null(w), at_or_null(b),
                                n.y.mutable_data_ptr(), out_or_null(n.sum), out_or_null(n.stats), rows, width, x2.stride(0),
                                residual ? r2.stride(0) : 0, type_of(x), type_of(out_type), w ? type_of(*w) : b ? type_of(*b) : 0,
                                static_cast<float>(eps), stream_of(x));
    TORCH_CHECK(rc == 0, "rl_norm_fwd: ", lib.norm_error());
    n.rows = residual ? n.sum : x2;
    return n;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias,
                                 const MaybeTensor& residual, double eps, at::ScalarType out_type) {
        ctx->set_materialize_grads(false);
        const Normed n = norm_forward(x, weight, bias, eps, residual, out_type, true);
        ctx->save_for_backward({n.rows, n.stats, weight ? weight->contiguous() : Tensor()});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["weight"] = weight.has_value();
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["w_type"] = static_cast<int64_t>(weight ? weight->scalar_type() : bias ? bias->scalar_type() : at::kFloat);
        return residual ? variable_list{n.y, n.sum} : variable_list{n.y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Library& lib = library();
        const auto saved = ctx->get_saved_variables();
        const Tensor &s = saved[0], &stats = saved[1], &weight = saved[2];
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const auto w_type = static_cast<at::ScalarType>(ctx->saved_data["w_type"].toInt());
        size_t edge = 0;   // of the inputs that were given, in their order
        const bool need_x = ctx->needs_input_grad(edge++);
        const bool need_w = ctx->saved_data["weight"].toBool() && ctx->needs_input_grad(edge++);
        const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(edge++);
        const bool need_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge++);
        const int64_t width = shape.back(), rows = stats.size(0);
        const Tensor gsum = grads.size() > 1 ? grads[1] : Tensor();
        Tensor dx, dw, db;
        const c10::cuda::CUDAGuard guard(s.device());
        if (rows == 0 || !grads[0].defined()) {   // nothing came through the norm: the stream's gradient passes as it is
            if (rows == 0) dx = make(shape, s.scalar_type(), s);
            else dx = gsum;
            if (need_w) dw = at::zeros({width}, s.options().dtype(w_type));
            if (need_b) db = at::zeros({width}, s.options().dtype(w_type));
        } else {
            const Tensor s2 = rows_of(s, width), gy = rows_of(grads[0], width);
            const Tensor gs = gsum.defined() ? rows_of(gsum, width) : Tensor();
            Tensor work;
            size_t bytes = 0;
            if (need_x || need_r) dx = make(shape, s.scalar_type(), s);
            if (need_w || need_b) {
                bytes = lib.norm_bwd_work_bytes(rows, width);
                work = make({static_cast<int64_t>(bytes / 4)}, at::kFloat, s);
            }
            if (need_w) dw = make({width}, w_type, s);
            if (need_b) db = make({width}, w_type, s);
            const int rc = lib.norm_bwd(gy.const_data_ptr(), gs.defined() ? gs.const_data_ptr() : nullptr, s2.const_data_ptr(),
                                        stats.const_data_ptr(), weight.defined() ? weight.const_data_ptr() : nullptr,
                                        out_or_null(dx), out_or_null(dw), out_or_null(db), rows, width, gy.stride(0),
                                        gs.defined() ? gs.stride(0) : 0, s2.stride(0), type_of(s), type_of(gy), type_of(w_type),
                                        out_or_null(work), bytes, stream_of(s));
            TORCH_CHECK(rc == 0, "rl_norm_bwd: ", lib.norm_error());
        }
        return without_graph({need_x ? dx : Tensor(), dw, db, need_r ? dx : Tensor(), Tensor(), Tensor()}, "layer_norm");
    }
};

void check_param(const char* name, const MaybeTensor& t, const Tensor& x) {
    TORCH_CHECK(!t || (t->dim() == 1 && t->size(0) == x.size(-1) && type_of(*t) >= 0 && t->device() == x.device()),
                "layer_norm: ", name, " must be [", x.size(-1), "], fp32, bf16 or fp16, on ", x.device(), "; got ", t->sizes(), " ",
                t->scalar_type(), " on ", t->device());
}

bool wants_grad(const MaybeTensor& t) { return t && t->requires_grad(); }

py::object layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, const MaybeTensor& residual,
                      std::optional<at::ScalarType> out_dtype) {
    const at::ScalarType out_type = out_dtype.value_or(x.scalar_type());
    TORCH_CHECK(x.is_cuda(), "layer_norm runs on the GPU only");
    TORCH_CHECK(type_of(x) >= 0, "layer_norm: x must be fp32, bf16 or fp16, got ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: x needs a last axis of at least one value, got shape ", x.sizes());
    check_param("weight", weight, x);
    check_param("bias", bias, x);
    TORCH_CHECK(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "layer_norm: weight (", weight->scalar_type(),
                ") and bias (", bias->scalar_type(), ") must have one type");
    TORCH_CHECK(!residual || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() &&
                              residual->device() == x.device()),
                "layer_norm: the residual must be as x, ", x.sizes(), " ", x.scalar_type(), " on ", x.device(), "; got ",
                residual->sizes(), " ", residual->scalar_type(), " on ", residual->device());
    TORCH_CHECK(out_type == x.scalar_type() || out_type == at::kFloat, "layer_norm: out_dtype must be ", x.scalar_type(),
                " or fp32, got ", out_type);
    no_tangent("layer_norm", x);
    for (const MaybeTensor* t : {&weight, &bias, &residual}) no_tangent("layer_norm", *t);
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y, sum;
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))) {
        const variable_list out = LayerNorm::apply(x, weight, bias, residual, eps, out_type);
        y = out[0];
        if (residual) sum = out[1];
    } else {
        const Normed n = norm_forward(x, weight, bias, eps, residual, out_type, false);
        y = n.y;
        sum = n.sum;
    }
    return residual ? py::object(py::make_tuple(y, sum)) : py::cast(y);
}

// ------------------------------------------------------------------ heads

constexpr int64_t kBytes = 19, kMoves = 324, kMaxWidth = 4096, kCond = 127;
constexpr int64_t kTables[10][2] = {{9, 3}, {9, 3}, {3, 3}, {9, 2}, {3, 2}, {3, 2}, {9, 2}, {3, 2}, {3, 2}, {2, 2}};

Tensor adjacent(const Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous(); }

Tensor check_logits(const char* what, const Tensor& l, int64_t width) {
    TORCH_CHECK(l.is_cuda(), what, " runs on the GPU only");
    TORCH_CHECK(l.dim() == 2 && type_of(l) >= 0 && (width == 0 || l.size(1) == width), what, ": logits must be [B, ",
                width ? std::to_string(width) : std::string("V"), "] fp32, bf16 or fp16, got ", l.sizes(), " ", l.scalar_type());
    return adjacent(l);
}

Tensor check_bytes(const char* what, const char* name, const Tensor& t, const Tensor& logits, int64_t width, int64_t or_width) {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == logits.size(0) && (t.size(1) == width || t.size(1) == or_width) &&
                    (t.scalar_type() == at::kByte || t.scalar_type() == at::kBool) && t.device() == logits.device(),
                what, ": ", name, " must be [", logits.size(0), ", ", width, "] bytes (uint8 or bool) on ", logits.device(), ", got ",
                t.sizes(), " ", t.scalar_type(), " on ", t.device());
    return adjacent(t);
}

Tensor check_row(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type, const Tensor& logits) {
    TORCH_CHECK(t.sizes() == shape && t.scalar_type() == type && t.device() == logits.device(), what, ": ", name, " must be ", shape,
                " ", type, " on ", logits.device(), ", got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
    return t.contiguous();
}

std::vector<Tensor> check_cond(const char* what, const std::optional<std::vector<Tensor>>& cond, const Tensor& logits) {
    std::vector<Tensor> out;
    if (!cond) return out;
    TORCH_CHECK(cond->size() == 10, what, ": cond must be ten tables, got ", cond->size());
    for (int t = 0; t < 10; ++t) {
        const Tensor& c = (*cond)[t];
        TORCH_CHECK(c.sizes() == at::IntArrayRef(kTables[t], 2) && type_of(c) >= 0 && c.scalar_type() == (*cond)[0].scalar_type() &&
                        c.device() == logits.device(),
                    what, ": table ", t, " of cond must be ", at::IntArrayRef(kTables[t], 2), ", fp32, bf16 or fp16 as the others, on ",
                    logits.device(), "; got ", c.sizes(), " ", c.scalar_type(), " on ", c.device());
        out.push_back(c.contiguous());
    }
    return out;
}

// The tables as the library takes them.
struct Tables {
    const void* at[10];
    const void* const* given;
    int type;
    explicit Tables(at::ArrayRef<Tensor> cond) : given(cond.empty() ? nullptr : at), type(cond.empty() ? 0 : type_of(cond[0])) {
        for (size_t t = 0; t < cond.size(); ++t) at[t] = cond[t].const_data_ptr();
    }
};

// temperature, top_k, top_p, min_p: a number each, or a tensor with one for each row.
struct Cut {
    double number[4] = {1.0, 0.0, 1.0, 0.0};
    Tensor each[4];

    Cut(const char* what, const Tensor& logits, const py::object (&given)[4]) {
        static const char* const names[4] = {"temperature", "top_k", "top_p", "min_p"};
        for (int i = 0; i < 4; ++i) {
            if (THPVariable_Check(given[i].ptr())) {
                const Tensor t = THPVariable_Unpack(given[i].ptr());
                const auto type = t.scalar_type();
                TORCH_CHECK(t.dim() == 1 && t.size(0) == logits.size(0) && t.device() == logits.device() &&
                                (i == 1 ? at::isIntegralType(type, false) : at::isIntegralType(type, false) || at::isFloatingType(type)),
                            what, ": ", names[i], " must be a number or [", logits.size(0), "] on ", logits.device(), ", got ", t.sizes(),
                            " ", type, " on ", t.device());
                Tensor v = t.detach();
                if (i == 1 && v.element_size() > 2 && type != at::kInt)   // numbers past 31 bits are no row's width, not their low bits
                    v = v.to(at::kLong).clamp(0, std::numeric_limits<int>::max());
                each[i] = v.to(i == 1 ? at::kInt : at::kFloat).contiguous();
            } else {
                TORCH_CHECK(PyFloat_Check(given[i].ptr()) || PyLong_Check(given[i].ptr()) || PyIndex_Check(given[i].ptr()) ||
                                PyNumber_Check(given[i].ptr()),
                            what, ": ", names[i], " must be a number or a tensor");
                number[i] = py::cast<double>(py::float_(given[i]));
            }
        }
        const double k = number[1];
        TORCH_CHECK(number[0] >= 0 && number[2] >= 0 && number[3] <= 1 && k >= 0 && k < 2147483648.0 && std::floor(k) == k, what,
                    ": temperature and top_p must be 0 or more, top_k a whole number of 0 or more, min_p at most 1; got temperature ",
                    number[0], ", top_k ", k, ", top_p ", number[2], ", min_p ", number[3]);
    }
    float value(int i) const { return static_cast<float>(number[i]); }
    int top_k() const { return static_cast<int>(number[1]); }
    const void* at(int i) const { return each[i].defined() ? each[i].const_data_ptr() : nullptr; }
};

py::tuple sample_moves(const Tensor& logits_, const std::optional<std::vector<Tensor>>& cond_, const Tensor& masks_, const Tensor& u_,
                       const py::object& temperature, const py::object& top_k, const py::object& top_p, const py::object& min_p) {
    const char* what = "sample_moves";
    const Library& lib = library();
    const Tensor logits = check_logits(what, logits_, kBytes);
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t rows = logits.size(0);
    const auto cond = check_cond(what, cond_, logits);
    const Tensor masks = check_bytes(what, "masks", masks_, logits, kBytes, kBytes);
    const Tensor u = check_row(what, "u", u_, {rows, 5}, at::kFloat, logits);
    const Cut cut(what, logits, {temperature, top_k, top_p, min_p});
    const Tensor ids = make({rows}, at::kShort, logits), logp = make({rows}, at::kFloat, logits);
    const Tables tables(cond);
    const int rc = lib.moves_sample(logits.const_data_ptr(), logits.stride(0), type_of(logits), tables.given, tables.type,
                                    masks.const_data_ptr(), masks.stride(0), u.const_data_ptr(), cut.value(0), cut.top_k(), cut.value(2),
                                    cut.value(3), cut.at(0), cut.at(1), cut.at(2), cut.at(3), ids.mutable_data_ptr(),
                                    logp.mutable_data_ptr(), rows, stream_of(logits));
    TORCH_CHECK(rc == 0, "rl_moves_sample: ", lib.heads_error());
    return py::make_tuple(ids, logp);
}

py::tuple sample(const Tensor& logits_, const Tensor& u_, const MaybeTensor& legal_, const py::object& temperature,
                 const py::object& top_k, const py::object& top_p, const py::object& min_p) {
    const char* what = "sample";
    const Library& lib = library();
    const Tensor logits = check_logits(what, logits_, 0);
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t rows = logits.size(0), width = logits.size(1);
    TORCH_CHECK(width >= 1 && width <= kMaxWidth, "sample: rows must have 1 to ", kMaxWidth, " choices, got ", width);
    MaybeTensor legal;
    if (legal_) legal = check_bytes(what, "legal", *legal_, logits, width, width == kMoves ? kBytes : width);
    const Tensor u = check_row(what, "u", u_, {rows}, at::kFloat, logits);
    const Cut cut(what, logits, {temperature, top_k, top_p, min_p});
    const Tensor choice = make({rows}, at::kLong, logits), logp = make({rows}, at::kFloat, logits);
    const int rc = lib.sample(logits.const_data_ptr(), logits.stride(0), type_of(logits), static_cast<int>(width), at_or_null(legal),
                              legal ? legal->stride(0) : 0, legal ? static_cast<int>(legal->size(1)) : 0, u.const_data_ptr(),
                              cut.value(0), cut.top_k(), cut.value(2), cut.value(3), cut.at(0), cut.at(1), cut.at(2), cut.at(3),
                              choice.mutable_data_ptr(), logp.mutable_data_ptr(), rows, stream_of(logits));
    TORCH_CHECK(rc == 0, "rl_sample: ", lib.heads_error());
    return py::make_tuple(choice, logp);
}

variable_list logp_forward(const Tensor& logits, const Tensor& masks, const Tensor& ids, at::TensorList cond) {
    const Library& lib = library();
    const int64_t rows = logits.size(0);
    const Tensor logp = make({rows}, at::kFloat, logits), entropy = make({rows}, at::kFloat, logits);
    const Tables tables(cond);
    const int rc = lib.moves_logp(logits.const_data_ptr(), logits.stride(0), type_of(logits), tables.given, tables.type,
                                  masks.const_data_ptr(), masks.stride(0), ids.const_data_ptr(), logp.mutable_data_ptr(),
                                  entropy.mutable_data_ptr(), rows, stream_of(logits));
    TORCH_CHECK(rc == 0, "rl_moves_logp: ", lib.heads_error());
    return {logp, entropy};
}

struct MovesLogp : torch::autograd::Function<MovesLogp> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& masks, const Tensor& ids, at::TensorList cond) {
        ctx->set_materialize_grads(false);
        variable_list keep{logits, masks, ids};
        keep.insert(keep.end(), cond.begin(), cond.end());
        ctx->save_for_backward(std::move(keep));
        return logp_forward(logits, masks, ids, cond);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return without_graph(gradients(ctx, std::move(grads)), "moves_logp");
    }

    static variable_list gradients(AutogradContext* ctx, variable_list grads) {
        const Library& lib = library();
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &masks = saved[1], &ids = saved[2];
        const at::ArrayRef<Tensor> cond = at::ArrayRef<Tensor>(saved).slice(3);
        const Tensor &glp = grads[0], &gent = grads[1];
        const int64_t rows = logits.size(0);
        bool need_cond = false;
        for (size_t t = 0; t < cond.size(); ++t) need_cond |= ctx->needs_input_grad(3 + t);
        const c10::cuda::CUDAGuard guard(logits.device());
        Tensor dlogits, dcond, work;
        if (ctx->needs_input_grad(0)) dlogits = make({rows, kBytes}, logits.scalar_type(), logits);
        if (need_cond) dcond = make({kCond}, at::kFloat, logits);
        if (rows == 0 || (!glp.defined() && !gent.defined())) {
            if (dlogits.defined()) dlogits.zero_();
            if (dcond.defined()) dcond.zero_();
        } else {
            size_t bytes = 0;
            if (need_cond) {
                bytes = lib.moves_logp_bwd_work_bytes();
                work = make({static_cast<int64_t>(bytes / 4)}, at::kFloat, logits);
            }
            const Tables tables(cond);
            const int rc = lib.moves_logp_bwd(glp.defined() ? glp.const_data_ptr() : nullptr, glp.defined() ? glp.stride(0) : 0,
                                              gent.defined() ? gent.const_data_ptr() : nullptr, gent.defined() ? gent.stride(0) : 0,
                                              logits.const_data_ptr(), logits.stride(0), type_of(logits), tables.given, tables.type,
                                              masks.const_data_ptr(), masks.stride(0), ids.const_data_ptr(), out_or_null(dlogits),
                                              out_or_null(dcond), rows, out_or_null(work), bytes, stream_of(logits));
            TORCH_CHECK(rc == 0, "rl_moves_logp_bwd: ", lib.heads_error());
        }
        variable_list out{dlogits, Tensor(), Tensor()};
        out.reserve(3 + cond.size());
        const at::AutoDispatchBelowADInplaceOrView below;   // the tables' gradients are parts of one tensor of our own
        int64_t at = 0;
        if (need_cond && cond[0].scalar_type() != at::kFloat) dcond = dcond.to(cond[0].scalar_type());
        for (size_t t = 0; t < cond.size(); ++t) {
            const int64_t a = kTables[t][0], b = kTables[t][1];
            out.push_back(ctx->needs_input_grad(3 + t) ? dcond.as_strided({a, b}, {b, 1}, at) : Tensor());
            at += a * b;
        }
        return out;
    }
};

py::tuple moves_logp(const Tensor& logits_, const std::optional<std::vector<Tensor>>& cond_, const Tensor& masks_, const Tensor& ids_) {
    const char* what = "moves_logp";
    no_tangent(what, logits_);
    if (cond_)
        for (const Tensor& t : *cond_) no_tangent(what, t);
    const Tensor logits = check_logits(what, logits_, kBytes);
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor masks = check_bytes(what, "masks", masks_, logits, kBytes, kBytes);
    const Tensor ids = check_row(what, "ids", ids_, {logits.size(0)}, at::kShort, logits);
    const auto cond = check_cond(what, cond_, logits);
    bool grad = logits.requires_grad();
    for (const Tensor& t : cond) grad |= t.requires_grad();
    const variable_list out = grad && at::GradMode::is_enabled() ? MovesLogp::apply(logits, masks, ids, at::TensorList(cond))
                                                                 : logp_forward(logits, masks, ids, cond);
    return py::make_tuple(out[0], out[1]);
}

}  // namespace

PYBIND11_MODULE(policy_ops_b200, m) {
    m.attr("built_for") = BUILT_FOR;   // build.py looks for it in the file
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm);
    m.def("sample_moves", &sample_moves);
    m.def("sample", &sample);
    m.def("moves_logp", &moves_logp);
}
