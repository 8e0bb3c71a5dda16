// Host side of the operators, in C++: checks of the arguments, outputs and
// workspaces from torch's allocator, autograd, and the calls of the library's
// C ABI on the current stream.
//
// In Python this work took 10 to 20 us a call, and a backward pass 60 us more
// (a ctypes call of a dozen arguments, autograd's way between its own thread
// and the interpreter): longer than many of the kernels.  Here a call takes
// 4 to 6 us and a backward pass needs no interpreter.
//
// The library is bound at run time, by the addresses of its functions, so that
// CRESSO_HIP_LIBRARY chooses it here as it does for ctypes.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <string>

#include "../../include/cresso_hip.h"
#include "overlap.hpp"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&cresso_hip_last_error) last_error;
    decltype(&cresso_embedding_forward) embedding_forward;
    decltype(&cresso_embedding_backward_workspace_bytes) embedding_backward_workspace_bytes;
    decltype(&cresso_embedding_backward) embedding_backward;
    decltype(&cresso_residual_norm_forward) residual_norm_forward;
    decltype(&cresso_residual_norm_backward_workspace_bytes) residual_norm_backward_workspace_bytes;
    decltype(&cresso_residual_norm_backward) residual_norm_backward;
    decltype(&cresso_distill_loss) distill_loss;
    decltype(&cresso_distill_backward) distill_backward;
    decltype(&cresso_block_product_workspace_bytes) block_product_workspace_bytes;
    decltype(&cresso_block_product) block_product;
    decltype(&cresso_block_quantize) block_quantize;
} g_api{};

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
    const auto take = [&](auto& fn, const char* name) {
        const auto it = at.find(name);
        TORCH_CHECK(it != at.end() && it->second, "CRESSO5 CUDA ops failed to load: no ", name);
        fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(it->second);
    };
    Api a{};
    take(a.last_error, "cresso_hip_last_error");
    take(a.embedding_forward, "cresso_embedding_forward");
    take(a.embedding_backward_workspace_bytes, "cresso_embedding_backward_workspace_bytes");
    take(a.embedding_backward, "cresso_embedding_backward");
    take(a.residual_norm_forward, "cresso_residual_norm_forward");
    take(a.residual_norm_backward_workspace_bytes, "cresso_residual_norm_backward_workspace_bytes");
    take(a.residual_norm_backward, "cresso_residual_norm_backward");
    take(a.distill_loss, "cresso_distill_loss");
    take(a.distill_backward, "cresso_distill_backward");
    take(a.block_product_workspace_bytes, "cresso_block_product_workspace_bytes");
    take(a.block_product, "cresso_block_product");
    take(a.block_quantize, "cresso_block_quantize");
    g_api = a;
}

// ---------------------------------------------------------------------------
// what the operators share
// ---------------------------------------------------------------------------
int32_t code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return CRESSO_F32;
        case at::kDouble: return CRESSO_F64;
        case at::kHalf: return CRESSO_F16;
        case at::kBFloat16: return CRESSO_BF16;
        default: return -1;
    }
}
bool row_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
const char* name_of(at::ScalarType t) { return c10::toString(t); }

void check_row_type(const char* what, const char* name, const Tensor& t) {
    TORCH_CHECK_VALUE(row_type(t.scalar_type()), what, ": ", name, " must be fp32, bf16 or fp16, not ", name_of(t.scalar_type()));
}
// Every tensor given lies on one GPU; there is no CPU path.  None is a dual
// tensor: the operators have no forward-mode derivatives, and an output without
// a tangent would say that its derivative is zero.
struct OneGpu {
    const char* what;
    const Tensor* first = nullptr;
    void add(const char* name, const Tensor& t) {
        if (!t.defined()) return;
        TORCH_CHECK(t.is_cuda(), what, ": ", name, " is on ", t.device(), "; the operators run on the GPU only");
        TORCH_CHECK(!t._fw_grad(0).defined(), what, ": ", name, " has a forward-mode derivative, the operators have reverse mode only");
        if (!first) first = &t;
        TORCH_CHECK(t.device() == first->device(), what, ": ", name, " is on ", t.device(), ", others on ", first->device());
    }
};
Tensor or_none(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
optional<Tensor> or_null(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

// t seen as rows of its last dimension: rows at one stride of at least their
// width, whatever dimensions they are counted by, are taken where they lie,
// anything else is copied.
Tensor rows_of(const Tensor& t, int64_t& stride) {
    const int64_t n = t.dim() - 1, width = n >= 0 ? t.size(n) : 1;
    int64_t at = 0, rows = 1;   // the rows' stride, 0 before a dimension has given it; rows counted so far
    bool taken = n >= 0 && (width < 2 || t.stride(n) == 1);
    for (int64_t i = n - 1; taken && i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (!at) {
            at = t.stride(i);
            taken = at >= width;
        }
        taken = taken && t.stride(i) == at * rows;
        rows *= t.size(i);
    }
    stride = taken && at ? at : width;
    return taken ? t : t.contiguous();
}
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void done(int32_t rc, const char* what) {
    TORCH_CHECK(rc == 0, "CRESSO5 ", what, " failed (", rc, "): ", g_api.last_error());
}
Tensor workspace(size_t bytes, const Tensor& like) {
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}
bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
// The kernels' gradients cannot be differentiated again: what a backward pass
// under create_graph returns says so when that is tried.
variable_list once(variable_list grads, const variable_list& from) {
    if (!at::GradMode::is_enabled()) return grads;
    bool any = false;
    for (const Tensor& t : from) any |= t.defined() && t.requires_grad();
    if (!any) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>("the operators' gradients cannot be differentiated twice",
                                                                 (int64_t)grads.size());
    variable_list in;
    for (const Tensor& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_(true) : Tensor());
    return (*error)(std::move(in));
}

// ---------------------------------------------------------------------------
// embedding
// ---------------------------------------------------------------------------
void check_ids(const char* what, const Tensor& ids) {
    TORCH_CHECK_VALUE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, what,
                      ": ids must be int32 or int64, not ", name_of(ids.scalar_type()));
}
Tensor embedding_rows(const Tensor& ids_, const Tensor& weight, double scale) {
    const Tensor ids = ids_.contiguous();
    const int64_t rows = weight.size(0), width = weight.size(1);
    int64_t stride;
    const Tensor w = rows_of(weight, stride);
    std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(width);
    Tensor out = at::empty(shape, weight.options().requires_grad(false));
    if (out.numel()) {
        const c10::DeviceGuard guard(weight.device());
        done(g_api.embedding_forward(ids.const_data_ptr(), (int32_t)ids.element_size(), ids.numel(), w.const_data_ptr(), rows, width,
                                     stride, code_of(w.scalar_type()), scale, out.mutable_data_ptr(), stream_of(w)),
             "embedding");
    }
    return out;
}
Tensor embedding_table(const Tensor& ids_, const Tensor& grad, int64_t rows, double scale) {
    const Tensor ids = ids_.contiguous();
    const int64_t width = grad.size(-1);
    int64_t stride;
    const Tensor g = rows_of(grad, stride);
    Tensor table = at::empty({rows, width}, grad.options().requires_grad(false));
    if (table.numel()) {
        const c10::DeviceGuard guard(grad.device());
        const int32_t code = code_of(g.scalar_type());
        const size_t bytes = g_api.embedding_backward_workspace_bytes(ids.numel(), width, code);
        const Tensor ws = workspace(bytes, g);
        done(g_api.embedding_backward(ids.const_data_ptr(), (int32_t)ids.element_size(), ids.numel(), g.const_data_ptr(), stride, rows,
                                      width, code, scale, table.mutable_data_ptr(), ws.mutable_data_ptr(), bytes, stream_of(g)),
             "embedding gradient");
    }
    return table;
}
struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale) {
        ctx->save_for_backward({ids});
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        return embedding_rows(ids, weight, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor ids = ctx->get_saved_variables()[0];
        Tensor table = embedding_table(ids, grads[0].detach(), ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble());
        return once({Tensor(), table, Tensor()}, grads);
    }
};
Tensor embedding(const Tensor& ids, const Tensor& weight, double scale) {
    const char* what = "embedding";
    OneGpu gpu{what};
    gpu.add("ids", ids);
    gpu.add("weight", weight);
    check_ids(what, ids);
    TORCH_CHECK_VALUE(weight.dim() == 2, what, ": weight must be [rows, width], not ", weight.sizes());
    check_row_type(what, "weight", weight);
    if (wants_grad({weight})) return EmbeddingFunction::apply(ids, weight, scale);
    return embedding_rows(ids, weight, scale);
}
Tensor embedding_grad(const Tensor& ids, const Tensor& grad, int64_t rows, double scale) {
    const char* what = "embedding";
    OneGpu gpu{what};
    gpu.add("ids", ids);
    gpu.add("grad", grad);
    check_ids(what, ids);
    check_row_type(what, "grad", grad);
    TORCH_CHECK_VALUE(grad.dim() == ids.dim() + 1 && grad.sizes().slice(0, ids.dim()) == ids.sizes(), what, ": grad of shape ",
                      grad.sizes(), " for ids of shape ", ids.sizes());
    TORCH_CHECK_VALUE(rows >= 0, what, ": rows must not be negative");
    return embedding_table(ids, grad.detach(), rows, scale);
}

// ---------------------------------------------------------------------------
// residual_norm
// ---------------------------------------------------------------------------
constexpr int64_t kMaxWidth = 16384;

struct Seam {
    Tensor in[6];   // residual, update, gate, post, pre, scale
    double scale, eps;
    int64_t act, rows_per_gate;
};
enum { RESIDUAL, UPDATE, GATE, POST, PRE, SCALE };

// Rows of `like` for each row of a gate (width,) or (leading dimensions of like, ones, width).
int64_t rows_per_gate(const Tensor& gate, const Tensor& like) {
    const int64_t width = like.size(-1), lead = like.dim() - 1;
    if (gate.dim() == 1 && gate.size(0) == width) return std::max<int64_t>(1, like.numel() / width);
    bool ok = gate.dim() == like.dim() && gate.size(-1) == width;
    int64_t k = 0, rows = 1;
    if (ok) {
        while (k < lead && gate.size(k) == like.size(k)) ++k;
        for (int64_t i = k; i < lead; ++i) {
            ok &= gate.size(i) == 1;
            rows *= like.size(i);
        }
    }
    TORCH_CHECK_VALUE(ok, "residual_norm: gate of shape ", gate.sizes(), " for rows of shape ", like.sizes(),
                      ": it must be (width,) or have the rows' own leading dimensions and then ones");
    return std::max<int64_t>(1, rows);
}
// The descriptor of a call; `keep` holds what it points to.
cresso_residual_norm_desc seam_desc(const Seam& s, std::vector<Tensor>& keep) {
    cresso_residual_norm_desc d{};
    const auto rows = [&](const Tensor& t, int64_t& stride) -> const void* {
        if (!t.defined()) return nullptr;
        keep.push_back(rows_of(t, stride));
        return keep.back().const_data_ptr();
    };
    const auto vec = [&](const Tensor& t, int32_t& code) -> const void* {
        if (!t.defined()) return nullptr;
        keep.push_back(t.contiguous());
        code = code_of(t.scalar_type());
        return keep.back().const_data_ptr();
    };
    d.residual = rows(s.in[RESIDUAL], d.residual_stride);
    d.update = rows(s.in[UPDATE], d.update_stride);
    d.gate = vec(s.in[GATE], d.gate_dtype);
    d.post = vec(s.in[POST], d.post_dtype);
    d.pre = vec(s.in[PRE], d.pre_dtype);
    d.scale_vec = vec(s.in[SCALE], d.scale_dtype);
    d.width = s.in[RESIDUAL].size(-1);
    d.gate_stride = d.width;
    d.rows = s.in[RESIDUAL].numel() / d.width;
    d.rows_per_gate = s.rows_per_gate;
    d.scale = (float)s.scale;
    d.eps = (float)s.eps;
    d.dtype = code_of(s.in[RESIDUAL].scalar_type());
    d.act = (int32_t)s.act;
    return d;
}
Tensor like_rows(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }

std::tuple<Tensor, Tensor> seam_forward(const Seam& s, const Tensor& stats) {
    const Tensor& h = s.in[RESIDUAL];
    Tensor out = like_rows(h), normed;
    if (s.in[PRE].defined()) normed = like_rows(h);
    if (h.numel()) {
        std::vector<Tensor> keep;
        keep.reserve(6);
        cresso_residual_norm_desc d = seam_desc(s, keep);
        d.out = out.mutable_data_ptr();
        if (normed.defined()) d.normed = normed.mutable_data_ptr();
        if (stats.defined()) d.stats = (float*)stats.mutable_data_ptr();
        const c10::DeviceGuard guard(h.device());
        done(g_api.residual_norm_forward(&d, stream_of(h)), "residual_norm");
    }
    return {out, normed};
}
struct SeamFunction : torch::autograd::Function<SeamFunction> {
    using Maybe = optional<Tensor>;
    static variable_list forward(AutogradContext* ctx, const Tensor& h, const Maybe& y, const Maybe& g, const Maybe& w1,
                                 const Maybe& w2, const Maybe& sv, double scale, double eps, int64_t act, int64_t per_gate) {
        const Seam s{{h, or_none(y), or_none(g), or_none(w1), or_none(w2), or_none(sv)}, scale, eps, act, per_gate};
        const Tensor stats = at::empty({h.numel() / h.size(-1), 2}, h.options().dtype(at::kFloat).requires_grad(false));
        auto [out, normed] = seam_forward(s, stats);
        ctx->save_for_backward({s.in[0], s.in[1], s.in[2], s.in[3], s.in[4], s.in[5], stats});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["act"] = act;
        ctx->saved_data["per_gate"] = per_gate;
        ctx->set_materialize_grads(false);
        if (normed.defined()) return {out, normed};
        return {out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        variable_list grads(10);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor d_out = arrive[0], d_normed = arrive.size() > 1 ? arrive[1] : Tensor();
        if (!d_out.defined() && !d_normed.defined()) return grads;
        Seam s{{}, ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt(),
               ctx->saved_data["per_gate"].toInt()};
        for (int i = 0, input = 0; i < 6; ++i) {
            s.in[i] = saved[i];
            if (saved[i].defined() && ctx->needs_input_grad(input++)) grads[i] = like_rows(saved[i]);
        }
        const Tensor& h = s.in[RESIDUAL];
        if (!h.numel()) {
            for (Tensor& g : grads)
                if (g.defined()) g.zero_();
            return grads;
        }
        std::vector<Tensor> keep;
        keep.reserve(8);
        cresso_residual_norm_desc d = seam_desc(s, keep);
        d.stats = (float*)saved[6].mutable_data_ptr();
        const auto arrives = [&](const Tensor& t, int64_t& stride) -> const void* {
            if (!t.defined()) return nullptr;
            keep.push_back(rows_of(t.detach(), stride));
            return keep.back().const_data_ptr();
        };
        d.d_out = arrives(d_out, d.d_out_stride);
        d.d_normed = arrives(d_normed, d.d_normed_stride);
        void** to[6] = {&d.d_residual, &d.d_update, &d.d_gate, &d.d_post, &d.d_pre, &d.d_scale};
        for (int i = 0; i < 6; ++i)
            if (grads[i].defined()) *to[i] = grads[i].mutable_data_ptr();
        const c10::DeviceGuard guard(h.device());
        const size_t bytes = g_api.residual_norm_backward_workspace_bytes(&d);
        const Tensor ws = workspace(bytes, h);
        done(g_api.residual_norm_backward(&d, ws.mutable_data_ptr(), bytes, stream_of(h)), "residual_norm gradient");
        variable_list from(arrive);
        from.insert(from.end(), saved.begin(), saved.begin() + 6);
        return once(std::move(grads), from);
    }
};
std::tuple<Tensor, optional<Tensor>> residual_norm(const Tensor& residual, const optional<Tensor>& update_, const optional<Tensor>& gate_,
                                                   int64_t act, const optional<Tensor>& post_, const optional<Tensor>& pre_,
                                                   const optional<Tensor>& scale_vec_, double scale, double eps) {
    const char* what = "residual_norm";
    Seam s{{residual, or_none(update_), or_none(gate_), or_none(post_), or_none(pre_), or_none(scale_vec_)}, scale, eps, act, 1};
    const char* names[6] = {"residual", "update", "gate", "post_weight", "pre_weight", "residual_scale"};
    OneGpu gpu{what};
    for (int i = 0; i < 6; ++i) gpu.add(names[i], s.in[i]);
    check_row_type(what, names[0], residual);
    TORCH_CHECK_VALUE(residual.dim() >= 1 && residual.size(-1) >= 1, what, ": the last dimension must not be empty");
    TORCH_CHECK_VALUE(residual.size(-1) <= kMaxWidth, what, ": width ", residual.size(-1), " above ", kMaxWidth);
    TORCH_CHECK_VALUE(eps > 0.0, what, ": eps must be positive");
    if (s.in[UPDATE].defined()) {
        TORCH_CHECK_VALUE(s.in[UPDATE].sizes() == residual.sizes() && s.in[UPDATE].scalar_type() == residual.scalar_type(), what,
                          ": update is ", name_of(s.in[UPDATE].scalar_type()), " ", s.in[UPDATE].sizes(), ", residual ",
                          name_of(residual.scalar_type()), " ", residual.sizes());
    } else {
        TORCH_CHECK_VALUE(!s.in[GATE].defined() && !s.in[POST].defined(), what, ": a gate or post_weight needs an update");
    }
    for (int i = GATE; i <= SCALE; ++i) {
        if (!s.in[i].defined()) continue;
        const auto t = s.in[i].scalar_type();
        TORCH_CHECK_VALUE(t == at::kFloat || t == residual.scalar_type(), what, ": ", names[i], " must be fp32 or ",
                          name_of(residual.scalar_type()), ", not ", name_of(t));
        if (i != GATE)
            TORCH_CHECK_VALUE(s.in[i].dim() == 1 && s.in[i].size(0) == residual.size(-1), what, ": ", names[i], " of shape ",
                              s.in[i].sizes(), " for a width of ", residual.size(-1));
    }
    if (s.in[GATE].defined()) s.rows_per_gate = rows_per_gate(s.in[GATE], residual);
    Tensor out, normed;
    if (wants_grad({s.in[0], s.in[1], s.in[2], s.in[3], s.in[4], s.in[5]})) {
        const variable_list both = SeamFunction::apply(s.in[0], or_null(s.in[1]), or_null(s.in[2]), or_null(s.in[3]),
                                                        or_null(s.in[4]), or_null(s.in[5]), scale, eps, act, s.rows_per_gate);
        out = both[0];
        if (both.size() > 1) normed = both[1];
    } else {
        std::tie(out, normed) = seam_forward(s, Tensor());
    }
    return {out, or_null(normed)};
}

// ---------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------
constexpr int64_t kMaxTop = 1024;

struct Distill {
    Tensor logits, index, teacher, labels, weights;
    double temperature, mix;
    int64_t ignore;
};
void check_distill(const Distill& c) {
    const char* what = "distill_loss";
    OneGpu gpu{what};
    gpu.add("logits", c.logits);
    gpu.add("teacher_index", c.index);
    gpu.add("teacher_logits", c.teacher);
    gpu.add("labels", c.labels);
    gpu.add("row_weights", c.weights);
    TORCH_CHECK_VALUE(c.logits.dim() == 2 && c.logits.size(1) >= 1, what, ": logits must be [rows, vocabulary], not ", c.logits.sizes());
    const int64_t rows = c.logits.size(0);
    TORCH_CHECK_VALUE(c.index.dim() == 2 && c.index.size(0) == rows && c.teacher.sizes() == c.index.sizes(), what, ": teacher_index ",
                      c.index.sizes(), " and teacher_logits ", c.teacher.sizes(), " must both be [", rows, ", entries]");
    TORCH_CHECK_VALUE(c.index.size(1) <= kMaxTop, what, ": ", c.index.size(1), " teacher entries a row: at most ", kMaxTop);
    check_row_type(what, "logits", c.logits);
    check_row_type(what, "teacher_logits", c.teacher);
    const auto whole = [](const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; };
    TORCH_CHECK_VALUE(whole(c.index), what, ": teacher_index must be int32 or int64");
    if (c.labels.defined()) {
        TORCH_CHECK_VALUE(whole(c.labels), what, ": labels must be int32 or int64");
        TORCH_CHECK_VALUE(c.labels.dim() == 1 && c.labels.size(0) == rows, what, ": labels must be [", rows, "]");
    }
    if (c.weights.defined())
        TORCH_CHECK_VALUE(c.weights.dim() == 1 && c.weights.size(0) == rows && c.weights.scalar_type() == at::kFloat, what,
                          ": row_weights must be fp32 [", rows, "]");
    TORCH_CHECK_VALUE(c.temperature > 0.0, what, ": temperature must be positive");
    TORCH_CHECK_VALUE(c.mix >= 0.0 && c.mix <= 1.0, what, ": mix must be within 0..1");
}
cresso_distill_desc distill_desc(const Distill& c, std::vector<Tensor>& keep) {
    cresso_distill_desc d{};
    const auto hold = [&](Tensor t) -> const void* {
        keep.push_back(std::move(t));
        return keep.back().const_data_ptr();
    };
    d.logits = hold(rows_of(c.logits, d.logits_stride));
    d.index = hold(rows_of(c.index, d.index_stride));
    d.teacher = hold(rows_of(c.teacher, d.teacher_stride));
    if (c.labels.defined()) {
        d.labels = hold(c.labels.contiguous());
        d.label_bytes = (int32_t)c.labels.element_size();
    }
    if (c.weights.defined()) d.weights = (const float*)hold(c.weights.contiguous());
    d.rows = c.logits.size(0);
    d.vocab = c.logits.size(1);
    d.top = (int32_t)c.index.size(1);
    d.weight = d.rows ? (float)(1.0 / (double)d.rows) : 0.0f;
    d.dtype = code_of(c.logits.scalar_type());
    d.teacher_dtype = code_of(c.teacher.scalar_type());
    d.index_bytes = (int32_t)c.index.element_size();
    d.temperature = (float)c.temperature;
    d.mix = (float)c.mix;
    d.ignore_index = c.ignore;
    return d;
}
// -> the rows' losses, and their sum if `sum` is set
std::tuple<Tensor, Tensor> distill_run(const Distill& c, bool sum, const Tensor& stats, const Tensor& grad) {
    const auto f32 = c.logits.options().dtype(at::kFloat).requires_grad(false);
    Tensor losses = at::empty({c.logits.size(0)}, f32), total;
    if (sum) total = at::empty({}, f32);
    std::vector<Tensor> keep;
    keep.reserve(5);
    cresso_distill_desc d = distill_desc(c, keep);
    d.loss = (float*)losses.mutable_data_ptr();
    if (sum) d.total = (float*)total.mutable_data_ptr();
    if (stats.defined()) d.stats = (float*)stats.mutable_data_ptr();
    if (grad.defined()) {
        d.grad = grad.mutable_data_ptr();
        d.grad_stride = grad.stride(0);
        const char* with = cresso::distill_overlap(d);
        TORCH_CHECK_VALUE(!with, "distill_loss: out shares memory with the ", with ? with : "",
                          " (it may take the logits' place: the same rows at the same stride)");
    }
    const c10::DeviceGuard guard(c.logits.device());
    done(g_api.distill_loss(&d, stream_of(c.logits)), "distill_loss");
    return {losses, total};
}
struct DistillFunction : torch::autograd::Function<DistillFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& index, const Tensor& teacher,
                          const optional<Tensor>& labels_, const optional<Tensor>& weights_, double temperature, double mix,
                          int64_t ignore, bool sum) {
        const Tensor labels = or_none(labels_), weights = or_none(weights_);
        const Tensor stats = at::empty({logits.size(0), 3}, logits.options().dtype(at::kFloat).requires_grad(false));
        auto [losses, total] = distill_run({logits, index, teacher, labels, weights, temperature, mix, ignore}, sum, stats, Tensor());
        ctx->save_for_backward({logits, index, teacher, labels, weights, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["mix"] = mix;
        ctx->saved_data["ignore"] = ignore;
        return sum ? total : losses;
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        const variable_list v = ctx->get_saved_variables();
        const Distill c{v[0], v[1], v[2], v[3], v[4], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["mix"].toDouble(),
                        ctx->saved_data["ignore"].toInt()};
        variable_list grads(9);
        grads[0] = at::empty(c.logits.sizes(), c.logits.options().requires_grad(false));
        if (grads[0].numel()) {
            std::vector<Tensor> keep;
            keep.reserve(5);
            cresso_distill_desc d = distill_desc(c, keep);
            const Tensor by = arrive[0].detach();
            d.stats = (float*)v[5].mutable_data_ptr();
            d.d_loss = (const float*)by.const_data_ptr();
            d.d_loss_stride = by.dim() ? by.stride(0) : 0;
            d.grad = grads[0].mutable_data_ptr();
            d.grad_stride = c.logits.size(1);
            const c10::DeviceGuard guard(c.logits.device());
            done(g_api.distill_backward(&d, stream_of(c.logits)), "distill_loss gradient");
        }
        return once(std::move(grads), {arrive[0], v[0]});
    }
};
Tensor distill_loss(const Tensor& logits, const Tensor& index, const Tensor& teacher, const optional<Tensor>& labels,
                    const optional<Tensor>& weights, double temperature, double mix, int64_t ignore, bool sum) {
    const Distill c{logits, index, teacher, or_none(labels), or_none(weights), temperature, mix, ignore};
    check_distill(c);
    if (wants_grad({logits}))
        return DistillFunction::apply(logits, index, teacher, or_null(c.labels), or_null(c.weights), temperature, mix, ignore, sum);
    auto [losses, total] = distill_run(c, sum, Tensor(), Tensor());
    return sum ? total : losses;
}
std::tuple<Tensor, Tensor> distill_loss_and_grad(const Tensor& logits, const Tensor& index, const Tensor& teacher,
                                                 const optional<Tensor>& labels, const optional<Tensor>& weights, double temperature,
                                                 double mix, int64_t ignore, const optional<Tensor>& out) {
    const char* what = "distill_loss";
    const at::NoGradGuard no_grad;
    OneGpu{what}.add("logits", logits);   // detach() drops a tangent
    const Distill c{logits.detach(), index, teacher, or_none(labels), or_none(weights), temperature, mix, ignore};
    check_distill(c);
    Tensor grad = or_none(out);
    if (grad.defined()) {
        OneGpu gpu{what};
        gpu.add("logits", logits);
        gpu.add("out", grad);
        TORCH_CHECK_VALUE(grad.sizes() == logits.sizes() && grad.scalar_type() == logits.scalar_type(), what, ": out is ",
                          name_of(grad.scalar_type()), " ", grad.sizes(), ", logits ", name_of(logits.scalar_type()), " ", logits.sizes());
        TORCH_CHECK_VALUE(grad.stride(1) == 1 && (grad.size(0) < 2 || grad.stride(0) >= grad.size(1)), what,
                          ": out must hold each row in one piece");
    } else {
        grad = at::empty(logits.sizes(), logits.options().requires_grad(false));
    }
    const Tensor stats = at::empty({logits.size(0), 3}, logits.options().dtype(at::kFloat).requires_grad(false));
    Tensor total = std::get<1>(distill_run(c, true, stats, grad));
    // written behind torch's back: what has saved it for its own gradient has to notice
    if (out.has_value()) grad.unsafeGetTensorImpl()->bump_version();
    return {total, grad};
}

// ---------------------------------------------------------------------------
// block_product
// ---------------------------------------------------------------------------
constexpr int64_t kBlock = 128;
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

Tensor product(const Tensor& x, const Tensor& values, const Tensor& scales, bool turned) {
    const int64_t depth = values.size(turned ? 0 : 1), cols = values.size(turned ? 1 : 0);
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = cols;
    Tensor out = at::empty(shape, x.options().requires_grad(false));
    if (out.numel()) {
        int64_t x_stride, w_stride;
        const Tensor xr = rows_of(x, x_stride), w = rows_of(values, w_stride), s = scales.contiguous();
        const int64_t rows = out.numel() / cols;
        const c10::DeviceGuard guard(x.device());
        const size_t bytes = g_api.block_product_workspace_bytes(rows, cols, depth, w.const_data_ptr(), w_stride, turned);
        const Tensor ws = workspace(bytes, x);
        done(g_api.block_product(xr.const_data_ptr(), x_stride, code_of(x.scalar_type()), rows, cols, depth, w.const_data_ptr(), w_stride,
                                 (const float*)s.const_data_ptr(), s.size(1), turned, out.mutable_data_ptr(), ws.mutable_data_ptr(), bytes,
                                 stream_of(x)),
             "block_product");
    }
    return out;
}
struct ProductFunction : torch::autograd::Function<ProductFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& values, const Tensor& scales) {
        ctx->save_for_backward({values, scales});
        return product(x, values, scales, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        const variable_list v = ctx->get_saved_variables();
        return once({product(arrive[0].detach(), v[0], v[1], true), Tensor(), Tensor()}, arrive);
    }
};
Tensor block_product(const Tensor& x, const Tensor& values, const Tensor& scales) {
    const char* what = "block_product";
    OneGpu gpu{what};
    gpu.add("x", x);
    gpu.add("values", values);
    gpu.add("scales", scales);
    TORCH_CHECK_VALUE(values.dim() == 2 && values.scalar_type() == at::kFloat8_e4m3fn, what,
                      ": values must be float8_e4m3fn [outputs, inputs], not ", name_of(values.scalar_type()), " ", values.sizes());
    TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == blocks_of(values.size(0)) &&
                          scales.size(1) == blocks_of(values.size(1)),
                      what, ": scales must be fp32 [", blocks_of(values.size(0)), ", ", blocks_of(values.size(1)), "], not ",
                      name_of(scales.scalar_type()), " ", scales.sizes());
    check_row_type(what, "x", x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == values.size(1), what, ": x of shape ", x.sizes(), " for a weight of ",
                      values.size(1), " inputs");
    if (wants_grad({x})) return ProductFunction::apply(x, values, scales);
    return product(x, values, scales, false);
}
std::tuple<Tensor, Tensor> quantize_blocks(const Tensor& weight) {
    const char* what = "quantize_blocks";
    OneGpu gpu{what};
    gpu.add("weight", weight);
    TORCH_CHECK_VALUE(weight.dim() == 2, what, ": weight must be [outputs, inputs], not ", weight.sizes());
    check_row_type(what, "weight", weight);
    const int64_t rows = weight.size(0), cols = weight.size(1);
    const auto options = weight.options().requires_grad(false);
    Tensor values = at::empty({rows, cols}, options.dtype(at::kFloat8_e4m3fn));
    Tensor scales = at::empty({blocks_of(rows), blocks_of(cols)}, options.dtype(at::kFloat));
    if (values.numel()) {
        int64_t stride;
        const Tensor w = rows_of(weight.detach(), stride);
        const c10::DeviceGuard guard(weight.device());
        done(g_api.block_quantize(w.const_data_ptr(), stride, code_of(w.scalar_type()), rows, cols, values.mutable_data_ptr(),
                                  (float*)scales.mutable_data_ptr(), stream_of(w)),
             "quantize_blocks");
    }
    return {values, scales};
}

}  // namespace

PYBIND11_MODULE(_operators, m) {
    namespace py = pybind11;
    const auto free = py::call_guard<py::gil_scoped_release>();
    m.def("bind", &bind);
    m.def("embedding", &embedding, free);
    m.def("embedding_grad", &embedding_grad, free);
    m.def("residual_norm", &residual_norm, free);
    m.def("distill_loss", &distill_loss, free);
    m.def("distill_loss_and_grad", &distill_loss_and_grad, free);
    m.def("block_product", &block_product, free);
    m.def("quantize_blocks", &quantize_blocks, free);
}
