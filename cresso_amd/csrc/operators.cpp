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
#include <ATen/MemoryOverlap.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
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
    decltype(&cresso_clip_workspace_bytes) clip_workspace_bytes;
    decltype(&cresso_clip_gradients) clip_gradients;
    decltype(&cresso_route_workspace_bytes) route_workspace_bytes;
    decltype(&cresso_route_forward) route_forward;
    decltype(&cresso_route_backward) route_backward;
    decltype(&cresso_dispatch_rows) dispatch_rows;
    decltype(&cresso_combine_rows) combine_rows;
    decltype(&cresso_combine_backward) combine_backward;
    decltype(&cresso_expert_product_workspace_bytes) expert_product_workspace_bytes;
    decltype(&cresso_expert_product) expert_product;
    decltype(&cresso_expert_product_weight_workspace_bytes) expert_product_weight_workspace_bytes;
    decltype(&cresso_expert_product_weight) expert_product_weight;
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
    take(a.clip_workspace_bytes, "cresso_clip_workspace_bytes");
    take(a.clip_gradients, "cresso_clip_gradients");
    take(a.route_workspace_bytes, "cresso_route_workspace_bytes");
    take(a.route_forward, "cresso_route_forward");
    take(a.route_backward, "cresso_route_backward");
    take(a.dispatch_rows, "cresso_dispatch_rows");
    take(a.combine_rows, "cresso_combine_rows");
    take(a.combine_backward, "cresso_combine_backward");
    take(a.expert_product_workspace_bytes, "cresso_expert_product_workspace_bytes");
    take(a.expert_product, "cresso_expert_product");
    take(a.expert_product_weight_workspace_bytes, "cresso_expert_product_weight_workspace_bytes");
    take(a.expert_product_weight, "cresso_expert_product_weight");
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
        TORCH_CHECK(!t.is_neg(), what, ": ", name, " is a view that stands for the negative of its memory (resolve_neg gives it its own)");
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
// A gradient that arrives at a backward pass, as the kernels read it: in its own
// memory where it is a view that stands for the negative of another's (autograd
// makes those of conjugated complex numbers), and not a dual tensor, whose
// tangent the result would lack.
Tensor arrived(const char* what, const Tensor& t) {
    TORCH_CHECK(!t._fw_grad(0).defined(), "the gradient that arrives at ", what,
                " has a forward-mode derivative, the operators have reverse mode only");
    return t.detach().resolve_neg();
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
        Tensor table = embedding_table(ids, arrived("embedding", grads[0]), ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble());
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
            keep.push_back(rows_of(arrived("residual_norm", t), stride));
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
            const Tensor by = arrived("distill_loss", arrive[0]);
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
        return once({product(arrived("block_product", arrive[0]), v[0], v[1], true), Tensor(), Tensor()}, arrive);
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

// ---------------------------------------------------------------------------
// gradient norm and clipping
// ---------------------------------------------------------------------------
// Bytes [at, end) of memory; of those, where `row` is not 0, `width` ones at `at`
// and at whole multiples of `row` behind it.
struct Written {
    uintptr_t at, end;
    bool out;
    uintptr_t row = 0, width = 0;
};
// A tensor's bytes.  Slices that leave gaps are rows of one piece each where their strides say so.
Written bytes_of(const Tensor& t, uintptr_t at, bool dense, bool out) {
    const uintptr_t size = (uintptr_t)t.element_size();
    if (dense) return {at, at + (uintptr_t)t.numel() * size, out};
    std::vector<std::pair<int64_t, int64_t>> dims;   // stride, size
    int64_t reach = 1;   // elements from the first to the last
    for (int64_t d = 0; d < t.dim(); ++d) {
        reach += (t.size(d) - 1) * t.stride(d);
        if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
    }
    std::sort(dims.begin(), dims.end());
    int64_t width = 1, row = 0;
    for (const auto& [stride, n] : dims) {
        if (!row && stride == width) width *= n;
        else if (!row) row = stride;
        if (row && (row <= width || stride % row)) return {at, at + (uintptr_t)reach * size, out};
    }
    return {at, at + (uintptr_t)reach * size, out, (uintptr_t)row * size, (uintptr_t)width * size};
}
// Whether bytes that are written are another's too, rows taken as whole blocks; spans by their begin.
template <typename It> bool overlaps(It first, It last) {
    uintptr_t any = 0, out = 0;
    for (; first != last; ++first) {
        if (first->at < out || (first->out && first->at < any)) return true;
        any = std::max(any, first->end);
        if (first->out) out = std::max(out, first->end);
    }
    return false;
}
bool before(const Written& a, const Written& b) { return a.at < b.at; }
// Whether memory that is written belongs to anything else of the call.  Slices
// that interleave share nothing where they are columns of the same rows, others
// count as sharing.
bool shares(std::vector<Written>& spans) {
    if (!std::is_sorted(spans.begin(), spans.end(), before)) std::sort(spans.begin(), spans.end(), before);
    if (!overlaps(spans.begin(), spans.end())) return false;
    for (auto first = spans.begin(); first != spans.end();) {
        uintptr_t end = first->end;
        auto last = first + 1;   // spans that hang together
        for (; last != spans.end() && last->at < end; ++last) end = std::max(end, last->end);
        if (overlaps(first, last)) {
            std::vector<Written> columns;
            for (auto s = first; s != last; ++s) {
                if (!s->row || s->row != first->row) return true;
                const uintptr_t at = (s->at - first->at) % s->row, to = at + s->width;
                columns.push_back({at, std::min(to, s->row), s->out});
                if (to > s->row) columns.push_back({0, to - s->row, s->out});
            }
            std::sort(columns.begin(), columns.end(), before);
            if (overlaps(columns.begin(), columns.end())) return true;
        }
        first = last;
    }
    return false;
}
// The tensors of a Python list, None among them, where they are: a program has
// hundreds, and a vector of counted references takes longer than the kernels.
struct Listed {
    PyObject* list;
    size_t size() const { return (size_t)PyList_GET_SIZE(list); }
    const Tensor* at(size_t i) const {
        PyObject* o = PyList_GET_ITEM(list, i);
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) throw pybind11::type_error("not a tensor");
        return &THPVariable_Unpack(o);
    }
};
Tensor clip(const char* what, const Listed& grads, double max_norm, int64_t kind, double grad_scale, const Listed* out, bool in_place) {
    const bool recorded = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    TORCH_CHECK_VALUE(max_norm >= 0.0, what, ": max_norm must not be negative");
    TORCH_CHECK_VALUE(std::isfinite(grad_scale), what, ": grad_scale must be finite");
    if (out) TORCH_CHECK_VALUE(out->size() == grads.size(), what, ": ", out->size(), " outputs for ", grads.size(), " gradients");
    OneGpu gpu{what};
    std::vector<cresso_grad_desc> descs;
    std::vector<Written> spans;
    std::vector<Tensor> keep;                             // copies
    std::vector<std::pair<const Tensor*, Tensor>> back;   // written in a copy: where it goes
    descs.reserve(grads.size());
    if (out || in_place) spans.reserve(out ? 2 * grads.size() : grads.size());
    const Tensor* first = nullptr;
    const auto span = [&](const Tensor& t, uintptr_t at, bool dense, bool out) {
        const Written s = bytes_of(t, at, dense, out);
        if (dense && !spans.empty() && !spans.back().row && spans.back().end == at && spans.back().out == out) spans.back().end = s.end;   // buckets hold them so
        else spans.push_back(s);
    };
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor* const given = grads.at(i);
        if (!given) continue;
        const Tensor& g = *given;
        TORCH_CHECK_VALUE(g.layout() == at::kStrided, what, ": gradient ", i, " is sparse");
        gpu.add("a gradient", g);
        const int32_t code = code_of(g.scalar_type());
        TORCH_CHECK_VALUE(code >= 0, what, ": gradient ", i, " must be fp32, fp64, bf16 or fp16, not ", name_of(g.scalar_type()));
        if (!first) first = &g;
        const Tensor* to = in_place ? &g : nullptr;
        if (out) {
            to = out->at(i);
            TORCH_CHECK_VALUE(to, what, ": no output for gradient ", i);
            TORCH_CHECK_VALUE(to->layout() == at::kStrided && to->sizes() == g.sizes() &&
                                  (to->scalar_type() == g.scalar_type() || (to->scalar_type() == at::kFloat && g.element_size() == 2)),
                              what, ": output ", i, " is ", name_of(to->scalar_type()), " ", to->sizes(), " for a gradient of ",
                              name_of(g.scalar_type()), " ", g.sizes(), " (its own type or, of 16 bits, fp32)");
            gpu.add("an output", *to);
        }
        // as torch's own operations in place, which refuse a leaf where they are recorded: a parameter in its gradient's stead
        TORCH_CHECK(!to || !recorded || !to->requires_grad() || !(to->is_leaf() || (to->is_view() && to->_base().is_leaf())), what, ": ",
                    in_place ? "gradient " : "output ", i, " is a leaf that requires a gradient, and would be scaled itself (a parameter instead of its .grad?)");
        const int64_t numel = g.numel();
        if (!numel) continue;
        cresso_grad_desc d{};
        d.numel = numel;
        d.dtype = code;
        d.grad = g.const_data_ptr();
        const bool dense = g.is_non_overlapping_and_dense();
        const bool same = to == &g || (to && to->const_data_ptr() == d.grad && to->scalar_type() == g.scalar_type() && to->strides() == g.strides());
        bool to_dense = dense;
        if (to) {
            if (!same) to_dense = to->is_non_overlapping_and_dense();
            TORCH_CHECK_VALUE(to_dense || at::has_internal_overlap(*to) != at::MemOverlap::Yes, what, ": output ", i,
                              " holds several elements in one place");
            span(*to, (uintptr_t)(same ? d.grad : to->const_data_ptr()), to_dense, true);
        }
        if (!same && out) span(g, (uintptr_t)d.grad, dense, false);
        const Tensor* from = &g;
        if (!dense) {   // any order of the elements serves a norm, gaps do not
            keep.push_back(g.contiguous());
            d.grad = keep.back().const_data_ptr();
        }
        if (to) {
            d.out_dtype = code_of(to->scalar_type());
            if (same) {
                d.out = const_cast<void*>(d.grad);
                if (!dense) back.emplace_back(to, keep.back());
            } else if (dense && to_dense && to->strides() == from->strides()) {
                d.out = to->mutable_data_ptr();
            } else {
                const Tensor rows = dense ? at::empty_strided(g.sizes(), g.strides(), to->options()) : at::empty(g.sizes(), to->options());
                d.out = rows.mutable_data_ptr();
                back.emplace_back(to, rows);
            }
        }
        descs.push_back(d);
    }
    TORCH_CHECK_VALUE(!(out || in_place) || !shares(spans), what,
                      ": memory that is written belongs to two gradients (a parameter that is given twice? slices that interleave and are no "
                      "columns of the same rows?), or to an input and another's output");
    if (!first) return at::zeros({}, at::device(at::kCUDA).dtype(at::kFloat));
    const c10::DeviceGuard guard(first->device());
    Tensor norm = at::empty({}, first->options().dtype(at::kFloat).requires_grad(false));
    const size_t bytes = g_api.clip_workspace_bytes(descs.data(), (int32_t)descs.size());
    const Tensor ws = workspace(bytes, norm);
    done(g_api.clip_gradients(descs.data(), (int32_t)descs.size(), (int32_t)kind, max_norm, grad_scale, (float*)norm.mutable_data_ptr(),
                              ws.mutable_data_ptr(), bytes, stream_of(*first)),
         what);
    for (auto& [to, from] : back) to->copy_(from);
    // written behind torch's back: what has saved them for its own gradient has to notice
    const Listed* written = out ? out : in_place ? &grads : nullptr;
    for (size_t i = 0; written && i < written->size(); ++i) {
        const Tensor* t = written->at(i);
        if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
    return norm;
}
Tensor gradient_norm(const pybind11::list& grads, int64_t kind) {
    return clip("gradient_norm", {grads.ptr()}, INFINITY, kind, 1.0, nullptr, false);
}
Tensor clip_gradients(const pybind11::list& grads, double max_norm, int64_t kind, double grad_scale, const optional<pybind11::list>& out) {
    const Listed to{out.has_value() ? out->ptr() : nullptr};
    return clip("clip_gradients", {grads.ptr()}, max_norm, kind, grad_scale, out.has_value() ? &to : nullptr, !out.has_value());
}

// ---------------------------------------------------------------------------
// layers of experts
// ---------------------------------------------------------------------------
constexpr int64_t kMaxExperts = 1024, kMaxExpertsOfToken = 32, kMaxTokens = (1 << 26) - 16;

struct Route {
    Tensor logits, bias;
    int64_t top, score;
    bool normalize;
    double scale;
};
cresso_route_desc route_desc(const Route& r, std::vector<Tensor>& keep) {
    cresso_route_desc d{};
    keep.push_back(rows_of(r.logits, d.logits_stride));
    d.logits = keep.back().const_data_ptr();
    if (r.bias.defined()) {
        keep.push_back(r.bias.contiguous());
        d.bias = (const float*)keep.back().const_data_ptr();
    }
    d.tokens = r.logits.size(0);
    d.num_experts = (int32_t)r.logits.size(1);
    d.top = (int32_t)r.top;
    d.dtype = code_of(r.logits.scalar_type());
    d.score = (int32_t)r.score;
    d.normalize = r.normalize;
    d.scale = (float)r.scale;
    return d;
}
// -> weights, experts, order, places, offsets
variable_list route_forward(const Route& r) {
    const int64_t tokens = r.logits.size(0);
    const auto f32 = r.logits.options().dtype(at::kFloat).requires_grad(false), i32 = f32.dtype(at::kInt);
    Tensor weights = at::empty({tokens, r.top}, f32), experts = at::empty({tokens, r.top}, i32);
    Tensor order = at::empty({tokens * r.top}, i32), places = at::empty({tokens, r.top}, i32), offsets = at::empty({r.logits.size(1) + 1}, i32);
    std::vector<Tensor> keep;
    keep.reserve(2);
    cresso_route_desc d = route_desc(r, keep);
    d.weights = (float*)weights.mutable_data_ptr();
    d.experts = (int32_t*)experts.mutable_data_ptr();
    d.order = (int32_t*)order.mutable_data_ptr();
    d.places = (int32_t*)places.mutable_data_ptr();
    d.offsets = (int32_t*)offsets.mutable_data_ptr();
    const c10::DeviceGuard guard(r.logits.device());
    const size_t bytes = g_api.route_workspace_bytes(&d);
    const Tensor ws = workspace(bytes, weights);
    done(g_api.route_forward(&d, ws.mutable_data_ptr(), bytes, stream_of(r.logits)), "route_experts");
    return {weights, experts, order, places, offsets};
}
struct RouteFunction : torch::autograd::Function<RouteFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const optional<Tensor>& bias, int64_t top, int64_t score,
                                 bool normalize, double scale) {
        variable_list got = route_forward({logits, or_none(bias), top, score, normalize, scale});
        ctx->save_for_backward({logits, got[0], got[1]});
        ctx->saved_data["top"] = top;
        ctx->saved_data["score"] = score;
        ctx->saved_data["normalize"] = normalize;
        ctx->saved_data["scale"] = scale;
        ctx->mark_non_differentiable({got[1], got[2], got[3], got[4]});
        ctx->set_materialize_grads(false);
        return got;
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        variable_list grads(6);
        if (!arrive[0].defined()) return grads;
        const variable_list v = ctx->get_saved_variables();
        const Route r{v[0], Tensor(), ctx->saved_data["top"].toInt(), ctx->saved_data["score"].toInt(), ctx->saved_data["normalize"].toBool(),
                      ctx->saved_data["scale"].toDouble()};
        grads[0] = at::empty(r.logits.sizes(), r.logits.options().requires_grad(false));
        if (grads[0].numel()) {
            std::vector<Tensor> keep;
            keep.reserve(2);
            cresso_route_desc d = route_desc(r, keep);
            d.weights = (float*)v[1].const_data_ptr();
            d.experts = (int32_t*)v[2].const_data_ptr();
            const Tensor by = arrived("route_experts", arrive[0]).contiguous();
            const c10::DeviceGuard guard(r.logits.device());
            done(g_api.route_backward(&d, (const float*)by.const_data_ptr(), grads[0].mutable_data_ptr(), stream_of(r.logits)),
                 "route_experts gradient");
        }
        return once(std::move(grads), {arrive[0], v[0]});
    }
};
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_experts(const Tensor& logits, int64_t top, int64_t score, bool normalize, double scale,
                                                                 const optional<Tensor>& bias_) {
    const char* what = "route_experts";
    const Tensor bias = or_none(bias_);
    OneGpu gpu{what};
    gpu.add("logits", logits);
    gpu.add("bias", bias);
    TORCH_CHECK_VALUE(logits.dim() == 2, what, ": logits must be [tokens, experts], not ", logits.sizes());
    check_row_type(what, "logits", logits);
    const int64_t experts = logits.size(1);
    TORCH_CHECK_VALUE(experts >= 1 && experts <= kMaxExperts, what, ": ", experts, " experts, 1 to ", kMaxExperts, " are taken");
    TORCH_CHECK_VALUE(top >= 1 && top <= std::min(experts, kMaxExpertsOfToken), what, ": top ", top, " of ", experts, " experts, 1 to ",
                      std::min(experts, kMaxExpertsOfToken), " are taken");
    TORCH_CHECK_VALUE(logits.size(0) <= kMaxTokens && logits.size(0) * top < (int64_t)1 << 31, what, ": ", logits.size(0), " tokens are more than one call takes");
    TORCH_CHECK_VALUE(std::isfinite(scale), what, ": scale must be finite");
    if (bias.defined())
        TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == experts && bias.scalar_type() == at::kFloat, what, ": bias must be fp32 [",
                          experts, "], not ", name_of(bias.scalar_type()), " ", bias.sizes());
    const variable_list got = wants_grad({logits}) ? RouteFunction::apply(logits, or_null(bias), top, score, normalize, scale)
                                                   : route_forward({logits, bias, top, score, normalize, scale});
    return {got[0], got[1], got[2], got[3], got[4]};
}

// experts and places [tokens, top] of a routing
void check_slots(const char* what, OneGpu& gpu, const Tensor& experts, const Tensor& places) {
    gpu.add("experts", experts);
    gpu.add("places", places);
    TORCH_CHECK_VALUE(experts.scalar_type() == at::kInt && places.scalar_type() == at::kInt && experts.dim() == 2 &&
                          places.sizes() == experts.sizes(),
                      what, ": the routing's experts and places must be int32 [tokens, top], not ", name_of(experts.scalar_type()), " ",
                      experts.sizes(), " and ", name_of(places.scalar_type()), " ", places.sizes());
    TORCH_CHECK_VALUE(experts.size(1) >= 1 && experts.size(1) <= kMaxExpertsOfToken, what, ": ", experts.size(1), " experts a token, 1 to ",
                      kMaxExpertsOfToken, " are taken");
    TORCH_CHECK_VALUE(experts.size(0) <= kMaxTokens && experts.numel() < (int64_t)1 << 31, what, ": ", experts.size(0),
                      " tokens are more than one call takes");
}
const int32_t* ints(const Tensor& t) { return (const int32_t*)t.const_data_ptr(); }

Tensor dispatch(const Tensor& x, const Tensor& experts_, const Tensor& places_) {
    Tensor rows = at::empty({experts_.numel(), x.size(1)}, x.options().requires_grad(false));
    if (rows.numel()) {
        int64_t stride;
        const Tensor from = rows_of(x, stride), experts = experts_.contiguous(), places = places_.contiguous();
        const c10::DeviceGuard guard(x.device());
        done(g_api.dispatch_rows(from.const_data_ptr(), stride, code_of(x.scalar_type()), x.size(0), (int32_t)experts.size(1), x.size(1),
                                 ints(experts), ints(places), rows.mutable_data_ptr(), stream_of(x)),
             "dispatch_rows");
    }
    return rows;
}
Tensor combine(const char* what, const Tensor& rows, const Tensor& experts_, const Tensor& places_, const Tensor& weights_) {
    Tensor out = at::empty({experts_.size(0), rows.size(1)}, rows.options().requires_grad(false));
    if (out.numel()) {
        int64_t stride;
        const Tensor from = rows_of(rows, stride), experts = experts_.contiguous(), places = places_.contiguous();
        const Tensor weights = weights_.defined() ? weights_.contiguous() : Tensor();
        const c10::DeviceGuard guard(rows.device());
        done(g_api.combine_rows(from.const_data_ptr(), stride, code_of(rows.scalar_type()), out.size(0), (int32_t)experts.size(1), rows.size(1),
                                ints(experts), ints(places), weights.defined() ? (const float*)weights.const_data_ptr() : nullptr,
                                out.mutable_data_ptr(), stream_of(rows)),
             what);
    }
    return out;
}
struct DispatchFunction : torch::autograd::Function<DispatchFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& experts, const Tensor& places) {
        ctx->save_for_backward({experts, places});
        return dispatch(x, experts, places);
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        const variable_list v = ctx->get_saved_variables();
        return once({combine("dispatch_rows gradient", arrived("dispatch_rows", arrive[0]), v[0], v[1], Tensor()), Tensor(), Tensor()}, arrive);
    }
};
struct CombineFunction : torch::autograd::Function<CombineFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& experts, const Tensor& places, const optional<Tensor>& weights) {
        ctx->save_for_backward({rows, experts, places, or_none(weights)});
        return combine("combine_rows", rows, experts, places, or_none(weights));
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        const variable_list v = ctx->get_saved_variables();
        const Tensor& rows = v[0];
        const bool to_rows = ctx->needs_input_grad(0), to_weights = v[3].defined() && ctx->needs_input_grad(3);
        variable_list grads(4);
        // places that are none of the rows' are not written
        if (to_rows) grads[0] = at::empty(rows.sizes(), rows.options().requires_grad(false));
        if (to_weights) grads[3] = at::empty(v[3].sizes(), v[3].options().requires_grad(false));
        if (v[1].numel() && (to_rows || to_weights)) {
            int64_t stride, by_stride;
            const Tensor from = rows_of(rows, stride), by = rows_of(arrived("combine_rows", arrive[0]), by_stride);
            const Tensor experts = v[1].contiguous(), places = v[2].contiguous(), weights = v[3].defined() ? v[3].contiguous() : Tensor();
            const c10::DeviceGuard guard(rows.device());
            done(g_api.combine_backward(from.const_data_ptr(), stride, by.const_data_ptr(), by_stride, code_of(rows.scalar_type()), by.size(0),
                                        (int32_t)experts.size(1), rows.size(1), ints(experts), ints(places),
                                        weights.defined() ? (const float*)weights.const_data_ptr() : nullptr,
                                        to_rows ? grads[0].mutable_data_ptr() : nullptr, to_weights ? (float*)grads[3].mutable_data_ptr() : nullptr,
                                        stream_of(rows)),
                 "combine_rows gradient");
        }
        return once(std::move(grads), {arrive[0], rows, v[3]});
    }
};
Tensor dispatch_rows(const Tensor& x, const Tensor& experts, const Tensor& places) {
    const char* what = "dispatch_rows";
    OneGpu gpu{what};
    gpu.add("x", x);
    check_slots(what, gpu, experts, places);
    check_row_type(what, "x", x);
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == experts.size(0), what, ": x must be [", experts.size(0), ", width], not ", x.sizes());
    if (wants_grad({x})) return DispatchFunction::apply(x, experts, places);
    return dispatch(x, experts, places);
}
Tensor combine_rows(const Tensor& rows, const Tensor& experts, const Tensor& places, const optional<Tensor>& weights_) {
    const char* what = "combine_rows";
    const Tensor weights = or_none(weights_);
    OneGpu gpu{what};
    gpu.add("rows", rows);
    check_slots(what, gpu, experts, places);
    gpu.add("weights", weights);
    check_row_type(what, "rows", rows);
    TORCH_CHECK_VALUE(rows.dim() == 2 && rows.size(0) == experts.numel(), what, ": rows must be [", experts.numel(), ", width], not ", rows.sizes());
    if (weights.defined())
        TORCH_CHECK_VALUE(weights.scalar_type() == at::kFloat && weights.sizes() == experts.sizes(), what, ": weights must be fp32 ",
                          experts.sizes(), ", not ", name_of(weights.scalar_type()), " ", weights.sizes());
    if (wants_grad({rows, weights})) return CombineFunction::apply(rows, experts, places, or_null(weights));
    return combine(what, rows, experts, places, weights);
}

// A stacked weight [experts, outputs, inputs] where it lies: rows along the
// inputs, or (turned) along the outputs, as a transposed view has them; any
// other layout is copied.
struct Stacked {
    Tensor t;
    int64_t expert, stride;
    bool turned;
};
Stacked stacked_of(const Tensor& w) {
    const int64_t n = w.size(1), k = w.size(2);
    if ((k < 2 || w.stride(2) == 1) && (n < 2 || w.stride(1) >= k) && (w.size(0) < 2 || w.stride(0) >= 0))
        return {w, w.size(0) < 2 ? 0 : w.stride(0), n < 2 ? k : w.stride(1), false};
    if ((n < 2 || w.stride(1) == 1) && (k < 2 || w.stride(2) >= n) && (w.size(0) < 2 || w.stride(0) >= 0))
        return {w, w.size(0) < 2 ? 0 : w.stride(0), k < 2 ? n : w.stride(2), true};
    return {w.contiguous(), n * k, k, false};
}
// x times the transposes of the matrices (forward), or times the matrices (the gradient of x)
Tensor group_product(const char* what, const Tensor& x, const Tensor& weight, const Tensor& offsets_, bool back) {
    const int64_t rows = x.size(0), cols = weight.size(back ? 2 : 1), depth = weight.size(back ? 1 : 2);
    const int32_t experts = (int32_t)weight.size(0), code = code_of(x.scalar_type());
    Tensor out = at::empty({rows, cols}, x.options().requires_grad(false));
    if (out.numel()) {
        int64_t stride;
        const Tensor from = rows_of(x, stride), offsets = offsets_.contiguous();
        const Stacked w = stacked_of(weight);
        const c10::DeviceGuard guard(x.device());
        const size_t bytes = g_api.expert_product_workspace_bytes(rows, cols, depth, experts, code);
        const Tensor ws = workspace(bytes, x);
        done(g_api.expert_product(from.const_data_ptr(), stride, code, rows, cols, depth, w.t.const_data_ptr(), w.expert, w.stride,
                                  w.turned != back, experts, ints(offsets), out.mutable_data_ptr(), ws.mutable_data_ptr(), bytes,
                                  stream_of(x)),
             what);
    }
    return out;
}
// [experts, outputs, inputs], held as the weight is
Tensor group_weight(const Tensor& x_, const Tensor& by_, const Tensor& weight, const Tensor& offsets_) {
    const bool turned = stacked_of(weight).turned;
    const Tensor &p_ = turned ? x_ : by_, &q_ = turned ? by_ : x_;
    const int64_t experts = weight.size(0), pw = p_.size(1), qw = q_.size(1);
    Tensor out = at::empty({experts, pw, qw}, weight.options().requires_grad(false));
    if (out.numel()) {
        int64_t ps, qs;
        const Tensor p = rows_of(p_, ps), q = rows_of(q_, qs), offsets = offsets_.contiguous();
        const int32_t code = code_of(weight.scalar_type());
        const c10::DeviceGuard guard(weight.device());
        const size_t bytes = g_api.expert_product_weight_workspace_bytes(p.size(0), pw, qw, (int32_t)experts, code);
        const Tensor ws = workspace(bytes, weight);
        done(g_api.expert_product_weight(p.const_data_ptr(), ps, pw, q.const_data_ptr(), qs, qw, code, p.size(0), (int32_t)experts,
                                         ints(offsets), out.mutable_data_ptr(), ws.mutable_data_ptr(), bytes, stream_of(weight)),
             "expert_product gradient of the weight");
    }
    return turned ? out.transpose(1, 2) : out;
}
struct ExpertFunction : torch::autograd::Function<ExpertFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& offsets) {
        ctx->save_for_backward({x, weight, offsets});
        return group_product("expert_product", x, weight, offsets, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list arrive) {
        const variable_list v = ctx->get_saved_variables();
        const Tensor by = arrived("expert_product", arrive[0]);
        variable_list grads(3);
        if (ctx->needs_input_grad(0)) grads[0] = group_product("expert_product gradient", by, v[1], v[2], true);
        if (ctx->needs_input_grad(1)) grads[1] = group_weight(v[0], by, v[1], v[2]);
        return once(std::move(grads), {arrive[0], v[0], v[1]});
    }
};
Tensor expert_product(const Tensor& x, const Tensor& weight, const Tensor& offsets) {
    const char* what = "expert_product";
    OneGpu gpu{what};
    gpu.add("x", x);
    gpu.add("weight", weight);
    gpu.add("offsets", offsets);
    TORCH_CHECK_VALUE(weight.dim() == 3, what, ": weight must be [experts, outputs, inputs], not ", weight.sizes());
    check_row_type(what, "x", x);
    TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type(), what, ": weight is ", name_of(weight.scalar_type()), ", x ",
                      name_of(x.scalar_type()));
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == weight.size(2), what, ": x must be [rows, ", weight.size(2), "], not ", x.sizes());
    TORCH_CHECK_VALUE(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.size(0) == weight.size(0) + 1, what,
                      ": offsets must be int32 [", weight.size(0) + 1, "], not ", name_of(offsets.scalar_type()), " ", offsets.sizes());
    TORCH_CHECK_VALUE(x.size(0) < (int64_t)1 << 31 && weight.size(0) <= 65536, what, ": more rows or experts than one call takes");
    if (wants_grad({x, weight})) return ExpertFunction::apply(x, weight, offsets);
    return group_product(what, x, weight, offsets, false);
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
    m.def("gradient_norm", &gradient_norm);   // these two read Python lists
    m.def("clip_gradients", &clip_gradients);
    m.def("route_experts", &route_experts, free);
    m.def("dispatch_rows", &dispatch_rows, free);
    m.def("combine_rows", &combine_rows, free);
    m.def("expert_product", &expert_product, free);
}
