// row_autograd.cpp -- the row operators (model/row_ops.py) as autograd nodes in C++: argument checks, allocation and the calls of section 10 of holoscene_hip.h.
//
// Why not in Python over ctypes, as the other operators: a training step of these is two to nine launches, and below ~0.1 ms of them the host is what takes the
// time.  Python's part of a forward and backward pass, much of it on autograd's own thread with cold caches, was more than the launches (host time of a step as
// medians, through Python and here: gated block of 300 x 300 x 1 000 bf16 170 -> 100 us, lookup of 4 096 rows 101 -> 54, dropout 80 -> 46; a product by a number
// with its gradient takes 27 to 45).
//
// The library is the one that hashencoder/backend.py has loaded and checked; bind() receives its entry points.  Errors are raised as RuntimeError (TORCH_CHECK).
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <array>
#include <cmath>
#include <string>

#include "holoscene_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
    decltype(&hs_embed_fwd) embed_fwd;
    decltype(&hs_embed_bwd_ws_bytes) embed_bwd_ws_bytes;
    decltype(&hs_embed_bwd) embed_bwd;
    decltype(&hs_dropout_rows) dropout_rows;
    decltype(&hs_gated_mlp_saved_bytes) gated_saved_bytes;
    decltype(&hs_gated_mlp_fwd_ws_bytes) gated_fwd_ws_bytes;
    decltype(&hs_gated_mlp_bwd_ws_bytes) gated_bwd_ws_bytes;
    decltype(&hs_gated_mlp_fwd) gated_fwd;
    decltype(&hs_gated_mlp_bwd) gated_bwd;
} lib = {};

void bind(const py::dict &entries, int64_t abi_version) {
    TORCH_CHECK(abi_version == HS_ABI_VERSION, "_row_autograd.so was built for ABI version ", HS_ABI_VERSION, " of libholoscene_hip.so, which has ", abi_version,
                " -- rebuild (python -m holoscene_amd.csrc.build)");
    auto at = [&](const char *name) { return reinterpret_cast<void *>(entries[name].cast<uintptr_t>()); };
    lib.embed_fwd = reinterpret_cast<decltype(lib.embed_fwd)>(at("hs_embed_fwd"));
    lib.embed_bwd_ws_bytes = reinterpret_cast<decltype(lib.embed_bwd_ws_bytes)>(at("hs_embed_bwd_ws_bytes"));
    lib.embed_bwd = reinterpret_cast<decltype(lib.embed_bwd)>(at("hs_embed_bwd"));
    lib.dropout_rows = reinterpret_cast<decltype(lib.dropout_rows)>(at("hs_dropout_rows"));
    lib.gated_saved_bytes = reinterpret_cast<decltype(lib.gated_saved_bytes)>(at("hs_gated_mlp_saved_bytes"));
    lib.gated_fwd_ws_bytes = reinterpret_cast<decltype(lib.gated_fwd_ws_bytes)>(at("hs_gated_mlp_fwd_ws_bytes"));
    lib.gated_bwd_ws_bytes = reinterpret_cast<decltype(lib.gated_bwd_ws_bytes)>(at("hs_gated_mlp_bwd_ws_bytes"));
    lib.gated_fwd = reinterpret_cast<decltype(lib.gated_fwd)>(at("hs_gated_mlp_fwd"));
    lib.gated_bwd = reinterpret_cast<decltype(lib.gated_bwd)>(at("hs_gated_mlp_bwd"));
}

// ------------------------------------------------------------------------------------------------ checks, small helpers
int64_t checked(int64_t rc, const char *what) {
    TORCH_CHECK(rc >= 0, what, rc == HS_ERR_ARG ? ": sizes or types that the kernels do not take" : rc == HS_ERR_LAUNCH ? ": HIP kernel launch failed" :
                rc == HS_ERR_NULL ? ": required pointer was NULL" : ": failed");
    return rc;
}

int32_t row_type(at::ScalarType t, const char *name) {
    if (t == at::kFloat) return HS_F32;
    if (t == at::kBFloat16) return HS_BF16;
    TORCH_CHECK(t == at::kHalf, name, ": unsupported type ", t);
    return HS_F16;
}

// What would lose the operator without an error: a tangent (the call past autograd computes the value alone), a trace (it would record the result's allocation,
// not the launch that fills it).
void check_plain(const Tensor &t, const char *name) {
    TORCH_CHECK(!t._fw_grad(0).defined(), name, " has a tangent: the row operators do not take part in forward mode differentiation");
    TORCH_CHECK(!torch::jit::tracer::isTracing(), "the row operators cannot be traced (torch.jit.trace)");
}

void check_dense(const Tensor &t, const char *name) {
    check_plain(t, name);
    TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.layout() == at::kStrided, name, " must be a dense tensor");
}

void check_like(const Tensor &t, const char *name, const Tensor &other) {
    check_dense(t, name);
    TORCH_CHECK(t.device() == other.device(), name, " is on ", t.device(), ", expected ", other.device());
    TORCH_CHECK(t.scalar_type() == other.scalar_type(), name, " must be a ", other.scalar_type(), " tensor, got ", t.scalar_type());
}

// [..., n] -> 2-D with consecutive elements in a row: the tensor itself (any row distance >= n), else a copy.  (Here and in dropout(): a view that is negated when
// it is read, such as the imaginary part of a conjugate, is written out first.)
Tensor as_rows(const Tensor &t) {
    Tensor r = t.resolve_neg();
    if (t.dim() != 2) {
        int64_t rows = 1;
        for (int64_t d = 0; d + 1 < t.dim(); d++) rows *= t.size(d);
        r = r.reshape({rows, t.size(-1)});
    }
    if (r.is_contiguous() || ((r.size(1) <= 1 || r.stride(1) == 1) && (r.size(0) <= 1 || r.stride(0) >= r.size(1)))) return r;
    return r.contiguous();
}

// (a matrix of one row may carry any stride)
int64_t row_distance(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor bytes_on(const Tensor &t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// Gradients that cannot be differentiated again: where the caller asks for a graph of them (create_graph), whoever follows it is told so.  A gradient leads
// to the incoming one where that requires a gradient itself, and with `operands` to the operands whatever the incoming one is: in
// grad(y, x, ones, create_graph=True), a gradient penalty, it is a constant.
variable_list no_second_derivative(const variable_list &grads, variable_list out, bool operands = false) {
    if (!at::GradMode::is_enabled()) return out;
    bool any = operands;
    for (const Tensor &g : grads) any = any || (g.defined() && g.requires_grad());
    if (!any) return out;
    for (Tensor &t : out)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    auto node = std::make_shared<torch::autograd::DelayedError>("the row operators' gradients cannot be differentiated again", (int64_t)out.size());
    return (*node)(std::move(out));
}

bool recorded(std::initializer_list<const Tensor *> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ------------------------------------------------------------------------------------------------ codes by index
Tensor embed(const Tensor &indices, const Tensor &table, double scale, at::ScalarType out_type) {
    std::vector<int64_t> sizes(indices.sizes().begin(), indices.sizes().end());
    sizes.push_back(table.size(1));
    Tensor out = at::empty(sizes, table.options().dtype(out_type));
    if (out.numel() == 0) return out;
    const c10::DeviceGuard guard(table.device());
    const Tensor rows = as_rows(table);
    checked(lib.embed_fwd(indices.const_data_ptr(), (int32_t)indices.element_size(), rows.const_data_ptr(), row_distance(rows), out.mutable_data_ptr(), indices.numel(),
                          rows.size(0), rows.size(1), (float)scale, row_type(table.scalar_type(), "table"), row_type(out_type, "out_dtype"), stream_of(out)), "hs_embed_fwd");
    return out;
}

struct EmbeddingRows : torch::autograd::Function<EmbeddingRows> {
    static Tensor forward(AutogradContext *ctx, const Tensor &indices, const Tensor &table, double scale, int64_t padding, int64_t out_type) {
        ctx->save_for_backward({indices});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["type"] = (int64_t)table.scalar_type();
        return embed(indices, table, scale, (at::ScalarType)out_type);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(5);
        {
            const at::AutoGradMode off(false);
            const Tensor indices = ctx->get_saved_variables()[0], &g = grads[0];
            const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
            const int64_t V = ctx->saved_data["rows"].toInt(), D = g.size(-1);
            const c10::DeviceGuard guard(g.device());
            out[1] = at::empty({V, D}, g.options().dtype(type));
            if (out[1].numel() > 0) {
                const Tensor rows = as_rows(g);
                const int64_t n = indices.numel(), bytes = checked(lib.embed_bwd_ws_bytes(n, V, D), "hs_embed_bwd");
                const Tensor ws = bytes_on(g, bytes);
                checked(lib.embed_bwd(indices.const_data_ptr(), (int32_t)indices.element_size(), rows.const_data_ptr(), row_distance(rows), out[1].mutable_data_ptr(), n, V, D,
                                      (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), row_type(g.scalar_type(), "grad"),
                                      row_type(type, "table"), ws.mutable_data_ptr(), bytes, stream_of(g)), "hs_embed_bwd");
            }
        }
        return no_second_derivative(grads, std::move(out));
    }
};

Tensor embedding_rows(const Tensor &indices, const Tensor &table, double scale, std::optional<int64_t> padding, std::optional<at::ScalarType> out_type) {
    check_dense(table, "table");
    row_type(table.scalar_type(), "table");
    check_dense(indices, "indices");
    TORCH_CHECK(indices.device() == table.device(), "indices is on ", indices.device(), ", expected ", table.device());
    TORCH_CHECK(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong, "indices: unsupported type ", indices.scalar_type());
    TORCH_CHECK(table.dim() == 2, "table must be [V, D], got ", table.sizes());
    TORCH_CHECK(!padding || (*padding >= 0 && *padding < table.size(0)), "padding_idx ", *padding, " is outside the table's ", table.size(0), " rows");
    const at::ScalarType type = out_type.value_or(table.scalar_type());
    row_type(type, "out_dtype");
    const Tensor idx = indices.resolve_neg().contiguous();
    if (!recorded({&table})) return embed(idx, table, scale, type);
    return EmbeddingRows::apply(idx, table, scale, padding.value_or(-1), (int64_t)type);
}

// ------------------------------------------------------------------------------------------------ dropout
Tensor dropout(const Tensor &x, const Tensor &residual, int64_t drop, const Tensor &rng) {
    const Tensor in = x.resolve_neg().contiguous();
    Tensor y = at::empty_like(in);
    if (y.numel() == 0) return y;
    const c10::DeviceGuard guard(in.device());
    const Tensor r = residual.defined() ? residual.resolve_neg().contiguous() : residual;
    checked(lib.dropout_rows(in.const_data_ptr(), r.defined() ? r.const_data_ptr() : nullptr, y.mutable_data_ptr(), in.numel(), row_type(in.scalar_type(), "x"), (int32_t)drop,
                             (const uint64_t *)rng.const_data_ptr(), stream_of(in)), "hs_dropout_rows");
    return y;
}

// (rng is saved as a variable: autograd refuses the backward pass if it has been written in the meantime)
struct DropoutRows : torch::autograd::Function<DropoutRows> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &rng, int64_t drop) {
        ctx->save_for_backward({rng});
        ctx->saved_data["drop"] = drop;
        return dropout(x, Tensor(), drop, rng);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(3);
        {
            const at::AutoGradMode off(false);
            out[0] = dropout(grads[0], Tensor(), ctx->saved_data["drop"].toInt(), ctx->get_saved_variables()[0]);
        }
        return no_second_derivative(grads, std::move(out));
    }
};

struct DropoutAddRows : torch::autograd::Function<DropoutAddRows> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &residual, const Tensor &rng, int64_t drop) {
        ctx->save_for_backward({rng});
        ctx->saved_data["drop"] = drop;
        return dropout(x, residual, drop, rng);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(4);
        {
            const at::AutoGradMode off(false);
            const Tensor rng = ctx->get_saved_variables()[0];
            if (ctx->needs_input_grad(0)) out[0] = dropout(grads[0], Tensor(), ctx->saved_data["drop"].toInt(), rng);
            if (ctx->needs_input_grad(1)) out[1] = grads[0];
        }
        return no_second_derivative(grads, std::move(out));
    }
};

Tensor dropout_rows(const Tensor &x, double p, const Tensor &rng, const std::optional<Tensor> &residual) {
    check_dense(x, "x");
    row_type(x.scalar_type(), "x");
    check_dense(rng, "rng");
    TORCH_CHECK(rng.device() == x.device(), "rng is on ", rng.device(), ", expected ", x.device());
    TORCH_CHECK(rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2 && rng.is_contiguous() && !rng.is_neg(), "rng must be two consecutive int64 (seed, number of the call)");
    if (residual) {
        check_like(*residual, "residual", x);
        TORCH_CHECK(residual->sizes() == x.sizes(), "residual ", residual->sizes(), " must have x's shape ", x.sizes());
    }
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p);
    const auto drop = (int64_t)std::floor(p * 65536 + 0.5);
    if (!residual) return recorded({&x}) ? DropoutRows::apply(x, rng, drop) : dropout(x, Tensor(), drop, rng);
    return recorded({&x, &*residual}) ? DropoutAddRows::apply(x, *residual, rng, drop) : dropout(x, *residual, drop, rng);
}

// ------------------------------------------------------------------------------------------------ gated block
hsGatedMlp gated_args(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation) {
    hsGatedMlp a = {};
    a.x = x.const_data_ptr();
    a.w_gate = wg.const_data_ptr();
    a.w_up = wu.const_data_ptr();
    a.w_down = wd.const_data_ptr();
    a.ldx = row_distance(x);
    a.ld_gate = row_distance(wg);
    a.ld_up = row_distance(wu);
    a.ld_down = row_distance(wd);
    a.rows = x.size(0);
    a.dim = x.size(1);
    a.hidden = wg.size(0);
    a.dtype = row_type(x.scalar_type(), "x");
    a.activation = (int32_t)activation;
    return a;
}

template <typename F> void gated_call(hsGatedMlp &a, F call, int64_t bytes, const Tensor &x, const char *what) {
    Tensor ws;
    if (checked(bytes, what) > 0) {
        ws = bytes_on(x, bytes);
        a.ws = ws.mutable_data_ptr();
        a.ws_bytes = bytes;
    }
    checked(call(&a, stream_of(x)), what);
}

// y, of the given shape (its own memory and no view of it: a caller may write a result in place, which autograd refuses for views that a node returns), from 2-D
// rows; saved: receives what the backward pass reads
Tensor gated(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation, at::IntArrayRef shape, Tensor *saved) {
    const c10::DeviceGuard guard(x.device());
    hsGatedMlp a = gated_args(x, wg, wu, wd, activation);
    Tensor y = at::empty(shape, x.options());
    a.y = y.mutable_data_ptr();
    if (saved) {
        *saved = bytes_on(x, checked(lib.gated_saved_bytes(&a), "hs_gated_mlp_fwd"));
        a.saved = saved->mutable_data_ptr();
    }
    gated_call(a, lib.gated_fwd, lib.gated_fwd_ws_bytes(&a), x, "hs_gated_mlp_fwd");
    return y;
}

struct GatedMlpRows : torch::autograd::Function<GatedMlpRows> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation) {
        ctx->saved_data["shape"] = x.sizes().vec();
        // (every gradient depends on x, Wg or Wu; where Wd alone takes one, it depends on nothing that does)
        ctx->saved_data["again"] = x.requires_grad() || wg.requires_grad() || wu.requires_grad();
        if (x.numel() == 0 || wg.numel() == 0) {
            ctx->save_for_backward({x, wg, wu, wd});
            return at::zeros_like(x);
        }
        const Tensor rows = as_rows(x), g = as_rows(wg), u = as_rows(wu), d = as_rows(wd);
        Tensor saved, y = gated(rows, g, u, d, activation, x.sizes(), &saved);
        ctx->save_for_backward({rows, g, u, d, saved});
        ctx->saved_data["activation"] = activation;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(5);
        {
            const at::AutoGradMode off(false);
            const variable_list in = ctx->get_saved_variables();
            const c10::DeviceGuard guard(grads[0].device());
            if (in.size() == 4) {
                for (int i = 0; i < 4; i++)
                    if (ctx->needs_input_grad(i)) out[i] = at::zeros_like(in[i]);
            } else {
                hsGatedMlp a = gated_args(in[0], in[1], in[2], in[3], ctx->saved_data["activation"].toInt());
                const Tensor g = as_rows(grads[0]);
                a.grad = g.const_data_ptr();
                a.ld_grad = row_distance(g);
                a.saved = in[4].mutable_data_ptr();
                void **const to[4] = {&a.gx, &a.gw_gate, &a.gw_up, &a.gw_down};
                for (int i = 0; i < 4; i++)
                    if (ctx->needs_input_grad(i)) {
                        out[i] = at::empty(in[i].sizes(), in[i].options());
                        *to[i] = out[i].mutable_data_ptr();
                    }
                gated_call(a, lib.gated_bwd, lib.gated_bwd_ws_bytes(&a), g, "hs_gated_mlp_bwd");
                if (out[0].defined() && ctx->saved_data["shape"].toIntVector().size() != 2) out[0] = out[0].view(ctx->saved_data["shape"].toIntVector());
            }
        }
        return no_second_derivative(grads, std::move(out), ctx->saved_data["again"].toBool());
    }
};

Tensor gated_mlp_rows(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation) {
    check_dense(x, "x");
    row_type(x.scalar_type(), "x");
    TORCH_CHECK(x.dim() >= 1, "x must be [..., dim]");
    check_like(wg, "w_gate", x);
    check_like(wu, "w_up", x);
    check_like(wd, "w_down", x);
    TORCH_CHECK(wg.dim() == 2 && wu.dim() == 2 && wd.dim() == 2 && x.size(-1) == wg.size(1) && wu.sizes() == wg.sizes() && wd.size(0) == wg.size(1) && wd.size(1) == wg.size(0),
                "x ", x.sizes(), ", w_gate ", wg.sizes(), ", w_up ", wu.sizes(), ", w_down ", wd.sizes(), ": expected [..., dim], [hidden, dim], [hidden, dim], [dim, hidden]");
    TORCH_CHECK(wg.size(0) <= HS_GATED_MLP_MAX && wg.size(1) <= HS_GATED_MLP_MAX, "dim ", wg.size(1), " and hidden ", wg.size(0), " must be at most ", HS_GATED_MLP_MAX);
    TORCH_CHECK(x.size(-1) == 0 || x.numel() / x.size(-1) <= HS_GATED_MLP_MAX_ROWS, "x ", x.sizes(), " has more than ", HS_GATED_MLP_MAX_ROWS, " rows");
    TORCH_CHECK(activation < HS_GATED_ONE_PLANE || x.scalar_type() != at::kFloat, "planes is for the 16-bit types: a float32 operand is always three bf16 planes");
    if (recorded({&x, &wg, &wu, &wd})) return GatedMlpRows::apply(x, wg, wu, wd, activation);
    if (x.numel() == 0 || wg.size(0) == 0) return at::zeros_like(x);
    return gated(as_rows(x), as_rows(wg), as_rows(wu), as_rows(wd), activation, x.sizes(), nullptr);
}

}  // namespace

PYBIND11_MODULE(_row_autograd, m) {
    m.def("bind", &bind);
    m.def("embedding_rows", &embedding_rows);
    m.def("dropout_rows", &dropout_rows);
    m.def("gated_mlp_rows", &gated_mlp_rows);
}
