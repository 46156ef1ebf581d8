// Autograd node of the token embedding for eager calls.
//
// A small training step is bound by the host, and a Python autograd Function costs it more than
// its kernels: 8,000 x 331 fp16, 1,021 tokens, lookup and gradient took 90 us a call that way and
// take 62 this way (an empty Python Function 38, a built-in view 34).  The node calls the C entry
// points, whose addresses bind() takes from the library that the package has loaded.  While
// torch.compile traces, the package uses its Python Function instead.
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "silogic_b200.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
    decltype(&slg_embed_fwd) embed_fwd;
    decltype(&slg_embed_bwd) embed_bwd;
    decltype(&slg_embed_bwd_workspace_bytes) embed_bwd_workspace_bytes;
    decltype(&slg_last_error) last_error;
} lib;

void check(int status, const char* name) {
    TORCH_CHECK(status == SLG_OK, name, " failed with status ", status, ": ", lib.last_error());
}

int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SLG_DT_F32;
        case at::kBFloat16: return SLG_DT_BF16;
        case at::kHalf: return SLG_DT_F16;
        default: TORCH_CHECK(false, "token_embedding: dtype ", t.scalar_type(), " not built");
    }
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

at::Tensor lookup(const at::Tensor& ids, const at::Tensor& weight, double scale) {
    const c10::DeviceGuard guard(weight.device());
    const at::Tensor w = weight.contiguous();
    auto shape = ids.sizes().vec();
    shape.push_back(w.size(1));
    at::Tensor out = at::empty(shape, w.options());
    check(lib.embed_fwd(ids.const_data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), w.const_data_ptr(), dtype_of(w),
                        w.size(0), w.size(1), (float)scale, out.mutable_data_ptr(), stream_of(w)),
          "slg_embed_fwd");
    return out;
}

at::Tensor gradient(const at::Tensor& ids, const at::Tensor& upstream, int64_t V, double scale, int64_t padding_idx) {
    const c10::DeviceGuard guard(upstream.device());
    const at::Tensor g = upstream.contiguous();
    const int64_t N = ids.numel(), D = g.size(-1);
    const int dt = dtype_of(g);
    at::Tensor gw = at::empty({V, D}, g.options());
    const int64_t bytes = lib.embed_bwd_workspace_bytes(N, V, D, dt);
    at::Tensor workspace = at::empty({bytes}, g.options().dtype(at::kByte));
    check(lib.embed_bwd(ids.const_data_ptr(), ids.scalar_type() == at::kLong, N, g.const_data_ptr(), dt, V, D, (float)scale,
                        padding_idx, gw.mutable_data_ptr(), workspace.mutable_data_ptr(), bytes, stream_of(g)),
          "slg_embed_bwd");
    return gw;
}

struct Lookup : torch::autograd::Function<Lookup> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& weight, double scale,
                              int64_t padding_idx);
    static variable_list backward(AutogradContext* ctx, variable_list g);
};

// The gradient as a (linear) function of the upstream one, for gradients of gradients.
struct Gradient : torch::autograd::Function<Gradient> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& g, int64_t V, double scale,
                              int64_t padding_idx);
    static variable_list backward(AutogradContext* ctx, variable_list gg);
};

void keep(AutogradContext* ctx, const at::Tensor& ids, int64_t V, double scale, int64_t padding_idx) {
    ctx->save_for_backward({ids});
    ctx->saved_data["V"] = V;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
}

at::Tensor Lookup::forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& weight, double scale,
                           int64_t padding_idx) {
    keep(ctx, ids, weight.size(0), scale, padding_idx);
    return lookup(ids, weight, scale);
}

variable_list Lookup::backward(AutogradContext* ctx, variable_list g) {
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const int64_t V = ctx->saved_data["V"].toInt(), pad = ctx->saved_data["padding_idx"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    // the grad mode is on under create_graph=True
    at::Tensor gw = at::GradMode::is_enabled() ? Gradient::apply(ids, g[0], V, scale, pad)
                                               : gradient(ids, g[0], V, scale, pad);
    return {at::Tensor(), std::move(gw), at::Tensor(), at::Tensor()};
}

at::Tensor Gradient::forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& g, int64_t V, double scale,
                             int64_t padding_idx) {
    keep(ctx, ids, V, scale, padding_idx);
    return gradient(ids, g, V, scale, padding_idx);
}

variable_list Gradient::backward(AutogradContext* ctx, variable_list gg) {
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const int64_t V = ctx->saved_data["V"].toInt(), pad = ctx->saved_data["padding_idx"].toInt();
    const at::Tensor rows = Lookup::apply(ids, gg[0], ctx->saved_data["scale"].toDouble(), pad);
    const at::Tensor counted = (ids >= 0) & (ids < V) & (ids != pad);       // the others add nothing to the gradient
    return {at::Tensor(), at::where(counted.unsqueeze(-1), rows, 0.0), at::Tensor(), at::Tensor(), at::Tensor()};
}

// Arguments are checked by the caller: CUDA tensors of one device, ids int32 or int64 and
// contiguous, weight [V, D], padding_idx in [-1, V).
at::Tensor token_embedding(const at::Tensor& ids, const at::Tensor& weight, double scale, int64_t padding_idx) {
    TORCH_CHECK(!weight._fw_grad(0).defined(), "token_embedding: forward-mode differentiation is not implemented");
    if (weight.requires_grad() && at::GradMode::is_enabled()) return Lookup::apply(ids, weight, scale, padding_idx);
    return lookup(ids, weight, scale);
}

void bind(uintptr_t embed_fwd, uintptr_t embed_bwd, uintptr_t embed_bwd_workspace_bytes, uintptr_t last_error) {
    lib.embed_fwd = reinterpret_cast<decltype(lib.embed_fwd)>(embed_fwd);
    lib.embed_bwd = reinterpret_cast<decltype(lib.embed_bwd)>(embed_bwd);
    lib.embed_bwd_workspace_bytes = reinterpret_cast<decltype(lib.embed_bwd_workspace_bytes)>(embed_bwd_workspace_bytes);
    lib.last_error = reinterpret_cast<decltype(lib.last_error)>(last_error);
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    m.def("bind", &bind);
    m.def("token_embedding", &token_embedding, pybind11::call_guard<pybind11::gil_scoped_release>());
}
