// Autograd nodes of the fused mHC layers in C++ over the C ABI of
// libmhc_hip (the role of the reference's Python autograd functions,
// src/python/mhc/ops.py:387-564, and of its pybind11 layer entries,
// src/python/bindings.cpp:600-952).  Forward and backward prepare their
// arguments exactly as mhc_ascend_amd/native.py does (same checks, dtypes,
// workspaces and error text) and call the same entry points, so results are
// identical bit for bit; doing it in C++ keeps the interpreter out of the
// forward and the autograd engine's hand-off to a Python backward out of
// every step.
//
// The fused MHCResidualWrapper (layer.py:269-322) has nodes of the same kind.
// These nodes are the package's only orchestration of the fused entries;
// tests/pyref_autograd.py restates them in Python for a bit-for-bit check.
//
// The entry points are not linked: bind() receives their addresses from the
// ctypes handle of the already loaded library, so both paths share one copy
// of it (one error state, one set of per-device caches) whichever build of
// it was loaded.
#include <torch/extension.h>

#include <ATen/hip/HIPContext.h>

#include <algorithm>
#include <map>
#include <string>
#include <vector>

#include "mhc_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

#define MHC_AUTOGRAD_ENTRIES(X)               \
    X(mhc_last_error)                         \
    X(mhc_layer_static_saved_size)            \
    X(mhc_layer_static_fwd)                   \
    X(mhc_layer_static_bwd_workspace_size)    \
    X(mhc_layer_static_bwd)                   \
    X(mhc_layer_dynamic_saved_size)           \
    X(mhc_layer_dynamic_fwd_workspace_size)   \
    X(mhc_layer_dynamic_fwd)                  \
    X(mhc_layer_dynamic_bwd_workspace_size)   \
    X(mhc_layer_dynamic_bwd)                  \
    X(mhc_layer_dynamic_packed_size)          \
    X(mhc_layer_dynamic_infer_workspace_size) \
    X(mhc_layer_dynamic_infer)                \
    X(mhc_sinkhorn_knopp_fwd)                 \
    X(mhc_sinkhorn_knopp_bwd)                 \
    X(mhc_rmsnorm_fwd)                        \
    X(mhc_rmsnorm_bwd_workspace_size)         \
    X(mhc_rmsnorm_bwd)                        \
    X(mhc_stream_aggregate_fwd)               \
    X(mhc_stream_aggregate_bwd)               \
    X(mhc_stream_distribute_mix_add_fwd)      \
    X(mhc_stream_distribute_mix_add_bwd)      \
    X(mhc_wrapper_dynamic_saved_size)         \
    X(mhc_wrapper_dynamic_fwd_workspace_need) \
    X(mhc_wrapper_dynamic_fwd)                \
    X(mhc_wrapper_dynamic_bwd_workspace_need) \
    X(mhc_wrapper_dynamic_bwd)                \
    X(mhc_wrapper_static_fwd)                 \
    X(mhc_wrapper_static_bwd_workspace_size)  \
    X(mhc_wrapper_static_bwd)                 \
    X(mhc_checkpoint_values_size)             \
    X(mhc_checkpoint_scales_size)             \
    X(mhc_checkpoint_pack)                    \
    X(mhc_checkpoint_unpack)                  \
    X(mhc_rmsnorm_checkpoint_fwd)             \
    X(mhc_rmsnorm_checkpoint_bwd_workspace_size) \
    X(mhc_rmsnorm_checkpoint_bwd)             \
    X(mhc_layer_static_checkpoint_fwd)        \
    X(mhc_layer_static_checkpoint_bwd_workspace_need) \
    X(mhc_layer_static_checkpoint_bwd)        \
    X(mhc_layer_dynamic_checkpoint_fwd)       \
    X(mhc_layer_dynamic_checkpoint_bwd_workspace_need) \
    X(mhc_layer_dynamic_checkpoint_bwd)       \
    X(mhc_dropout)                            \
    X(mhc_rmsnorm_residual_fwd)               \
    X(mhc_rmsnorm_residual_bwd_workspace_size) \
    X(mhc_rmsnorm_residual_bwd)               \
    X(mhc_qk_norm_rope_fwd)                   \
    X(mhc_qk_norm_rope_bwd_workspace_size)    \
    X(mhc_qk_norm_rope_bwd)                   \
    X(mhc_qk_norm_rope_axes_fwd)              \
    X(mhc_qk_norm_rope_axes_bwd)              \
    X(mhc_qk_rope)

struct Entries {
#define MHC_DECLARE(name) decltype(&::name) name = nullptr;
    MHC_AUTOGRAD_ENTRIES(MHC_DECLARE)
#undef MHC_DECLARE
};

Entries lib;
bool bound = false;

void bind(const std::map<std::string, int64_t>& addrs) {
    Entries e;
#define MHC_BIND(name)                                                                            \
    {                                                                                             \
        auto it = addrs.find(#name);                                                              \
        TORCH_CHECK(it != addrs.end() && it->second != 0, "mhc autograd: no address for " #name); \
        e.name = reinterpret_cast<decltype(e.name)>(static_cast<intptr_t>(it->second));           \
    }
    MHC_AUTOGRAD_ENTRIES(MHC_BIND)
#undef MHC_BIND
    lib = e;
    bound = true;
}

std::vector<std::string> entry_names() {
    return {
#define MHC_NAME(name) #name,
        MHC_AUTOGRAD_ENTRIES(MHC_NAME)
#undef MHC_NAME
    };
}

void require_bound() { TORCH_CHECK(bound, "mhc autograd: bind() the HIP library's entry points first"); }

int dtype_code(at::ScalarType t) {
    if (t == at::kFloat) return MHC_DTYPE_F32;
    if (t == at::kBFloat16) return MHC_DTYPE_BF16;
    TORCH_CHECK(false, "mhc_ascend_amd: unsupported storage dtype ", t, " (float32 or bfloat16)");
    return -1;
}

void check(int rc, const char* name) {
    TORCH_CHECK(rc == 0, name, " failed (status ", rc, "): ", lib.mhc_last_error());
}

void check_device(const char* fn, std::initializer_list<const Tensor*> ts) {
    c10::optional<c10::Device> dev;
    for (const Tensor* t : ts) {
        TORCH_CHECK(t->is_cuda(), fn, ": tensors must be on a HIP device (got ", t->device(),
                    "); mhc_ascend_amd has no CPU path");
        if (!dev) {
            dev = t->device();
        } else {
            TORCH_CHECK(t->device() == *dev, fn, ": all tensors must be on the same device (", *dev, " vs ",
                        t->device(), ")");
        }
    }
}

bool storage_dtype(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

Tensor layer_x(const char* fn, const Tensor& x) {
    TORCH_CHECK(x.dim() == 3, fn, ": x must be 3D [B, n, C]");
    return (storage_dtype(x.scalar_type()) ? x : x.to(at::kFloat)).contiguous();
}

Tensor weight(const Tensor& w) { return (storage_dtype(w.scalar_type()) ? w : w.to(at::kFloat)).contiguous(); }

Tensor f32c(const Tensor& t) {
    if (t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
    return t.to(at::kFloat).contiguous();
}

// alpha as a one-element fp32 device tensor of its own shape (a device
// pointer: no host sync)
Tensor scalar_param(const Tensor& a, c10::Device dev) {
    TORCH_CHECK(a.numel() == 1, "alpha must have one element, got shape ", a.sizes());
    if (a.device() == dev) return f32c(a);
    return a.detach().to(dev, at::kFloat).contiguous();
}

// A contiguous tensor of `sizes` over part of a contiguous buffer, from
// element `offset` on.
Tensor part_of(const Tensor& buf, at::IntArrayRef sizes, int64_t offset) {
    c10::SmallVector<int64_t, 4> strides(sizes.size());
    int64_t st = 1;
    for (size_t i = sizes.size(); i-- > 0;) {
        strides[i] = st;
        st *= sizes[i] > 0 ? sizes[i] : 1;
    }
    return buf.as_strided(sizes, strides, offset);
}

// Appends the gradients of (phi_pre, phi_post, phi_res, alpha_pre, alpha_post,
// alpha_res, b_pre, b_post, b_res), in the parameters' shapes, over the
// entry's three gradient buffers.
void push_param_grads(tensor_list& out, const at::IntArrayRef (&shapes)[9], int64_t n, const Tensor& gphi,
                      const Tensor& galpha, const Tensor& gb) {
    const Tensor* bufs[3] = {&gphi, &galpha, &gb};
    const int64_t nC = gphi.size(1);
    const int64_t want[3][3] = {{n * nC, n * nC, n * n * nC}, {1, 1, 1}, {n, n, n * n}};
    for (int k = 0; k < 3; ++k) {
        int64_t off = 0;
        for (int i = 0; i < 3; ++i) {
            const at::IntArrayRef shape = shapes[3 * k + i];
            TORCH_CHECK(c10::multiply_integers(shape) == want[k][i], "dynamic layer: parameter of shape ", shape,
                        " does not match n = ", n);
            out.push_back(part_of(*bufs[k], shape, off));
            off += want[k][i];
        }
    }
}

Tensor workspace(size_t nbytes, const Tensor& like) {
    return at::empty({(int64_t)std::max<size_t>(nbytes, 1)}, like.options().dtype(at::kByte));
}

void* stream() { return at::hip::getCurrentHIPStream().stream(); }

float* fp(const Tensor& t) { return t.data_ptr<float>(); }

// ---- 8-bit checkpoints of saved rows ---------------------------------------------
// A node called with a format (MHC_CHECKPOINT_INT8 / _E4M3) saves the rows its
// backward reads in 8 bits; MHC_CHECKPOINT_NONE saves them as they are.
struct Held {
    Tensor values, scales;
};

Held held_alloc(const Tensor& x) {
    const int64_t C = x.size(-1), rows = C > 0 ? x.numel() / C : 0;
    TORCH_CHECK(C >= 1 && C <= INT32_MAX, "checkpoint: rows of ", C, " values");
    const auto opt = x.options().dtype(at::kByte);
    return {at::empty({(int64_t)lib.mhc_checkpoint_values_size(rows, (int32_t)C)}, opt),
            at::empty({(int64_t)lib.mhc_checkpoint_scales_size(rows, (int32_t)C)}, opt)};
}

// The same in the shapes that a caller sees: [..., ceil16(C)] and [..., ceil(C / 32)].
Held packed_alloc(const Tensor& x) {
    const auto opt = x.options().dtype(at::kByte);
    at::DimVector shape(x.sizes());
    const int64_t C = shape.back();
    shape.back() = (C + 15) / 16 * 16;
    Tensor values = at::empty(shape, opt);
    shape.back() = (C + 31) / 32;
    return {values, at::empty(shape, opt)};
}

// x contiguous, in storage dtype
Held hold(const Tensor& x, int64_t fmt) {
    Held h = held_alloc(x);
    const int64_t C = x.size(-1);
    check(lib.mhc_checkpoint_pack(x.data_ptr(), dtype_code(x.scalar_type()), (int32_t)fmt, h.values.data_ptr(),
                                  h.scales.data_ptr(), x.numel() / C, (int32_t)C, stream()),
          "mhc_checkpoint_pack");
    return h;
}

Tensor held_rows(const Tensor& values, const Tensor& scales, int64_t fmt, at::IntArrayRef sizes, at::ScalarType dt) {
    Tensor x = at::empty(sizes, values.options().dtype(dt));
    const int64_t C = sizes.back();
    check(lib.mhc_checkpoint_unpack(values.data_ptr(), scales.data_ptr(), (int32_t)fmt, x.data_ptr(), dtype_code(dt),
                                    x.numel() / C, (int32_t)C, stream()),
          "mhc_checkpoint_unpack");
    return x;
}

// The format a call runs with: none where no backward will read the rows.
int64_t format_for(int64_t fmt, std::initializer_list<const Tensor*> inputs) {
    TORCH_CHECK(fmt >= MHC_CHECKPOINT_NONE && fmt <= MHC_CHECKPOINT_E4M3, "unknown checkpoint format ", fmt);
    if (fmt == MHC_CHECKPOINT_NONE || !at::GradMode::is_enabled()) return MHC_CHECKPOINT_NONE;
    for (const Tensor* t : inputs)
        if (t->requires_grad()) return fmt;
    return MHC_CHECKPOINT_NONE;
}

// The format a node saved its rows in, under "fmt"; a node without one saves none.
int64_t saved_format(AutogradContext* ctx) {
    const auto it = ctx->saved_data.find("fmt");
    return it == ctx->saved_data.end() ? MHC_CHECKPOINT_NONE : it->second.toInt();
}

// ---- static H: mhc_ascend_amd.ops.MHCLayerStaticFunction (layer.py:142-170) --
struct StaticLayer : public torch::autograd::Function<StaticLayer> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in, const Tensor& hp_in,
                          const Tensor& hq_in, const Tensor& hr_in, int64_t iters, double sk_eps, double rms_eps,
                          int64_t fmt) {
        const char* fn = "mhc_layer_static_fwd";
        check_device(fn, {&x_in, &w_in, &hp_in, &hq_in, &hr_in});
        const at::DeviceGuard guard(x_in.device());
        const Tensor x = layer_x(fn, x_in);
        const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
        TORCH_CHECK(w_in.numel() == C && hp_in.numel() == n && hq_in.numel() == n && hr_in.numel() == n * n,
                    "mhc_layer_static_fwd: parameter shapes do not match x [B, n, C]");
        const Tensor w = weight(w_in), hp = f32c(hp_in), hq = f32c(hq_in), hr = f32c(hr_in);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor out = at::empty({B, n, C}, f32);
        Tensor saved = at::empty({(int64_t)(lib.mhc_layer_static_saved_size((int32_t)n, (int32_t)C) / 4)}, f32);
        ctx->saved_data["x_dtype"] = (int64_t)x_in.scalar_type();
        ctx->saved_data["cfg"] = std::vector<double>{(double)iters, sk_eps, rms_eps};
        if (fmt != MHC_CHECKPOINT_NONE) {
            ctx->saved_data["fmt"] = fmt;
            const Held held = held_alloc(x);
            check(lib.mhc_layer_static_checkpoint_fwd(
                      x.data_ptr(), dtype_code(x.scalar_type()), w.data_ptr(), dtype_code(w.scalar_type()), fp(hp),
                      fp(hq), fp(hr), fp(out), fp(saved), (int32_t)fmt, held.values.data_ptr(),
                      held.scales.data_ptr(), B, (int32_t)n, (int32_t)C, (int32_t)iters, (float)sk_eps,
                      (float)rms_eps, stream()),
                  "mhc_layer_static_checkpoint_fwd");
            ctx->saved_data["sizes"] = x.sizes().vec();
            ctx->saved_data["store"] = (int64_t)x.scalar_type();
            ctx->save_for_backward({held.values, w, hp, hq, hr, saved, held.scales});
            return out;
        }
        Tensor rms = at::empty({B}, f32);
        check(lib.mhc_layer_static_fwd(x.data_ptr(), dtype_code(x.scalar_type()), w.data_ptr(),
                                       dtype_code(w.scalar_type()), fp(hp), fp(hq), fp(hr), fp(out), fp(rms),
                                       fp(saved), B, (int32_t)n, (int32_t)C, (int32_t)iters, (float)sk_eps,
                                       (float)rms_eps, stream()),
              fn);
        ctx->save_for_backward({x, w, hp, hq, hr, saved});
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "mhc_layer_static_bwd";
        const auto sv = ctx->get_saved_variables();
        const Tensor &x = sv[0], &w = sv[1], &hp = sv[2], &hq = sv[3], &hr = sv[4], &saved = sv[5];
        check_device(fn, {&grads[0], &x});
        const at::DeviceGuard guard(x.device());
        const auto cfg = ctx->saved_data["cfg"].toDoubleVector();
        const int64_t fmt = saved_format(ctx);
        const bool is_held = fmt != MHC_CHECKPOINT_NONE;  // x is the checkpoint's values then
        const auto sizes = is_held ? ctx->saved_data["sizes"].toIntVector() : x.sizes().vec();
        const auto store = is_held ? (at::ScalarType)ctx->saved_data["store"].toInt() : x.scalar_type();
        const int64_t B = sizes[0], n = sizes[1], C = sizes[2];
        TORCH_CHECK(grads[0].sizes() == sizes, "mhc_layer_static_bwd: grad_out must match x [B, n, C]");
        const Tensor g = f32c(grads[0]);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor grad_x = at::empty(sizes, x.options().dtype(store));
        Tensor gw = at::empty({C}, w.options());
        Tensor ghp = at::empty(hp.sizes(), f32), ghq = at::empty(hq.sizes(), f32), ghr = at::empty(hr.sizes(), f32);
        const int xd = dtype_code(store);
        if (is_held) {
            const size_t wsb = lib.mhc_layer_static_checkpoint_bwd_workspace_need(
                fp(g), grad_x.data_ptr(), fp(saved), B, (int32_t)n, (int32_t)C, xd);
            Tensor ws = workspace(wsb, x);
            check(lib.mhc_layer_static_checkpoint_bwd(
                      fp(g), x.data_ptr(), sv[6].data_ptr(), (int32_t)fmt, xd, dtype_code(w.scalar_type()), fp(hp),
                      fp(hq), fp(hr), fp(saved), grad_x.data_ptr(), gw.data_ptr(), fp(ghp), fp(ghq), fp(ghr),
                      ws.data_ptr(), wsb, B, (int32_t)n, (int32_t)C, (int32_t)cfg[0], (float)cfg[1], (float)cfg[2],
                      stream()),
                  "mhc_layer_static_checkpoint_bwd");
        } else {
            const size_t wsb = lib.mhc_layer_static_bwd_workspace_size(B, (int32_t)n, (int32_t)C, xd);
            Tensor ws = workspace(wsb, x);
            check(lib.mhc_layer_static_bwd(fp(g), x.data_ptr(), xd, dtype_code(w.scalar_type()), fp(hp), fp(hq),
                                           fp(hr), fp(saved), grad_x.data_ptr(), gw.data_ptr(), fp(ghp), fp(ghq),
                                           fp(ghr), ws.data_ptr(), wsb, B, (int32_t)n, (int32_t)C, (int32_t)cfg[0],
                                           (float)cfg[1], (float)cfg[2], stream()),
                  fn);
        }
        const auto x_dtype = (at::ScalarType)ctx->saved_data["x_dtype"].toInt();
        return {grad_x.to(x_dtype), gw, ghp, ghq, ghr, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ---- dynamic H: mhc_ascend_amd.ops.MHCLayerDynamicFunction (ops.py:387-564) --
std::vector<Tensor> phi_parts(const Tensor& pre, const Tensor& post, const Tensor& res, int64_t n, int64_t nC) {
    std::vector<Tensor> parts = {f32c(pre), f32c(post), f32c(res)};
    const int64_t rows[3] = {n, n, n * n};
    for (int i = 0; i < 3; ++i) {
        TORCH_CHECK(parts[i].numel() == rows[i] * nC, "dynamic layer: projection of ", parts[i].sizes(),
                    " does not match [", rows[i], ", ", nC, "]");
    }
    return parts;
}

struct DynamicLayer : public torch::autograd::Function<DynamicLayer> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in, const Tensor& pp_in,
                          const Tensor& pq_in, const Tensor& pr_in, const Tensor& ap_in, const Tensor& aq_in,
                          const Tensor& ar_in, const Tensor& bp_in, const Tensor& bq_in, const Tensor& br_in,
                          int64_t iters, double sk_eps, double rms_eps, int64_t fmt) {
        const char* fn = "mhc_layer_dynamic_fwd";
        check_device(fn, {&x_in, &w_in, &pp_in, &pq_in, &pr_in, &bp_in, &bq_in, &br_in});
        const at::DeviceGuard guard(x_in.device());
        const Tensor x = layer_x(fn, x_in);
        const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
        const Tensor w = weight(w_in);
        TORCH_CHECK(w.numel() == C, "mhc_layer_dynamic_fwd: rmsnorm_weight must have C elements");
        const auto ph = phi_parts(pp_in, pq_in, pr_in, n, n * C);
        const Tensor ap = scalar_param(ap_in, x.device()), aq = scalar_param(aq_in, x.device()),
                     ar = scalar_param(ar_in, x.device());
        const Tensor bp = f32c(bp_in), bq = f32c(bq_in), br = f32c(br_in);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor out = at::empty({B, n, C}, f32);
        Tensor saved = at::empty({(int64_t)(lib.mhc_layer_dynamic_saved_size(B, (int32_t)n, (int32_t)C) / 4)}, f32);
        const size_t wsb = lib.mhc_layer_dynamic_fwd_workspace_size(B, (int32_t)n, (int32_t)C);
        Tensor ws = workspace(wsb, x);
        ctx->saved_data["x_dtype"] = (int64_t)x_in.scalar_type();
        ctx->saved_data["cfg"] = std::vector<double>{(double)iters, sk_eps, rms_eps};
        if (fmt != MHC_CHECKPOINT_NONE) {
            ctx->saved_data["fmt"] = fmt;
            const Held held = held_alloc(x);
            check(lib.mhc_layer_dynamic_checkpoint_fwd(
                      x.data_ptr(), dtype_code(x.scalar_type()), w.data_ptr(), dtype_code(w.scalar_type()), fp(ph[0]),
                      fp(ph[1]), fp(ph[2]), fp(ap), fp(aq), fp(ar), fp(bp), fp(bq), fp(br), fp(out), fp(saved),
                      (int32_t)fmt, held.values.data_ptr(), held.scales.data_ptr(), ws.data_ptr(), wsb, B, (int32_t)n,
                      (int32_t)C, (int32_t)iters, (float)sk_eps, (float)rms_eps, stream()),
                  "mhc_layer_dynamic_checkpoint_fwd");
            ctx->saved_data["sizes"] = x.sizes().vec();
            ctx->saved_data["store"] = (int64_t)x.scalar_type();
            ctx->save_for_backward(
                {held.values, w, saved, ph[0], ph[1], ph[2], ap, aq, ar, bp, bq, br, held.scales});
            return out;
        }
        check(lib.mhc_layer_dynamic_fwd(x.data_ptr(), dtype_code(x.scalar_type()), w.data_ptr(),
                                        dtype_code(w.scalar_type()), fp(ph[0]), fp(ph[1]), fp(ph[2]), fp(ap), fp(aq),
                                        fp(ar), fp(bp), fp(bq), fp(br), fp(out), fp(saved), ws.data_ptr(), wsb, B,
                                        (int32_t)n, (int32_t)C, (int32_t)iters, (float)sk_eps, (float)rms_eps,
                                        stream()),
              fn);
        ctx->save_for_backward({x, w, saved, ph[0], ph[1], ph[2], ap, aq, ar, bp, bq, br});
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "mhc_layer_dynamic_bwd";
        const auto sv = ctx->get_saved_variables();
        const Tensor &x = sv[0], &w = sv[1], &saved = sv[2];
        check_device(fn, {&grads[0], &x});
        const at::DeviceGuard guard(x.device());
        const auto cfg = ctx->saved_data["cfg"].toDoubleVector();
        const int64_t fmt = saved_format(ctx);
        const bool is_held = fmt != MHC_CHECKPOINT_NONE;  // x is the checkpoint's values then
        const auto sizes = is_held ? ctx->saved_data["sizes"].toIntVector() : x.sizes().vec();
        const auto store = is_held ? (at::ScalarType)ctx->saved_data["store"].toInt() : x.scalar_type();
        const int64_t B = sizes[0], n = sizes[1], C = sizes[2], np = 2 * n + n * n;
        TORCH_CHECK(grads[0].sizes() == sizes, "mhc_layer_dynamic_bwd: grad_output must match x [B, n, C]");
        const Tensor g = f32c(grads[0]);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor grad_x = at::empty(sizes, x.options().dtype(store));
        Tensor gw = at::empty({C}, w.options());
        Tensor gphi = at::empty({np, n * C}, f32);
        Tensor galpha = at::empty({3}, f32);
        Tensor gb = at::empty({np}, f32);
        const int xd = dtype_code(store);
        if (is_held) {
            const size_t wsb = lib.mhc_layer_dynamic_checkpoint_bwd_workspace_need(
                fp(g), grad_x.data_ptr(), fp(saved), B, (int32_t)n, (int32_t)C, xd, (int32_t)cfg[0]);
            Tensor ws = workspace(wsb, x);
            check(lib.mhc_layer_dynamic_checkpoint_bwd(
                      fp(g), x.data_ptr(), sv[12].data_ptr(), (int32_t)fmt, xd, dtype_code(w.scalar_type()), fp(sv[3]),
                      fp(sv[4]), fp(sv[5]), fp(sv[6]), fp(sv[7]), fp(sv[8]), fp(sv[9]), fp(sv[10]), fp(sv[11]),
                      fp(saved), grad_x.data_ptr(), gw.data_ptr(), fp(gphi), fp(galpha), fp(gb), ws.data_ptr(), wsb, B,
                      (int32_t)n, (int32_t)C, (int32_t)cfg[0], (float)cfg[1], (float)cfg[2], stream()),
                  "mhc_layer_dynamic_checkpoint_bwd");
        } else {
            const size_t wsb = lib.mhc_layer_dynamic_bwd_workspace_size(B, (int32_t)n, (int32_t)C, xd);
            Tensor ws = workspace(wsb, x);
            check(lib.mhc_layer_dynamic_bwd(fp(g), x.data_ptr(), xd, dtype_code(w.scalar_type()), fp(sv[3]),
                                            fp(sv[4]), fp(sv[5]), fp(sv[6]), fp(sv[7]), fp(sv[8]), fp(sv[9]),
                                            fp(sv[10]), fp(sv[11]), fp(saved), grad_x.data_ptr(), gw.data_ptr(),
                                            fp(gphi), fp(galpha), fp(gb), ws.data_ptr(), wsb, B, (int32_t)n,
                                            (int32_t)C, (int32_t)cfg[0], (float)cfg[1], (float)cfg[2], stream()),
                  fn);
        }
        const auto x_dtype = (at::ScalarType)ctx->saved_data["x_dtype"].toInt();
        tensor_list out;
        out.reserve(15);
        out.push_back(grad_x.to(x_dtype));
        out.push_back(gw);
        push_param_grads(out,
                         {sv[3].sizes(), sv[4].sizes(), sv[5].sizes(), sv[6].sizes(), sv[7].sizes(), sv[8].sizes(),
                          sv[9].sizes(), sv[10].sizes(), sv[11].sizes()},
                         n, gphi, galpha, gb);
        out.resize(15);
        return out;
    }
};

// ---- fused MHCResidualWrapper (layer.py:269-322) ----------------------------
// residual / branch [tokens, hidden] as the kernels read them: residual in
// fp32 or bf16 (others become fp32), branch in the residual's dtype.
std::pair<Tensor, Tensor> wrapper_inputs(const char* fn, const Tensor& residual, const Tensor& branch) {
    check_device(fn, {&residual, &branch});
    TORCH_CHECK(residual.sizes() == branch.sizes() && residual.dim() == 2, fn,
                ": residual and branch must both be [tokens, hidden] of one shape");
    Tensor r = (storage_dtype(residual.scalar_type()) ? residual : residual.to(at::kFloat)).contiguous();
    return {r, branch.to(r.scalar_type()).contiguous()};
}

int32_t wrapper_mode(const std::string& mode, int64_t n, const char* fn) {
    TORCH_CHECK_VALUE(mode == "decay" || mode == "zero", "Unknown residual_mode: ", mode);
    // the reference writes stream 1 (layer.py:301), which needs n >= 2
    TORCH_CHECK(n >= 2, fn, ": expansion_rate must be >= 2 (stream 1 holds the branch)");
    return mode == "decay" ? MHC_WRAPPER_DECAY : MHC_WRAPPER_ZERO;
}

// The wrapper's saved list: its two rows, `rest`, and with a checkpoint the
// rows' scales behind them.
void save_wrapper_rows(AutogradContext* ctx, int64_t fmt, const Tensor& r, const Tensor& b, tensor_list rest) {
    tensor_list sv = {r, b};
    if (fmt != MHC_CHECKPOINT_NONE) {
        ctx->saved_data["fmt"] = fmt;
        const Held hr = hold(r, fmt), hb = hold(b, fmt);
        sv = {hr.values, hb.values};
        rest.push_back(hr.scales);
        rest.push_back(hb.scales);
        ctx->saved_data["sizes"] = r.sizes().vec();
        ctx->saved_data["store"] = (int64_t)r.scalar_type();
    }
    sv.insert(sv.end(), rest.begin(), rest.end());
    ctx->save_for_backward(std::move(sv));
}

std::pair<Tensor, Tensor> wrapper_rows(AutogradContext* ctx, const tensor_list& sv) {
    const int64_t fmt = saved_format(ctx);
    if (fmt == MHC_CHECKPOINT_NONE) return {sv[0], sv[1]};
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const auto store = (at::ScalarType)ctx->saved_data["store"].toInt();
    return {held_rows(sv[0], sv[sv.size() - 2], fmt, sizes, store),
            held_rows(sv[1], sv[sv.size() - 1], fmt, sizes, store)};
}

struct StaticWrapper : public torch::autograd::Function<StaticWrapper> {
    static Tensor forward(AutogradContext* ctx, const Tensor& res_in, const Tensor& br_in, const Tensor& w_in,
                          const Tensor& hp_in, const Tensor& hq_in, const Tensor& hr_in, int64_t mode, int64_t n,
                          int64_t iters, double sk_eps, double rms_eps, int64_t fmt) {
        const char* fn = "wrapper_static_fwd";
        auto [r, b] = wrapper_inputs(fn, res_in, br_in);
        check_device(fn, {&r, &w_in, &hp_in, &hq_in, &hr_in});
        const at::DeviceGuard guard(r.device());
        const int64_t T = r.size(0), C = r.size(1);
        const Tensor w = weight(w_in);
        TORCH_CHECK(w.numel() == C && hp_in.numel() == n && hq_in.numel() == n && hr_in.numel() == n * n,
                    "wrapper_static_fwd: parameter shapes do not match n and C");
        const Tensor hp = f32c(hp_in), hq = f32c(hq_in), hr = f32c(hr_in);
        const auto f32 = r.options().dtype(at::kFloat);
        Tensor out = at::empty({T, C}, f32);
        Tensor saved = at::empty({(int64_t)(lib.mhc_layer_static_saved_size((int32_t)n, (int32_t)C) / 4)}, f32);
        check(lib.mhc_wrapper_static_fwd(r.data_ptr(), b.data_ptr(), dtype_code(r.scalar_type()), (int32_t)mode,
                                         w.data_ptr(), dtype_code(w.scalar_type()), fp(hp), fp(hq), fp(hr), fp(out),
                                         fp(saved), T, (int32_t)n, (int32_t)C, (int32_t)iters, (float)sk_eps,
                                         (float)rms_eps, stream()),
              "mhc_wrapper_static_fwd");
        save_wrapper_rows(ctx, fmt, r, b, {w, hp, hq, hr, saved});
        ctx->saved_data["dtypes"] = std::vector<int64_t>{(int64_t)res_in.scalar_type(), (int64_t)br_in.scalar_type()};
        ctx->saved_data["cfg"] = std::vector<double>{(double)mode, (double)n, (double)iters, sk_eps, rms_eps};
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "wrapper_static_bwd";
        const auto sv = ctx->get_saved_variables();
        check_device(fn, {&grads[0], &sv[0]});
        const at::DeviceGuard guard(sv[0].device());
        const auto [r, b] = wrapper_rows(ctx, sv);
        const Tensor &w = sv[2], &saved = sv[6];
        const auto cfg = ctx->saved_data["cfg"].toDoubleVector();
        const int64_t T = r.size(0), C = r.size(1), n = (int64_t)cfg[1];
        const int32_t mode = (int32_t)cfg[0];
        TORCH_CHECK(grads[0].sizes() == r.sizes(), "wrapper_static_bwd: grad_out must be [tokens, hidden]");
        const Tensor g = f32c(grads[0]);
        const auto f32 = r.options().dtype(at::kFloat);
        Tensor gr = at::empty_like(r), gb = at::empty_like(b);
        Tensor gw = at::empty({C}, w.options());
        Tensor ghp = at::empty(sv[3].sizes(), f32), ghq = at::empty(sv[4].sizes(), f32),
               ghr = at::empty(sv[5].sizes(), f32);
        const int dt = dtype_code(r.scalar_type());
        const size_t wsb = lib.mhc_wrapper_static_bwd_workspace_size(T, (int32_t)n, (int32_t)C, dt, mode);
        Tensor ws = workspace(wsb, r);
        check(lib.mhc_wrapper_static_bwd(fp(g), r.data_ptr(), b.data_ptr(), dt, mode, dtype_code(w.scalar_type()),
                                         fp(sv[3]), fp(sv[4]), fp(sv[5]), fp(saved), gr.data_ptr(), gb.data_ptr(),
                                         gw.data_ptr(), fp(ghp), fp(ghq), fp(ghr), ws.data_ptr(), wsb, T, (int32_t)n,
                                         (int32_t)C, (int32_t)cfg[2], (float)cfg[3], (float)cfg[4], stream()),
              "mhc_wrapper_static_bwd");
        const auto dts = ctx->saved_data["dtypes"].toIntVector();
        return {gr.to((at::ScalarType)dts[0]), gb.to((at::ScalarType)dts[1]), gw, ghp, ghq, ghr, Tensor(), Tensor(),
                Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

struct DynamicWrapper : public torch::autograd::Function<DynamicWrapper> {
    static Tensor forward(AutogradContext* ctx, const Tensor& res_in, const Tensor& br_in, const Tensor& w_in,
                          const Tensor& pp_in, const Tensor& pq_in, const Tensor& pr_in, const Tensor& ap_in,
                          const Tensor& aq_in, const Tensor& ar_in, const Tensor& bp_in, const Tensor& bq_in,
                          const Tensor& bres_in, int64_t mode, int64_t n, int64_t iters, double sk_eps,
                          double rms_eps, int64_t fmt) {
        const char* fn = "wrapper_dynamic_fwd";
        auto [r, b] = wrapper_inputs(fn, res_in, br_in);
        check_device(fn, {&r, &w_in, &pp_in, &pq_in, &pr_in, &bp_in, &bq_in, &bres_in});
        const at::DeviceGuard guard(r.device());
        const int64_t T = r.size(0), C = r.size(1);
        const Tensor w = weight(w_in);
        TORCH_CHECK(w.numel() == C, "wrapper_dynamic_fwd: rmsnorm_weight must have C elements");
        const auto ph = phi_parts(pp_in, pq_in, pr_in, n, n * C);
        const Tensor ap = scalar_param(ap_in, r.device()), aq = scalar_param(aq_in, r.device()),
                     ar = scalar_param(ar_in, r.device());
        const Tensor bp = f32c(bp_in), bq = f32c(bq_in), bres = f32c(bres_in);
        const auto f32 = r.options().dtype(at::kFloat);
        Tensor out = at::empty({T, C}, f32);
        Tensor saved =
            at::empty({(int64_t)(lib.mhc_wrapper_dynamic_saved_size(T, (int32_t)n, (int32_t)C) / 4)}, f32);
        const size_t wsb = lib.mhc_wrapper_dynamic_fwd_workspace_need(
            r.data_ptr(), b.data_ptr(), dtype_code(r.scalar_type()), T, (int32_t)n, (int32_t)C);
        Tensor ws = workspace(wsb, r);
        check(lib.mhc_wrapper_dynamic_fwd(r.data_ptr(), b.data_ptr(), dtype_code(r.scalar_type()), (int32_t)mode,
                                          w.data_ptr(), dtype_code(w.scalar_type()), fp(ph[0]), fp(ph[1]), fp(ph[2]),
                                          fp(ap), fp(aq), fp(ar), fp(bp), fp(bq), fp(bres), fp(out), fp(saved),
                                          ws.data_ptr(), wsb, T, (int32_t)n, (int32_t)C, (int32_t)iters,
                                          (float)sk_eps, (float)rms_eps, stream()),
              "mhc_wrapper_dynamic_fwd");
        save_wrapper_rows(ctx, fmt, r, b, {w, saved, ph[0], ph[1], ph[2], ap, aq, ar, bres});
        // b_pre and b_post are not read by the backward: their shapes only
        ctx->saved_data["b_pre"] = bp.sizes().vec();
        ctx->saved_data["b_post"] = bq.sizes().vec();
        ctx->saved_data["dtypes"] = std::vector<int64_t>{(int64_t)res_in.scalar_type(), (int64_t)br_in.scalar_type()};
        ctx->saved_data["cfg"] = std::vector<double>{(double)mode, (double)n, (double)iters, sk_eps, rms_eps};
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "wrapper_dynamic_bwd";
        const auto sv = ctx->get_saved_variables();
        check_device(fn, {&grads[0], &sv[0]});
        const at::DeviceGuard guard(sv[0].device());
        const auto [r, b] = wrapper_rows(ctx, sv);
        const Tensor &w = sv[2], &saved = sv[3];
        const auto cfg = ctx->saved_data["cfg"].toDoubleVector();
        const int64_t T = r.size(0), C = r.size(1), n = (int64_t)cfg[1], np = 2 * n + n * n;
        const int32_t mode = (int32_t)cfg[0];
        TORCH_CHECK(grads[0].sizes() == r.sizes(), "wrapper_dynamic_bwd: grad_out must be [tokens, hidden]");
        const Tensor g = f32c(grads[0]);
        const auto f32 = r.options().dtype(at::kFloat);
        Tensor gr = at::empty_like(r), gb = at::empty_like(b);
        Tensor gw = at::empty({C}, w.options());
        Tensor gphi = at::empty({np, n * C}, f32);
        Tensor galpha = at::empty({3}, f32);
        Tensor gbias = at::empty({np}, f32);
        const int dt = dtype_code(r.scalar_type());
        const size_t wsb = lib.mhc_wrapper_dynamic_bwd_workspace_need(
            fp(g), r.data_ptr(), b.data_ptr(), gr.data_ptr(), gb.data_ptr(), dt, mode, T, (int32_t)n, (int32_t)C,
            (int32_t)cfg[2], (float)cfg[3]);
        Tensor ws = workspace(wsb, r);
        check(lib.mhc_wrapper_dynamic_bwd(fp(g), r.data_ptr(), b.data_ptr(), dt, mode, dtype_code(w.scalar_type()),
                                          fp(sv[4]), fp(sv[5]), fp(sv[6]), fp(sv[7]), fp(sv[8]), fp(sv[9]),
                                          fp(sv[10]), fp(saved), gr.data_ptr(), gb.data_ptr(), gw.data_ptr(),
                                          fp(gphi), fp(galpha), fp(gbias), ws.data_ptr(), wsb, T, (int32_t)n,
                                          (int32_t)C, (int32_t)cfg[2], (float)cfg[3], (float)cfg[4], stream()),
              "mhc_wrapper_dynamic_bwd");
        const auto dts = ctx->saved_data["dtypes"].toIntVector();
        tensor_list out;
        out.reserve(18);
        out.push_back(gr.to((at::ScalarType)dts[0]));
        out.push_back(gb.to((at::ScalarType)dts[1]));
        out.push_back(gw);
        const auto bp = ctx->saved_data["b_pre"].toIntVector(), bq = ctx->saved_data["b_post"].toIntVector();
        push_param_grads(out,
                         {sv[4].sizes(), sv[5].sizes(), sv[6].sizes(), sv[7].sizes(), sv[8].sizes(), sv[9].sizes(), bp,
                          bq, sv[10].sizes()},
                         n, gphi, galpha, gbias);
        out.resize(18);
        return out;
    }
};

// ---- forward-only dynamic layer (ops.py:337-380) ------------------------------
Tensor dynamic_infer(const Tensor& x_in, const Tensor& packed, const Tensor& ap_in, const Tensor& aq_in,
                     const Tensor& ar_in, const Tensor& bp_in, const Tensor& bq_in, const Tensor& br_in, int64_t iters,
                     double sk_eps, double rms_eps, bool out_bf16) {
    require_bound();
    const char* fn = "mhc_layer_dynamic_infer";
    const at::NoGradGuard no_grad;
    check_device(fn, {&x_in, &packed, &bp_in, &bq_in, &br_in});
    const at::DeviceGuard guard(x_in.device());
    const Tensor x = layer_x(fn, x_in);
    const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
    TORCH_CHECK(packed.scalar_type() == at::kByte &&
                    (size_t)packed.numel() >= lib.mhc_layer_dynamic_packed_size((int32_t)n, (int32_t)C),
                fn, ": packed parameters do not match x [B, n, C]");
    const Tensor ap = scalar_param(ap_in, x.device()), aq = scalar_param(aq_in, x.device()),
                 ar = scalar_param(ar_in, x.device());
    const Tensor bp = f32c(bp_in), bq = f32c(bq_in), br = f32c(br_in);
    TORCH_CHECK(bp.numel() == n && bq.numel() == n && br.numel() == n * n, fn,
                ": b_pre/b_post must have n and b_res n*n elements");
    Tensor out = at::empty({B, n, C}, x.options().dtype(out_bf16 ? at::kBFloat16 : at::kFloat));
    const size_t wsb = lib.mhc_layer_dynamic_infer_workspace_size(B, (int32_t)n, (int32_t)C);
    Tensor ws = workspace(wsb, x);
    check(lib.mhc_layer_dynamic_infer(x.data_ptr(), dtype_code(x.scalar_type()), packed.data_ptr(), fp(ap), fp(aq),
                                      fp(ar), fp(bp), fp(bq), fp(br), out.data_ptr(),
                                      out_bf16 ? MHC_DTYPE_BF16 : MHC_DTYPE_F32, ws.data_ptr(), wsb, B, (int32_t)n,
                                      (int32_t)C, (int32_t)iters, (float)sk_eps, (float)rms_eps, stream()),
          fn);
    return out;
}

// ---- standalone operators (ops.py:32-265) -------------------------------------
// The same checks, dtypes and error text as the functions of
// mhc_ascend_amd/native.py; the tensors saved are the caller's own.
Tensor storage(const Tensor& t) { return (storage_dtype(t.scalar_type()) ? t : t.to(at::kFloat)).contiguous(); }

// A per-token coefficient tensor as (fp32 tensor, batch stride): one that is
// broadcast over the batch (stride 0) is passed once.
std::pair<Tensor, int64_t> coef_view(const char* fn, const Tensor& t_in, int64_t B, int64_t per) {
    const Tensor t = t_in.to(at::kFloat);
    if (t.dim() >= 2 && t.size(0) == B && t.stride(0) == 0) {
        const Tensor one = t.select(0, 0).contiguous();
        TORCH_CHECK(one.numel() == per, fn, ": coefficient shape ", t.sizes(), " does not match n");
        return {one, 0};
    }
    const Tensor c = t.contiguous();
    TORCH_CHECK(c.numel() == B * per, fn, ": coefficient shape ", t.sizes(), " does not match [B=", B, ", ", per, "]");
    return {c, per};
}

struct Sinkhorn : public torch::autograd::Function<Sinkhorn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& inp, int64_t iters, double eps) {
        check_device("sinkhorn_knopp_fwd", {&inp});
        const at::DeviceGuard guard(inp.device());
        TORCH_CHECK(inp.dim() == 3, "Input must be 3D tensor [B, M, N]");
        TORCH_CHECK(inp.size(1) == inp.size(2), "Sinkhorn-Knopp requires square matrices (M == N), got M=",
                    inp.size(1), ", N=", inp.size(2));
        TORCH_CHECK(inp.scalar_type() == at::kFloat, "inp must be float32");
        const Tensor a = inp.contiguous();
        Tensor out = at::empty_like(a);
        check(lib.mhc_sinkhorn_knopp_fwd(fp(a), fp(out), a.size(0), (int32_t)a.size(1), (int32_t)iters, (float)eps,
                                         stream()),
              "mhc_sinkhorn_knopp_fwd");
        ctx->save_for_backward({inp, out});
        ctx->saved_data["iters"] = iters;
        ctx->saved_data["eps"] = eps;
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto sv = ctx->get_saved_variables();
        const Tensor g = f32c(grads[0]);
        check_device("sinkhorn_knopp_bwd", {&g, &sv[0]});
        const at::DeviceGuard guard(g.device());
        TORCH_CHECK(g.sizes() == sv[0].sizes(), "grad_out shape must match inp");
        const Tensor a = sv[0].contiguous();
        Tensor gi = at::empty_like(a);
        check(lib.mhc_sinkhorn_knopp_bwd(fp(g), fp(a), nullptr, fp(gi), a.size(0), (int32_t)a.size(1),
                                         (int32_t)ctx->saved_data["iters"].toInt(),
                                         (float)ctx->saved_data["eps"].toDouble(), stream()),
              "mhc_sinkhorn_knopp_bwd");
        return {gi, Tensor(), Tensor()};
    }
};

struct RmsNorm : public torch::autograd::Function<RmsNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& inp, const Tensor& w_in, double eps) {
        check_device("rmsnorm_fwd", {&inp, &w_in});
        const at::DeviceGuard guard(inp.device());
        TORCH_CHECK(inp.dim() == 2, "Input must be 2D tensor [B, C]");
        const Tensor x = storage(inp);
        const int64_t B = x.size(0), C = x.size(1);
        TORCH_CHECK(w_in.numel() == C, "weight must have C elements");
        const Tensor w = f32c(w_in);
        Tensor out = at::empty_like(x);
        Tensor rms = at::empty({B}, x.options().dtype(at::kFloat));
        check(lib.mhc_rmsnorm_fwd(x.data_ptr(), dtype_code(x.scalar_type()), fp(w), out.data_ptr(), fp(rms), B,
                                  (int32_t)C, (float)eps, stream()),
              "mhc_rmsnorm_fwd");
        ctx->save_for_backward({inp, w_in, rms});
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto sv = ctx->get_saved_variables();
        const Tensor &inp = sv[0], &w_in = sv[1], &rms = sv[2];
        check_device("rmsnorm_bwd", {&grads[0], &inp, &w_in, &rms});
        const at::DeviceGuard guard(inp.device());
        const Tensor x = storage(inp);
        const int64_t B = x.size(0), C = x.size(1);
        const Tensor g = grads[0].to(x.scalar_type()).contiguous();
        TORCH_CHECK(g.sizes() == x.sizes(), "grad_out shape must match inp");
        const Tensor w = f32c(w_in);
        Tensor gx = at::empty_like(x);
        Tensor gw = at::empty({C}, x.options().dtype(at::kFloat));
        const int dt = dtype_code(x.scalar_type());
        const size_t wsb = lib.mhc_rmsnorm_bwd_workspace_size(B, (int32_t)C, dt);
        Tensor ws = workspace(wsb, x);
        check(lib.mhc_rmsnorm_bwd(g.data_ptr(), x.data_ptr(), dt, fp(w), fp(rms), gx.data_ptr(), fp(gw), ws.data_ptr(),
                                  wsb, B, (int32_t)C, stream()),
              "mhc_rmsnorm_bwd");
        return {gx.to(inp.scalar_type()), gw, Tensor()};
    }
};

// RMSNorm whose backward reads an 8-bit checkpoint of its input's rows.
struct RmsNormHeld : public torch::autograd::Function<RmsNormHeld> {
    static Tensor forward(AutogradContext* ctx, const Tensor& inp, const Tensor& w_in, double eps, int64_t fmt) {
        check_device("rmsnorm_fwd", {&inp, &w_in});
        const at::DeviceGuard guard(inp.device());
        TORCH_CHECK(inp.dim() == 2, "Input must be 2D tensor [B, C]");
        const Tensor x = storage(inp);
        const int64_t B = x.size(0), C = x.size(1);
        TORCH_CHECK(w_in.numel() == C, "weight must have C elements");
        const Tensor w = f32c(w_in);
        Tensor out = at::empty_like(x);
        const Held held = held_alloc(x);
        check(lib.mhc_rmsnorm_checkpoint_fwd(x.data_ptr(), dtype_code(x.scalar_type()), fp(w), out.data_ptr(),
                                             (int32_t)fmt, held.values.data_ptr(), held.scales.data_ptr(), B,
                                             (int32_t)C, (float)eps, stream()),
              "mhc_rmsnorm_checkpoint_fwd");
        ctx->save_for_backward({held.values, held.scales, w_in});
        ctx->saved_data["x_dtype"] = (int64_t)inp.scalar_type();
        ctx->saved_data["store"] = (int64_t)x.scalar_type();
        ctx->saved_data["B"] = B;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["fmt"] = fmt;
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto sv = ctx->get_saved_variables();
        const Tensor &values = sv[0], &scales = sv[1], &w_in = sv[2];
        check_device("rmsnorm_bwd", {&grads[0], &values, &w_in});
        const at::DeviceGuard guard(values.device());
        const auto store = (at::ScalarType)ctx->saved_data["store"].toInt();
        const int64_t B = ctx->saved_data["B"].toInt(), C = w_in.numel(), fmt = ctx->saved_data["fmt"].toInt();
        const Tensor g = grads[0].to(store).contiguous();
        TORCH_CHECK(g.dim() == 2 && g.size(0) == B && g.size(1) == C, "grad_out shape must match inp");
        const Tensor w = f32c(w_in);
        Tensor gx = at::empty({B, C}, g.options());
        Tensor gw = at::empty({C}, g.options().dtype(at::kFloat));
        const int dt = dtype_code(store);
        const size_t wsb = lib.mhc_rmsnorm_checkpoint_bwd_workspace_size(B, (int32_t)C, dt, (int32_t)fmt);
        Tensor ws = workspace(wsb, g);
        check(lib.mhc_rmsnorm_checkpoint_bwd(g.data_ptr(), dt, values.data_ptr(), scales.data_ptr(), (int32_t)fmt,
                                             fp(w), gx.data_ptr(), fp(gw), ws.data_ptr(), wsb, B, (int32_t)C,
                                             (float)ctx->saved_data["eps"].toDouble(), stream()),
              "mhc_rmsnorm_checkpoint_bwd");
        return {gx.to((at::ScalarType)ctx->saved_data["x_dtype"].toInt()), gw, Tensor(), Tensor()};
    }
};

struct Aggregate : public torch::autograd::Function<Aggregate> {
    static Tensor forward(AutogradContext* ctx, const Tensor& inp, const Tensor& h_in, int64_t fmt) {
        const char* fn = "stream_aggregate_fwd";
        check_device(fn, {&inp, &h_in});
        const at::DeviceGuard guard(inp.device());
        TORCH_CHECK(inp.dim() == 3, "Input must be 3D tensor [B, n, C]");
        const Tensor x = storage(inp);
        const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
        const auto [h, hs] = coef_view(fn, h_in, B, n);
        Tensor out = at::empty({B, C}, x.options());
        Tensor act = at::empty({B, n}, x.options().dtype(at::kFloat));
        check(lib.mhc_stream_aggregate_fwd(x.data_ptr(), dtype_code(x.scalar_type()), fp(h), hs, out.data_ptr(),
                                           fp(act), B, (int32_t)n, (int32_t)C, stream()),
              "mhc_stream_aggregate_fwd");
        if (fmt != MHC_CHECKPOINT_NONE) {
            ctx->saved_data["fmt"] = fmt;
            const Held held = hold(x, fmt);
            ctx->saved_data["sizes"] = x.sizes().vec();
            ctx->saved_data["store"] = (int64_t)x.scalar_type();
            ctx->saved_data["x_dtype"] = (int64_t)inp.scalar_type();
            ctx->save_for_backward({held.values, act, held.scales});
            return out;
        }
        ctx->save_for_backward({inp, act});
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto sv = ctx->get_saved_variables();
        const Tensor &inp = sv[0], &act = sv[1];
        check_device("stream_aggregate_bwd", {&grads[0], &inp, &act});
        const at::DeviceGuard guard(inp.device());
        const int64_t fmt = saved_format(ctx);
        const bool is_held = fmt != MHC_CHECKPOINT_NONE;
        const Tensor x = is_held ? held_rows(inp, sv[2], fmt, ctx->saved_data["sizes"].toIntVector(),
                                             (at::ScalarType)ctx->saved_data["store"].toInt())
                                 : storage(inp);
        const auto x_dtype = is_held ? (at::ScalarType)ctx->saved_data["x_dtype"].toInt() : inp.scalar_type();
        const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
        const Tensor g = grads[0].to(x.scalar_type()).contiguous();
        TORCH_CHECK(g.dim() == 2 && g.size(0) == B && g.size(1) == C, "grad_out must be [B, C]");
        Tensor gx = at::empty_like(x);
        Tensor graw = at::empty({B, n}, act.options());
        check(lib.mhc_stream_aggregate_bwd(g.data_ptr(), x.data_ptr(), dtype_code(x.scalar_type()), fp(act), n,
                                           gx.data_ptr(), nullptr, fp(graw), B, (int32_t)n, (int32_t)C, stream()),
              "mhc_stream_aggregate_bwd");
        return {gx.to(x_dtype), graw, Tensor()};
    }
};

struct Distribute : public torch::autograd::Function<Distribute> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y_in, const Tensor& h_in, const Tensor& m_in,
                          const Tensor& x_in, int64_t fmt) {
        const char* fn = "stream_distribute_mix_add_fwd";
        check_device(fn, {&y_in, &h_in, &m_in, &x_in});
        const at::DeviceGuard guard(x_in.device());
        TORCH_CHECK(x_in.dim() == 3, "x_inp must be 3D tensor [B, n, C]");
        const Tensor x = storage(x_in);
        const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
        const Tensor y = y_in.to(x.scalar_type()).contiguous();
        TORCH_CHECK(y.dim() == 2 && y.size(0) == B && y.size(1) == C, "y_norm must be [B, C]");
        const auto [h, hs] = coef_view(fn, h_in, B, n);
        const auto [m, ms] = coef_view(fn, m_in, B, n * n);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor out = at::empty({B, n, C}, f32);
        Tensor act = at::empty({B, n}, f32);
        check(lib.mhc_stream_distribute_mix_add_fwd(y.data_ptr(), fp(h), hs, fp(m), ms, x.data_ptr(),
                                                    dtype_code(x.scalar_type()), fp(out), fp(act), B, (int32_t)n,
                                                    (int32_t)C, stream()),
              "mhc_stream_distribute_mix_add_fwd");
        if (fmt != MHC_CHECKPOINT_NONE) {
            ctx->saved_data["fmt"] = fmt;
            const Held hx = hold(x, fmt), hy = hold(y, fmt);
            ctx->saved_data["sizes"] = x.sizes().vec();
            ctx->saved_data["store"] = (int64_t)x.scalar_type();
            ctx->saved_data["dtypes"] = std::vector<int64_t>{(int64_t)x_in.scalar_type(), (int64_t)y_in.scalar_type()};
            ctx->save_for_backward({hx.values, hy.values, m_in, act, hx.scales, hy.scales});
            return out;
        }
        ctx->save_for_backward({x_in, y_in, m_in, act});
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "stream_distribute_mix_add_bwd";
        const auto sv = ctx->get_saved_variables();
        const Tensor &x_in = sv[0], &y_in = sv[1], &m_in = sv[2], &act = sv[3];
        check_device(fn, {&grads[0], &x_in, &y_in, &m_in, &act});
        const at::DeviceGuard guard(x_in.device());
        const int64_t fmt = saved_format(ctx);
        Tensor x, y;
        at::ScalarType x_dtype = x_in.scalar_type(), y_dtype = y_in.scalar_type();
        if (fmt != MHC_CHECKPOINT_NONE) {
            const auto sizes = ctx->saved_data["sizes"].toIntVector();
            const auto store = (at::ScalarType)ctx->saved_data["store"].toInt();
            const auto dts = ctx->saved_data["dtypes"].toIntVector();
            x = held_rows(x_in, sv[4], fmt, sizes, store);
            y = held_rows(y_in, sv[5], fmt, {sizes[0], sizes[2]}, store);
            x_dtype = (at::ScalarType)dts[0];
            y_dtype = (at::ScalarType)dts[1];
        } else {
            x = storage(x_in);
            y = y_in.to(x.scalar_type()).contiguous();
        }
        const int64_t B = x.size(0), n = x.size(1), C = x.size(2);
        const Tensor g = f32c(grads[0]);
        TORCH_CHECK(g.sizes() == x.sizes(), "grad_out shape must match x_inp");
        const auto [m, ms] = coef_view(fn, m_in, B, n * n);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor gx = at::empty_like(x), gy = at::empty({B, C}, x.options());
        Tensor gm = at::empty({B, n, n}, f32), graw = at::empty({B, n}, f32);
        check(lib.mhc_stream_distribute_mix_add_bwd(fp(g), x.data_ptr(), y.data_ptr(), dtype_code(x.scalar_type()),
                                                    fp(m), ms, fp(act), n, gx.data_ptr(), gy.data_ptr(), fp(gm),
                                                    nullptr, fp(graw), B, (int32_t)n, (int32_t)C, stream()),
              "mhc_stream_distribute_mix_add_bwd");
        return {gy.to(y_dtype), graw, gm, gx.to(x_dtype), Tensor()};
    }
};

// Whether a call of a C++ node is needed: a backward may run, or an input has a
// forward-mode tangent (forward mode runs without grad mode too), which a C++
// node refuses.
bool needs_node(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->_fw_grad(0).defined() || (at::GradMode::is_enabled() && t->requires_grad())) return true;
    return false;
}

// ---- dropout, RMSNorm of a residual's sum ---------------------------------------
// What a call drops: the numbers of `seed` (a tensor where one is defined).
struct Drop {
    int64_t threshold, value, offset;
    Tensor seed;

    const void* ptr() const { return seed.defined() ? seed.data_ptr() : nullptr; }
    std::vector<int64_t> ints() const { return {threshold, value, offset}; }
    static Drop saved(const std::vector<int64_t>& v, const Tensor& seed) { return {v[0], v[1], v[2], seed}; }
};

// A seed that is not given is drawn from x's device's generator.
Drop make_drop(const char* fn, const Tensor& x, double p, const c10::optional<Tensor>& seed,
               const c10::optional<int64_t>& value, int64_t offset) {
    TORCH_CHECK(p >= 0.0 && p <= 1.0, fn, ": the probability must be in 0 .. 1, got ", p);
    TORCH_CHECK(offset >= 0, fn, ": offset must be >= 0, got ", offset);
    Drop d{(int64_t)std::nearbyint(p * 65536), value.value_or(0), offset, Tensor()};
    if (seed.has_value()) {
        check_device(fn, {&x, &*seed});
        TORCH_CHECK(seed->scalar_type() == at::kLong && seed->numel() == 1, fn, ": seed must be one int64, got ",
                    seed->scalar_type(), " ", seed->sizes());
        d.seed = *seed;
    } else if (!value.has_value() && d.threshold > 0) {
        const at::DeviceGuard guard(x.device());
        d.seed = at::empty({1}, x.options().dtype(at::kLong).requires_grad(false)).random_();
    }
    if (d.threshold == 0) d.seed = Tensor();
    return d;
}

// Rows [B, C] of a contiguous tensor [..., C].
int64_t rows_of(const Tensor& t) { return t.size(-1) > 0 ? t.numel() / t.size(-1) : 0; }

void check_rows(const char* fn, const Tensor& x) {
    TORCH_CHECK(x.dim() >= 1 && at::isFloatingType(x.scalar_type()), fn,
                ": x must be a floating-point tensor [..., C]");
    TORCH_CHECK(x.size(-1) >= 1 && x.size(-1) <= INT32_MAX, fn, ": rows of ", x.size(-1), " channels");
}

Tensor run_dropout(const Tensor& x, const Drop& d) {
    Tensor out = at::empty_like(x);
    check(lib.mhc_dropout(x.data_ptr(), dtype_code(x.scalar_type()), out.data_ptr(), (int32_t)d.threshold,
                          (uint64_t)d.value, d.ptr(), (uint64_t)d.offset, rows_of(x), (int32_t)x.size(-1), stream()),
          "mhc_dropout");
    return out;
}

struct Dropout : public torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Drop& d) {
        const at::DeviceGuard guard(x_in.device());
        const Tensor x = storage(x_in);
        if (ctx) {
            ctx->save_for_backward({d.seed});
            ctx->saved_data["drop"] = d.ints();
            ctx->saved_data["x_dtype"] = (int64_t)x_in.scalar_type();
        }
        return run_dropout(x, d);
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const Drop d = Drop::saved(ctx->saved_data["drop"].toIntVector(), ctx->get_saved_variables()[0]);
        const auto dt = (at::ScalarType)ctx->saved_data["x_dtype"].toInt();
        // linear: its gradient's gradient is a call on the cotangent
        const Tensor dx = needs_node({&grads[0]}) ? Dropout::apply(grads[0], d) : forward(nullptr, grads[0], d);
        return {dx.to(dt), Tensor()};
    }
};

struct RmsNormResidual : public torch::autograd::Function<RmsNormResidual> {
    // (y, h); with y_fmt (values, scales, h)
    static tensor_list forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& res_in, const Tensor& w_in,
                               double eps, const Drop& d, int64_t fmt, int64_t y_fmt) {
        const char* fn = "mhc_rmsnorm_residual_fwd";
        const at::DeviceGuard guard(x_in.device());
        const Tensor x = storage(x_in), res = storage(res_in), w = weight(w_in);
        const int64_t C = x.size(-1), B = rows_of(x);
        Tensor h = at::empty_like(res), y;
        Held hy, hh;
        if (y_fmt != MHC_CHECKPOINT_NONE) hy = packed_alloc(x);
        else y = at::empty_like(x);
        if (fmt != MHC_CHECKPOINT_NONE) hh = held_alloc(res);
        const auto at_ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
        check(lib.mhc_rmsnorm_residual_fwd(
                  x.data_ptr(), dtype_code(x.scalar_type()), res.data_ptr(), dtype_code(res.scalar_type()),
                  w.data_ptr(), dtype_code(w.scalar_type()), h.data_ptr(), at_ptr(y), (int32_t)y_fmt,
                  at_ptr(hy.values), at_ptr(hy.scales), (int32_t)fmt, at_ptr(hh.values), at_ptr(hh.scales),
                  (int32_t)d.threshold, (uint64_t)d.value, d.ptr(), (uint64_t)d.offset, B, (int32_t)C, (float)eps,
                  stream()),
              fn);
        if (y_fmt != MHC_CHECKPOINT_NONE) return {hy.values, hy.scales, h};
        if (!ctx) return {y, h};  // no backward will run
        ctx->set_materialize_grads(false);
        if (fmt != MHC_CHECKPOINT_NONE) ctx->save_for_backward({w, d.seed, hh.values, hh.scales});
        else ctx->save_for_backward({w, d.seed, h});
        ctx->saved_data["drop"] = d.ints();
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["sizes"] = x.sizes().vec();
        ctx->saved_data["ints"] = std::vector<int64_t>{fmt, (int64_t)x.scalar_type(), (int64_t)res.scalar_type(),
                                                       (int64_t)x_in.scalar_type(), (int64_t)res_in.scalar_type(),
                                                       (int64_t)w_in.scalar_type()};
        return {y, h};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "mhc_rmsnorm_residual_bwd";
        TORCH_CHECK(!at::GradMode::is_enabled(), "rmsnorm_residual: no second derivative (create_graph)");
        tensor_list out(7);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const auto sv = ctx->get_saved_variables();
        const auto v = ctx->saved_data["ints"].toIntVector();
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const Drop d = Drop::saved(ctx->saved_data["drop"].toIntVector(), sv[1]);
        const Tensor& w = sv[0];
        const int64_t fmt = v[0], C = sizes.back();
        const bool is_held = fmt != MHC_CHECKPOINT_NONE;
        const auto xt = (at::ScalarType)v[1], rt = (at::ScalarType)v[2];
        const at::DeviceGuard guard(w.device());
        const auto opt = w.options();
        const Tensor gy = grads[0].defined() ? grads[0].to(xt).contiguous() : at::zeros(sizes, opt.dtype(xt));
        const Tensor gh = grads[1].defined() ? grads[1].to(rt).contiguous() : Tensor();
        TORCH_CHECK(gy.sizes() == sizes && (!gh.defined() || gh.sizes() == sizes), fn,
                    ": the cotangents must match the outputs");
        const bool want_x = ctx->needs_input_grad(0), want_res = ctx->needs_input_grad(1),
                   want_w = ctx->needs_input_grad(2);
        // without dropout and in one type both are the same array
        const bool one = d.threshold == 0 && xt == rt;
        Tensor gres, gx, gw, ws;
        if (want_res || (one && want_x)) gres = at::empty(sizes, opt.dtype(rt));
        if (want_x) gx = one ? gres : at::empty(sizes, opt.dtype(xt));
        const int64_t B = rows_of(gy);
        size_t wsb = 0;
        if (want_w) {
            gw = at::empty({C}, opt);
            wsb = lib.mhc_rmsnorm_residual_bwd_workspace_size(B, (int32_t)C, dtype_code(xt), dtype_code(rt));
            ws = workspace(wsb, w);
        }
        const auto at_ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
        check(lib.mhc_rmsnorm_residual_bwd(
                  gy.data_ptr(), dtype_code(xt), at_ptr(gh), dtype_code(rt), is_held ? nullptr : sv[2].data_ptr(),
                  (int32_t)fmt, is_held ? sv[2].data_ptr() : nullptr, is_held ? sv[3].data_ptr() : nullptr,
                  w.data_ptr(), dtype_code(w.scalar_type()), one ? nullptr : at_ptr(gx), at_ptr(gres), at_ptr(gw),
                  (int32_t)d.threshold, (uint64_t)d.value, d.ptr(), (uint64_t)d.offset, at_ptr(ws), wsb, B, (int32_t)C,
                  (float)ctx->saved_data["eps"].toDouble(), stream()),
              fn);
        if (want_x) out[0] = gx.to((at::ScalarType)v[3]);
        if (want_res) out[1] = gres.to((at::ScalarType)v[4]);
        if (want_w) out[2] = gw.to((at::ScalarType)v[5]);
        return out;
    }
};

// ---- per-head norm of queries and keys, with the rotation of positions ----------
// What the entries take besides rows: weights in one dtype, fp32 tables.
struct QkTables {
    Tensor wq, wk, cos, sin, pos;
    int64_t period;

    QkTables(const Tensor& wq_in, const Tensor& wk_in, const Tensor& cos_in, const Tensor& sin_in,
             const Tensor& pos_in, int64_t period_in)
        : cos(f32c(cos_in)), sin(f32c(sin_in)), pos(pos_in), period(period_in) {
        const bool one = wq_in.scalar_type() == wk_in.scalar_type() && storage_dtype(wq_in.scalar_type());
        wq = one ? wq_in.contiguous() : f32c(wq_in);
        wk = one ? wk_in.contiguous() : f32c(wk_in);
    }
    int w_dtype() const { return dtype_code(wq.scalar_type()); }
    const void* pos_ptr() const { return pos.defined() ? pos.data_ptr() : nullptr; }
    int32_t pos_bytes() const { return pos.defined() ? (int32_t)pos.element_size() : 0; }
};

// The axes of a call's positions: none named, or the pairs of each.
struct QkAxes {
    std::vector<int64_t> sections;
    bool dealt = false;
    int32_t host[4] = {0, 0, 0, 0};

    QkAxes(const std::vector<int64_t>& sections_, bool dealt_) : sections(sections_), dealt(dealt_) {
        for (size_t i = 0; i < sections.size() && i < 4; ++i) host[i] = (int32_t)sections[i];
    }
    bool any() const { return !sections.empty(); }
    int32_t count() const { return (int32_t)sections.size(); }
    const int32_t* ptr() const { return any() ? host : nullptr; }
};

// Rows as the kernels read them: storage dtype, channels next to each other.
Tensor qk_rows(const Tensor& t, at::ScalarType dt) {
    const Tensor s = t.to(dt);
    return s.stride(2) == 1 || s.size(2) == 1 ? s : s.contiguous();
}

QkAxes saved_axes(AutogradContext* ctx) {
    const auto it = ctx->saved_data.find("sections");
    if (it == ctx->saved_data.end()) return QkAxes({}, false);
    return QkAxes(it->second.toIntVector(), ctx->saved_data["dealt"].toBool());
}

struct QkNormRope : public torch::autograd::Function<QkNormRope> {
    static tensor_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& wq_in,
                               const Tensor& wk_in, const Tensor& cos, const Tensor& sin,
                               const c10::optional<Tensor>& positions, int64_t period, double eps, bool interleaved,
                               int64_t fmt, const QkAxes& axes) {
        const char* fn = "qk_norm_rope_fwd";
        const at::DeviceGuard guard(q_in.device());
        const auto dt = storage_dtype(q_in.scalar_type()) ? q_in.scalar_type() : at::kFloat;
        const Tensor q = qk_rows(q_in, dt), k = qk_rows(k_in, dt);
        const QkTables t(wq_in, wk_in, cos, sin, positions.has_value() ? positions->contiguous() : Tensor(), period);
        const int64_t T = q.size(0), H = q.size(1), K = k.size(1), D = q.size(2);
        Tensor qo = at::empty({T, H, D}, q.options()), ko = at::empty({T, K, D}, k.options());
        Held hq, hk;
        if (fmt != MHC_CHECKPOINT_NONE) {
            hq = held_alloc(q);
            hk = held_alloc(k);
        }
        const auto held = [&](const Tensor& h) { return h.defined() ? h.data_ptr() : nullptr; };
        const auto run = [&](auto entry, auto... more) {
            return entry(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                         dtype_code(dt), t.wq.data_ptr(), t.wk.data_ptr(), t.w_dtype(), fp(t.cos), fp(t.sin),
                         t.cos.size(0), t.pos_ptr(), t.pos_bytes(), t.period, more..., qo.data_ptr(), ko.data_ptr(),
                         (int32_t)fmt, held(hq.values), held(hq.scales), held(hk.values), held(hk.scales), T,
                         (int32_t)H, (int32_t)K, (int32_t)D, (int32_t)(2 * t.cos.size(1)), interleaved, (float)eps,
                         stream());
        };
        check(axes.any() ? run(lib.mhc_qk_norm_rope_axes_fwd, axes.count(), axes.ptr(), (int32_t)axes.dealt)
                         : run(lib.mhc_qk_norm_rope_fwd),
              fn);
        if (!ctx) return {qo, ko};  // no backward will run
        tensor_list sv = {t.wq, t.wk, t.cos, t.sin};
        if (fmt != MHC_CHECKPOINT_NONE) {
            sv.insert(sv.end(), {hq.values, hk.values, hq.scales, hk.scales});
        } else {
            sv.insert(sv.end(), {q, k});
        }
        if (t.pos.defined()) sv.push_back(t.pos);
        ctx->save_for_backward(std::move(sv));
        ctx->saved_data["ints"] = std::vector<int64_t>{T, H, K, D, t.period, interleaved, fmt, t.pos.defined(),
                                                       (int64_t)dt, (int64_t)q_in.scalar_type(),
                                                       (int64_t)k_in.scalar_type(), (int64_t)wq_in.scalar_type(),
                                                       (int64_t)wk_in.scalar_type()};
        ctx->saved_data["eps"] = eps;
        if (axes.any()) {
            ctx->saved_data["sections"] = axes.sections;
            ctx->saved_data["dealt"] = axes.dealt;
        }
        return {qo, ko};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const char* fn = "qk_norm_rope_bwd";
        const auto sv = ctx->get_saved_variables();
        const auto v = ctx->saved_data["ints"].toIntVector();
        const int64_t T = v[0], H = v[1], K = v[2], D = v[3], fmt = v[6];
        const bool is_held = fmt != MHC_CHECKPOINT_NONE;
        const auto dt = (at::ScalarType)v[8];
        check_device(fn, {&grads[0], &grads[1], &sv[0]});
        const at::DeviceGuard guard(sv[0].device());
        const QkTables t(sv[0], sv[1], sv[2], sv[3], v[7] ? sv.back() : Tensor(), v[4]);
        const Tensor gq = qk_rows(grads[0], dt), gk = qk_rows(grads[1], dt);
        TORCH_CHECK(gq.sizes() == at::IntArrayRef({T, H, D}) && gk.sizes() == at::IntArrayRef({T, K, D}), fn,
                    ": the cotangents must match the outputs");
        Tensor dq = at::empty({T, H, D}, gq.options()), dk = at::empty({T, K, D}, gk.options());
        Tensor dw = at::empty({2, D}, t.wq.options());
        const size_t wsb = lib.mhc_qk_norm_rope_bwd_workspace_size(T, (int32_t)H, (int32_t)K, (int32_t)D,
                                                                   (int32_t)(2 * t.cos.size(1)), (int32_t)v[5]);
        Tensor ws = workspace(wsb, dq);
        const Tensor none;
        const Tensor &q = is_held ? none : sv[4], &k = is_held ? none : sv[5];
        const auto at_ptr = [](const Tensor& h) { return h.defined() ? h.data_ptr() : nullptr; };
        const auto st = [](const Tensor& h, int d) { return h.defined() ? h.stride(d) : (int64_t)0; };
        const QkAxes axes = saved_axes(ctx);
        const auto run = [&](auto entry, auto... more) {
            return entry(gq.data_ptr(), gq.stride(0), gq.stride(1), gk.data_ptr(), gk.stride(0), gk.stride(1),
                         at_ptr(q), st(q, 0), st(q, 1), at_ptr(k), st(k, 0), st(k, 1), dtype_code(dt), (int32_t)fmt,
                         is_held ? sv[4].data_ptr() : nullptr, is_held ? sv[6].data_ptr() : nullptr,
                         is_held ? sv[5].data_ptr() : nullptr, is_held ? sv[7].data_ptr() : nullptr, t.wq.data_ptr(),
                         t.wk.data_ptr(), t.w_dtype(), fp(t.cos), fp(t.sin), t.cos.size(0), t.pos_ptr(),
                         t.pos_bytes(), t.period, more..., dq.data_ptr(), dk.data_ptr(), dw.data_ptr(),
                         ws.data_ptr(), wsb, T, (int32_t)H, (int32_t)K, (int32_t)D, (int32_t)(2 * t.cos.size(1)),
                         (int32_t)v[5], (float)ctx->saved_data["eps"].toDouble(), stream());
        };
        check(axes.any() ? run(lib.mhc_qk_norm_rope_axes_bwd, axes.count(), axes.ptr(), (int32_t)axes.dealt)
                         : run(lib.mhc_qk_norm_rope_bwd),
              fn);
        tensor_list out = {dq.to((at::ScalarType)v[9]), dk.to((at::ScalarType)v[10]),
                           dw.select(0, 0).to((at::ScalarType)v[11]), dw.select(0, 1).to((at::ScalarType)v[12])};
        out.resize(12);
        return out;
    }
};

// The rotation alone: its backward is the rotation by the negative angle.
struct QkRope : public torch::autograd::Function<QkRope> {
    static tensor_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& cos_in,
                               const Tensor& sin_in, const c10::optional<Tensor>& positions, int64_t period,
                               bool interleaved, const QkAxes& axes, bool inverse) {
        const at::DeviceGuard guard(q_in.device());
        const auto dt = storage_dtype(q_in.scalar_type()) ? q_in.scalar_type() : at::kFloat;
        const Tensor q = qk_rows(q_in, dt), k = qk_rows(k_in, dt), cos = f32c(cos_in), sin = f32c(sin_in);
        const Tensor pos = positions.has_value() && positions->defined() ? positions->contiguous() : Tensor();
        if (ctx) {
            ctx->save_for_backward({cos, sin, pos});
            ctx->saved_data["ints"] =
                std::vector<int64_t>{period, interleaved, (int64_t)dt, (int64_t)q_in.scalar_type(),
                                     (int64_t)k_in.scalar_type(), inverse};
            if (axes.any()) {
                ctx->saved_data["sections"] = axes.sections;
                ctx->saved_data["dealt"] = axes.dealt;
            }
        }
        const int64_t T = q.size(0), H = q.size(1), K = k.size(1), D = q.size(2);
        Tensor qo = at::empty({T, H, D}, q.options()), ko = at::empty({T, K, D}, k.options());
        check(lib.mhc_qk_rope(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                              dtype_code(dt), fp(cos), fp(sin), cos.size(0), pos.defined() ? pos.data_ptr() : nullptr,
                              pos.defined() ? (int32_t)pos.element_size() : 0, period, axes.count(), axes.ptr(),
                              (int32_t)axes.dealt, qo.data_ptr(), ko.data_ptr(), T, (int32_t)H, (int32_t)K,
                              (int32_t)D, (int32_t)(2 * cos.size(1)), interleaved, inverse, stream()),
              "mhc_qk_rope");
        return {qo, ko};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto sv = ctx->get_saved_variables();
        const auto v = ctx->saved_data["ints"].toIntVector();
        check_device("qk_rope_bwd", {&grads[0], &grads[1], &sv[0]});
        const auto dt = (at::ScalarType)v[2];
        const QkAxes axes = saved_axes(ctx);
        const Tensor gq = grads[0].to(dt), gk = grads[1].to(dt);
        // linear: its gradient's gradient is a call on the cotangents
        const tensor_list d =
            needs_node({&gq, &gk})
                ? QkRope::apply(gq, gk, sv[0], sv[1], sv[2], v[0], v[1] != 0, axes, v[5] == 0)
                : forward(nullptr, gq, gk, sv[0], sv[1], sv[2], v[0], v[1] != 0, axes, v[5] == 0);
        tensor_list out = {d[0].to((at::ScalarType)v[3]), d[1].to((at::ScalarType)v[4])};
        out.resize(9);
        return out;
    }
};

Tensor dropout(const Tensor& x, double p, const c10::optional<Tensor>& seed, const c10::optional<int64_t>& value,
               int64_t offset) {
    require_bound();
    const char* fn = "dropout";
    check_device(fn, {&x});
    check_rows(fn, x);
    const Drop d = make_drop(fn, x, p, seed, value, offset);
    return needs_node({&x}) ? Dropout::apply(x, d) : Dropout::forward(nullptr, x, d);
}

tensor_list rmsnorm_residual(const Tensor& x, const Tensor& residual, const Tensor& w, double eps, double p,
                             const c10::optional<Tensor>& seed, const c10::optional<int64_t>& value, int64_t offset,
                             int64_t checkpoint, int64_t y_fmt) {
    require_bound();
    const char* fn = "rmsnorm_residual";
    check_device(fn, {&x, &residual, &w});
    check_rows(fn, x);
    TORCH_CHECK(residual.sizes() == x.sizes() && at::isFloatingType(residual.scalar_type()), fn,
                ": x and residual must be floating-point tensors of one shape, got ", x.sizes(), " and ",
                residual.sizes());
    TORCH_CHECK(w.dim() == 1 && w.numel() == x.size(-1), fn, ": weight must be [C], got ", w.sizes());
    const bool node = needs_node({&x, &residual, &w});
    TORCH_CHECK(y_fmt == MHC_CHECKPOINT_NONE || !node, fn,
                ": no gradient flows through an output in 8 bits (call it under torch.no_grad())");
    const int64_t fmt = format_for(checkpoint, {&x, &residual, &w});
    const Drop d = make_drop(fn, x, p, seed, value, offset);
    return node ? RmsNormResidual::apply(x, residual, w, eps, d, fmt, y_fmt)
                : RmsNormResidual::forward(nullptr, x, residual, w, eps, d, fmt, y_fmt);
}

// (values, scales) of x [..., C]: uint8 [..., ceil16(C)] and [..., ceil(C / 32)]
std::tuple<Tensor, Tensor> checkpoint_pack(const Tensor& x_in, int64_t fmt) {
    require_bound();
    const char* fn = "checkpoint_pack";
    const at::NoGradGuard no_grad;
    check_device(fn, {&x_in});
    TORCH_CHECK(x_in.dim() >= 1 && at::isFloatingType(x_in.scalar_type()), fn,
                ": x must be a floating-point tensor [..., C]");
    TORCH_CHECK(x_in.size(-1) >= 1, fn, ": x must have at least one channel");
    const at::DeviceGuard guard(x_in.device());
    const Tensor x = storage(x_in);
    const int64_t C = x.size(-1);
    Held h = hold(x, fmt);
    auto shape = x.sizes().vec();
    shape.back() = (C + 15) / 16 * 16;
    const Tensor values = h.values.view(shape);
    shape.back() = (C + 31) / 32;
    return {values, h.scales.view(shape)};
}

// The values [..., hidden] that a checkpoint stands for, in dtype.
Tensor checkpoint_unpack(const Tensor& values_in, const Tensor& scales_in, int64_t fmt, int64_t hidden,
                         at::ScalarType dtype) {
    require_bound();
    const char* fn = "checkpoint_unpack";
    const at::NoGradGuard no_grad;
    check_device(fn, {&values_in, &scales_in});
    TORCH_CHECK(values_in.scalar_type() == at::kByte && scales_in.scalar_type() == at::kByte, fn,
                ": values and scales must be uint8");
    const auto &vs = values_in.sizes(), &ss = scales_in.sizes();
    TORCH_CHECK(hidden >= 1 && hidden <= INT32_MAX && vs.size() >= 1 && vs.size() == ss.size() && vs.back() == (hidden + 15) / 16 * 16 &&
                    ss.back() == (hidden + 31) / 32 && vs.slice(0, vs.size() - 1) == ss.slice(0, ss.size() - 1),
                fn, ": values ", vs, " and scales ", ss, " do not match hidden=", hidden);
    const at::DeviceGuard guard(values_in.device());
    Tensor values = values_in.contiguous();
    if (reinterpret_cast<uintptr_t>(values.data_ptr()) % 16 != 0) values = values.clone();
    auto shape = vs.vec();
    shape.back() = hidden;
    return held_rows(values, scales_in.contiguous(), fmt, shape, dtype);
}

Tensor sinkhorn_knopp(const Tensor& inp, int64_t iters, double eps) {
    require_bound();
    return Sinkhorn::apply(inp, iters, eps);
}

Tensor rmsnorm(const Tensor& inp, const Tensor& w, double eps, int64_t checkpoint) {
    require_bound();
    const int64_t fmt = format_for(checkpoint, {&inp, &w});
    return fmt == MHC_CHECKPOINT_NONE ? RmsNorm::apply(inp, w, eps) : RmsNormHeld::apply(inp, w, eps, fmt);
}

Tensor stream_aggregate(const Tensor& inp, const Tensor& h, int64_t checkpoint) {
    require_bound();
    return Aggregate::apply(inp, h, format_for(checkpoint, {&inp, &h}));
}

Tensor stream_distribute_mix_add(const Tensor& y, const Tensor& h, const Tensor& m, const Tensor& x,
                                 int64_t checkpoint) {
    require_bound();
    return Distribute::apply(y, h, m, x, format_for(checkpoint, {&y, &h, &m, &x}));
}

// What the two entries share: q and k as [tokens, heads, D], their leading sizes and
// the positions' period.
struct QkCall {
    Tensor q, k;
    at::DimVector lead;
    int64_t period;

    QkCall(const char* fn, const Tensor& q_in, const Tensor& k_in, const Tensor& cos, const Tensor& sin,
           const c10::optional<Tensor>& positions, const QkAxes& axes, std::initializer_list<const Tensor*> weights) {
        if (positions.has_value()) check_device(fn, {&q_in, &*positions});
        const int64_t dims = q_in.dim();
        TORCH_CHECK((dims == 3 || dims == 4) && k_in.dim() == dims, fn,
                    ": q and k must both be [tokens, heads, D] or [batch, seq, heads, D], got ", q_in.sizes(), " and ",
                    k_in.sizes());
        lead = q_in.sizes().slice(0, dims - 2);
        TORCH_CHECK(at::IntArrayRef(lead) == k_in.sizes().slice(0, dims - 2) && q_in.size(-1) == k_in.size(-1), fn,
                    ": q and k must have the same tokens and head_dim, got ", q_in.sizes(), " and ", k_in.sizes());
        TORCH_CHECK(q_in.scalar_type() == k_in.scalar_type() && at::isFloatingType(q_in.scalar_type()), fn,
                    ": q and k must have one floating dtype, got ", q_in.scalar_type(), " and ", k_in.scalar_type());
        const int64_t D = q_in.size(-1);
        for (const Tensor* w : weights)
            TORCH_CHECK(w->numel() == D && w->dim() == 1, fn, ": the weights must be [head_dim]");
        TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes(), fn,
                    ": cos and sin must be [positions, rotary_dim / 2]");
        TORCH_CHECK(!cos.requires_grad() && !sin.requires_grad() && !cos._fw_grad(0).defined() &&
                        !sin._fw_grad(0).defined(),
                    fn, ": cos and sin get no gradient");
        TORCH_CHECK(q_in.size(-2) <= INT32_MAX && k_in.size(-2) <= INT32_MAX && D <= INT32_MAX &&
                        2 * cos.size(1) <= D,
                    fn, ": rotary_dim must be at most head_dim, and the sizes 32-bit");
        if (axes.any()) {
            int64_t sum = 0;
            for (const int64_t n : axes.sections) {
                TORCH_CHECK(n >= 0 && n <= cos.size(1), fn, ": sections must be in 0 .. rotary_dim / 2, got ", n);
                sum += n;
            }
            TORCH_CHECK(axes.count() <= 4 && sum == cos.size(1), fn,
                        ": sections must name at most 4 axes and add up to rotary_dim / 2 = ", cos.size(1));
            TORCH_CHECK(positions.has_value(), fn, ": sections need positions");
        }
        period = lead.back();
        if (positions.has_value()) {
            const auto pt = positions->scalar_type();
            at::IntArrayRef ps = positions->sizes();
            if (axes.any()) {
                TORCH_CHECK(positions->dim() >= 1 && ps[0] == axes.count(), fn, ": positions must be [",
                            axes.count(), ", ...], one row an axis, got ", ps);
                ps = ps.slice(1);
            }
            TORCH_CHECK(ps == at::IntArrayRef(lead) || ps == at::IntArrayRef(lead).slice(lead.size() - 1), fn,
                        ": positions must be ", at::IntArrayRef(lead), " or ",
                        at::IntArrayRef(lead).slice(lead.size() - 1), axes.any() ? " an axis" : "", ", got ", ps);
            TORCH_CHECK(pt == at::kLong || pt == at::kInt, fn, ": positions must be int64 or int32, got ", pt);
            period = c10::multiply_integers(ps);
        }
        period = std::max<int64_t>(period, 1);
        q = dims == 4 ? q_in.flatten(0, 1) : q_in;
        k = dims == 4 ? k_in.flatten(0, 1) : k_in;
    }

    std::tuple<Tensor, Tensor> shaped(const tensor_list& out) const {
        if (lead.size() == 1) return {out[0], out[1]};
        return {out[0].unflatten(0, lead), out[1].unflatten(0, lead)};
    }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q_in, const Tensor& k_in, const Tensor& wq, const Tensor& wk,
                                        const Tensor& cos, const Tensor& sin, const c10::optional<Tensor>& positions,
                                        double eps, bool interleaved, int64_t checkpoint,
                                        const std::vector<int64_t>& sections, bool dealt) {
    require_bound();
    const char* fn = "qk_norm_rope";
    check_device(fn, {&q_in, &k_in, &wq, &wk, &cos, &sin});
    const QkAxes axes(sections, dealt);
    const QkCall call(fn, q_in, k_in, cos, sin, positions, axes, {&wq, &wk});
    const Tensor &q = call.q, &k = call.k;
    const int64_t fmt = format_for(checkpoint, {&q, &k, &wq, &wk});
    return call.shaped(needs_node({&q, &k, &wq, &wk})
                           ? QkNormRope::apply(q, k, wq, wk, cos, sin, positions, call.period, eps, interleaved, fmt,
                                               axes)
                           : QkNormRope::forward(nullptr, q, k, wq, wk, cos, sin, positions, call.period, eps,
                                                 interleaved, fmt, axes));
}

std::tuple<Tensor, Tensor> qk_rope(const Tensor& q_in, const Tensor& k_in, const Tensor& cos, const Tensor& sin,
                                   const c10::optional<Tensor>& positions, bool interleaved,
                                   const std::vector<int64_t>& sections, bool dealt) {
    require_bound();
    const char* fn = "qk_rope";
    check_device(fn, {&q_in, &k_in, &cos, &sin});
    const QkAxes axes(sections, dealt);
    const QkCall call(fn, q_in, k_in, cos, sin, positions, axes, {});
    return call.shaped(needs_node({&call.q, &call.k})
                           ? QkRope::apply(call.q, call.k, cos, sin, positions, call.period, interleaved, axes, false)
                           : QkRope::forward(nullptr, call.q, call.k, cos, sin, positions, call.period, interleaved,
                                             axes, false));
}

Tensor static_layer(const Tensor& x, const Tensor& w, const Tensor& hp, const Tensor& hq, const Tensor& hr,
                    int64_t iters, double sk_eps, double rms_eps, int64_t checkpoint) {
    require_bound();
    return StaticLayer::apply(x, w, hp, hq, hr, iters, sk_eps, rms_eps,
                              format_for(checkpoint, {&x, &w, &hp, &hq, &hr}));
}

Tensor dynamic_layer(const Tensor& x, const Tensor& w, const Tensor& pp, const Tensor& pq, const Tensor& pr,
                     const Tensor& ap, const Tensor& aq, const Tensor& ar, const Tensor& bp, const Tensor& bq,
                     const Tensor& br, int64_t iters, double sk_eps, double rms_eps, int64_t checkpoint) {
    require_bound();
    return DynamicLayer::apply(x, w, pp, pq, pr, ap, aq, ar, bp, bq, br, iters, sk_eps, rms_eps,
                               format_for(checkpoint, {&x, &w, &pp, &pq, &pr, &ap, &aq, &ar, &bp, &bq, &br}));
}

Tensor static_wrapper(const Tensor& residual, const Tensor& branch, const Tensor& w, const Tensor& hp,
                      const Tensor& hq, const Tensor& hr, const std::string& mode, int64_t n, int64_t iters,
                      double sk_eps, double rms_eps, int64_t checkpoint) {
    require_bound();
    const int32_t m = wrapper_mode(mode, n, "wrapper_static_fwd");
    return StaticWrapper::apply(residual, branch, w, hp, hq, hr, (int64_t)m, n, iters, sk_eps, rms_eps,
                                format_for(checkpoint, {&residual, &branch, &w, &hp, &hq, &hr}));
}

Tensor dynamic_wrapper(const Tensor& residual, const Tensor& branch, const Tensor& w, const Tensor& pp,
                       const Tensor& pq, const Tensor& pr, const Tensor& ap, const Tensor& aq, const Tensor& ar,
                       const Tensor& bp, const Tensor& bq, const Tensor& bres, const std::string& mode, int64_t n,
                       int64_t iters, double sk_eps, double rms_eps, int64_t checkpoint) {
    require_bound();
    const int32_t m = wrapper_mode(mode, n, "wrapper_dynamic_fwd");
    return DynamicWrapper::apply(residual, branch, w, pp, pq, pr, ap, aq, ar, bp, bq, bres, (int64_t)m, n, iters,
                                 sk_eps, rms_eps,
                                 format_for(checkpoint, {&residual, &branch, &w, &pp, &pq, &pr, &ap, &aq, &ar, &bp,
                                                         &bq, &bres}));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.doc() = "C++ autograd nodes of the fused mHC layers and the standalone operators over libmhc_hip's C ABI";
    m.def("entry_names", &entry_names, "C-ABI entry points bind() needs");
    m.def("bind", &bind, "set the C-ABI entry points from {name: address}");
    m.def("static_layer", &static_layer,
          "static-H layer with autograd: (x, weight, H_pre, H_post, H_res, num_iters, sinkhorn_eps, "
          "rmsnorm_eps) -> fp32 [B, n, C]",
          py::arg("x"), py::arg("weight"), py::arg("H_pre"), py::arg("H_post"), py::arg("H_res"), py::arg("num_iters"),
          py::arg("sinkhorn_eps"), py::arg("rmsnorm_eps"), py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("dynamic_layer", &dynamic_layer,
          "dynamic-H layer with autograd: (x, weight, phi_pre, phi_post, phi_res, alpha_pre, alpha_post, "
          "alpha_res, b_pre, b_post, b_res, num_iters, sinkhorn_eps, rmsnorm_eps) -> fp32 [B, n, C]",
          py::arg("x"), py::arg("weight"), py::arg("phi_pre"), py::arg("phi_post"), py::arg("phi_res"),
          py::arg("alpha_pre"), py::arg("alpha_post"), py::arg("alpha_res"), py::arg("b_pre"), py::arg("b_post"),
          py::arg("b_res"), py::arg("num_iters"), py::arg("sinkhorn_eps"), py::arg("rmsnorm_eps"),
          py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("static_wrapper", &static_wrapper,
          "fused static-H MHCResidualWrapper with autograd: (residual, branch, weight, H_pre, H_post, H_res, "
          "residual_mode, n, num_iters, sinkhorn_eps, rmsnorm_eps) -> fp32 [tokens, C]",
          py::arg("residual"), py::arg("branch"), py::arg("weight"), py::arg("H_pre"), py::arg("H_post"),
          py::arg("H_res"), py::arg("residual_mode"), py::arg("n"), py::arg("num_iters"), py::arg("sinkhorn_eps"),
          py::arg("rmsnorm_eps"), py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("dynamic_wrapper", &dynamic_wrapper,
          "fused dynamic-H MHCResidualWrapper with autograd: (residual, branch, weight, phi_pre, phi_post, phi_res, "
          "alpha_pre, alpha_post, alpha_res, b_pre, b_post, b_res, residual_mode, n, num_iters, sinkhorn_eps, "
          "rmsnorm_eps) -> fp32 [tokens, C]",
          py::arg("residual"), py::arg("branch"), py::arg("weight"), py::arg("phi_pre"), py::arg("phi_post"),
          py::arg("phi_res"), py::arg("alpha_pre"), py::arg("alpha_post"), py::arg("alpha_res"), py::arg("b_pre"),
          py::arg("b_post"), py::arg("b_res"), py::arg("residual_mode"), py::arg("n"), py::arg("num_iters"),
          py::arg("sinkhorn_eps"), py::arg("rmsnorm_eps"), py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("dynamic_infer", &dynamic_infer,
          "forward-only dynamic-H layer: (x, packed, alpha_pre, alpha_post, alpha_res, b_pre, b_post, b_res, "
          "num_iters, sinkhorn_eps, rmsnorm_eps, out_bf16) -> [B, n, C]");
    m.def("sinkhorn_knopp", &sinkhorn_knopp, "(inp [B, n, n] fp32, num_iters, eps) with autograd");
    m.def("rmsnorm", &rmsnorm, "(inp [B, C], weight, eps) with autograd",
          py::arg("inp"), py::arg("weight"), py::arg("eps"), py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("stream_aggregate", &stream_aggregate, "(inp [B, n, C], H_pre_raw [B, n]) with autograd",
          py::arg("inp"), py::arg("H_pre_raw"), py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("stream_distribute_mix_add", &stream_distribute_mix_add,
          "(y_norm [B, C], H_post_raw [B, n], M [B, n, n], x_inp [B, n, C]) -> fp32 [B, n, C] with autograd",
          py::arg("y_norm"), py::arg("H_post_raw"), py::arg("M"), py::arg("x_inp"),
          py::arg("checkpoint") = MHC_CHECKPOINT_NONE);
    m.def("checkpoint_pack", &checkpoint_pack, "(x [..., C], format) -> (values, scales), without autograd");
    m.def("checkpoint_unpack",
          [](const Tensor& values, const Tensor& scales, int64_t fmt, int64_t hidden, bool bf16) {
              return checkpoint_unpack(values, scales, fmt, hidden, bf16 ? at::kBFloat16 : at::kFloat);
          },
          "(values, scales, format, hidden, bf16) -> [..., hidden]");
    m.def("dropout", &dropout, "(x [..., C], p, seed tensor or None, seed value or None, offset) with autograd");
    m.def("rmsnorm_residual", &rmsnorm_residual,
          "(x [..., C], residual [..., C], weight, eps, p, seed tensor or None, seed value or None, offset, checkpoint, "
          "y_format) -> [y, h] with autograd, or [values, scales, h]");
    m.def("qk_norm_rope", &qk_norm_rope,
          "(q [..., H, D], k [..., K, D], q_weight, k_weight, cos, sin, positions or None, eps, interleaved, "
          "checkpoint, sections, dealt) -> (q, k) with autograd",
          py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"), py::arg("sin"),
          py::arg("positions"), py::arg("eps"), py::arg("interleaved"), py::arg("checkpoint"),
          py::arg("sections") = std::vector<int64_t>{}, py::arg("dealt") = false);
    m.def("qk_rope", &qk_rope,
          "(q [..., H, D], k [..., K, D], cos, sin, positions or None, interleaved, sections, dealt) -> (q, k) with "
          "autograd");
}
