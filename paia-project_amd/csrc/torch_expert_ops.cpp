// torch.library custom ops of the feed-forward half of a layer with experts: residual and norms, each token's experts, the
// experts' products. Same conduct as torch_ops.cpp: tensors are checked here, the C ABI is called on torch's current HIP
// stream of the operands' device, Meta kernels give shapes.
#include <ATen/hip/EmptyTensor.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>
#include <string>
#include <tuple>

#include "paia_gemv.h"
#include "torch_operands.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

// A new tensor beside `like`; on a GPU straight from its allocator (through the dispatcher each took as long as a launch).
at::Tensor new_like(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type)
{
    if (like.is_cuda()) return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
    return at::empty(sizes, like.options().dtype(type));
}

bool is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }

// -------------------------------------------------------------------------------------------------------------
void add_norm_out(const at::Tensor& x, const OptTensor& residual, const at::Tensor& norm, const OptTensor& post_norm,
                  const OptTensor& gate, const OptTensor& weights, double scale, double eps, bool plus_one,
                  const at::Tensor& out, const at::Tensor& residual_out)
{
    TORCH_CHECK(x.is_cuda(), "x must be on a GPU, found ", x.device());
    TORCH_CHECK((x.dim() == 2 || x.dim() == 3) && is_bf16(x) && (x.numel() == 0 || x.size(-1) == 1 || x.stride(-1) == 1),
                "x must be bfloat16 [M, D] or [M, pairs, D], its last dimension contiguous");
    const int64_t M = x.size(0), D = x.size(-1), pairs = x.dim() == 3 ? x.size(1) : 0;
    TORCH_CHECK(D > 0 && (x.dim() == 2 || pairs > 0), "x must have values");
    TORCH_CHECK((x.dim() == 3) == weights.has_value(), "weights go with an x of [M, pairs, D]");
    const bool wide = residual.has_value() && residual->scalar_type() == at::kFloat;
    const auto check_rows = [&](const at::Tensor& t, at::ScalarType type, const char* name) {
        TORCH_CHECK(rows_of(t) && t.scalar_type() == type && t.size(0) == M && t.size(1) == D, name, " must be ",
                    at::toString(type), " [", M, ", ", D, "] with contiguous rows");
        on_device_of(x, t, name);
    };
    if (residual.has_value()) {
        TORCH_CHECK(wide || is_bf16(*residual), "residual must be bfloat16 or float32");
        check_rows(*residual, wide ? at::kFloat : at::kBFloat16, "residual");
    }
    long long gate_stride = 0;
    if (gate.has_value()) {
        if (gate->dim() == 1) {
            opt_ptr(gate, at::kBFloat16, D, x, "gate");
        } else {
            check_rows(*gate, at::kBFloat16, "gate");
            gate_stride = stride_of(*gate, 0);
        }
    }
    check_rows(out, at::kBFloat16, "out");
    check_rows(residual_out, wide ? at::kFloat : at::kBFloat16, "residual_out");
    c10::DeviceGuard g(x.device());
    check_rc(paia_add_norm(x.data_ptr(), stride_of(x, 0),
                           opt_ptr(weights, at::kFloat, M * pairs, x, "weights"), pairs > 0 ? stride_of(x, 1) : 0,
                           to_int(pairs, "pairs"), residual.has_value() ? residual->data_ptr() : nullptr,
                           residual.has_value() ? stride_of(*residual, 0) : 0, wide,
                           opt_ptr(post_norm, at::kBFloat16, D, x, "post_norm"),
                           gate.has_value() ? gate->data_ptr() : nullptr, gate_stride, (float)scale,
                           opt_ptr(norm, at::kBFloat16, D, x, "norm"), plus_one, (float)eps, out.data_ptr(),
                           stride_of(out, 0), residual_out.data_ptr(), stride_of(residual_out, 0), to_int(M, "M"),
                           to_int(D, "D"), stream_of(x)),
             "paia_add_norm");
}
std::tuple<at::Tensor, at::Tensor> add_norm_new(const at::Tensor& x, const OptTensor& residual)
{
    TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "x must be [M, D] or [M, pairs, D]");
    return {new_like(x, {x.size(0), x.size(-1)}, at::kBFloat16),
            new_like(x, {x.size(0), x.size(-1)}, residual.has_value() ? residual->scalar_type() : at::kBFloat16)};
}
std::tuple<at::Tensor, at::Tensor> add_norm(const at::Tensor& x, const OptTensor& residual, const at::Tensor& norm,
                                            const OptTensor& post_norm, const OptTensor& gate, const OptTensor& weights,
                                            double scale, double eps, bool plus_one)
{
    auto made = add_norm_new(x, residual);
    add_norm_out(x, residual, norm, post_norm, gate, weights, scale, eps, plus_one, std::get<0>(made), std::get<1>(made));
    return made;
}

// -------------------------------------------------------------------------------------------------------------
using Route = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

bool by_sigmoid(c10::string_view scoring)
{
    TORCH_CHECK(scoring == "softmax" || scoring == "sigmoid", "scoring must be \"softmax\" or \"sigmoid\"");
    return scoring == "sigmoid";
}
long long route_need(int64_t M, int64_t E, int64_t k)
{
    const long long need = paia_route_experts_workspace(to_int(M, "M"), to_int(E, "experts"), to_int(k, "k"));
    check_rc(need < 0 ? (int)need : 0, "paia_route_experts");
    return need;
}
Route route_new(const at::Tensor& logits, int64_t k)
{
    TORCH_CHECK(logits.dim() == 2 && k > 0, "logits must be [M, experts], k positive");
    const int64_t M = logits.size(0);
    return {new_like(logits, {M, k}, at::kInt), new_like(logits, {M, k}, at::kFloat), new_like(logits, {M * k}, at::kInt),
            new_like(logits, {logits.size(1) + 1}, at::kInt)};
}
Route route_experts(const at::Tensor& logits, int64_t k, const OptTensor& bias, c10::string_view scoring, bool renormalize,
                    double scale, const OptTensor& workspace)
{
    TORCH_CHECK(logits.is_cuda(), "logits must be on a GPU, found ", logits.device());
    TORCH_CHECK(rows_of(logits) && (is_bf16(logits) || logits.scalar_type() == at::kFloat),
                "logits must be bfloat16 or float32 [M, experts] with contiguous rows");
    const int64_t M = logits.size(0), E = logits.size(1);
    const bool sigmoid = by_sigmoid(scoring);
    TORCH_CHECK(sigmoid || !bias.has_value(), "bias goes with sigmoid scoring");
    TORCH_CHECK(k > 0 && k <= E, "k must be between 1 and the number of experts (", E, ")");
    c10::DeviceGuard g(logits.device());
    const long long need = route_need(M, E, k);
    const Workspace space(workspace, need, logits);
    const Route made = route_new(logits, k);
    const auto& [ids, weights, order, offsets] = made;
    check_rc(paia_route_experts(logits.data_ptr(), logits.scalar_type() == at::kFloat, stride_of(logits, 0),
                                opt_ptr(bias, at::kFloat, E, logits, "bias"), sigmoid, renormalize, (float)scale,
                                ids.data_ptr(), weights.data_ptr(), order.data_ptr(), offsets.data_ptr(), (int)M, (int)E,
                                (int)k, space.data, space.bytes, stream_of(logits)),
             "paia_route_experts");
    return made;
}

using Order = std::tuple<at::Tensor, at::Tensor>;
Order order_new(const at::Tensor& ids, int64_t experts)
{
    TORCH_CHECK(ids.dim() == 2 && experts > 0, "ids must be [M, k], experts positive");
    return {new_like(ids, {ids.numel()}, at::kInt), new_like(ids, {experts + 1}, at::kInt)};
}
Order expert_order(const at::Tensor& ids, int64_t experts, const OptTensor& workspace)
{
    TORCH_CHECK(ids.is_cuda(), "ids must be on a GPU, found ", ids.device());
    TORCH_CHECK(ids.dim() == 2 && ids.scalar_type() == at::kInt && ids.is_contiguous() && ids.size(1) > 0,
                "ids must be contiguous int32 [M, k]");
    const int64_t M = ids.size(0), k = ids.size(1);
    c10::DeviceGuard g(ids.device());
    const long long need = route_need(M, experts, k);
    const Workspace space(workspace, need, ids);
    const Order made = order_new(ids, experts);
    check_rc(paia_expert_order(ids.data_ptr(), std::get<0>(made).data_ptr(), std::get<1>(made).data_ptr(), (int)M,
                               (int)experts, (int)k, space.data, space.bytes, stream_of(ids)),
             "paia_expert_order");
    return made;
}
int64_t route_experts_workspace(int64_t M, int64_t experts, int64_t k) { return route_need(M, experts, k); }

// -------------------------------------------------------------------------------------------------------------
// What the formats share: rows, order and output of a call.
struct Call {
    int64_t E, N, K;
    int pairs, x_rows;
    const void* bias;
};
Call call_of(const at::Tensor& W, int64_t K, const at::Tensor& x, const at::Tensor& order, const at::Tensor& offsets,
             const OptTensor& bias, bool gated, const at::Tensor& out)
{
    TORCH_CHECK(W.is_cuda(), "the weights must be on a GPU, found ", W.device());
    Call c{W.size(0), W.size(1), K, 0, 0, nullptr};
    TORCH_CHECK(c.E > 0 && c.N > 0 && K > 0, "the weights must not be empty");
    TORCH_CHECK(is_bf16(x) && rows_of(x) && x.size(1) == K, "x must be bfloat16 [rows, ", K, "] with contiguous rows");
    on_device_of(W, x, "x");
    TORCH_CHECK(order.dim() == 1, "order must be one row of pairs");
    check_index(order, at::kInt, order.numel(), W, "order");
    check_index(offsets, at::kInt, c.E + 1, W, "offsets");
    c.pairs = to_int(order.numel(), "the number of pairs");
    c.x_rows = to_int(x.size(0), "the rows of x");
    TORCH_CHECK(c.pairs == 0 || (c.x_rows > 0 && c.pairs % c.x_rows == 0), "the pairs (", c.pairs,
                ") must be a multiple of the rows of x (", c.x_rows, ")");
    TORCH_CHECK(!gated || c.N % 2 == 0, "gated experts have an even number of rows, found ", c.N);
    TORCH_CHECK(is_bf16(out) && rows_of(out) && out.size(0) == c.pairs && out.size(1) == (gated ? c.N / 2 : c.N),
                "out must be bfloat16 [", c.pairs, ", ", gated ? c.N / 2 : c.N, "] with contiguous rows");
    on_device_of(W, out, "out");
    if (bias.has_value()) {
        TORCH_CHECK(bias->dim() == 2, "bias must be [experts, N]");
        c.bias = opt_ptr(bias, at::kBFloat16, c.E * c.N, W, "bias");
    }
    return c;
}
void check_meta(const at::Tensor& W, const at::Tensor& t, at::ScalarType type, int64_t n, const char* name)
{
    opt_ptr(t, type, n, W, name);
}
at::Tensor experts_new(const at::Tensor& W, const at::Tensor& x, const at::Tensor& order, bool gated)
{
    TORCH_CHECK(W.dim() == 3 && order.dim() == 1, "W must be [experts, N, ...], order one row of pairs");
    return new_like(x, {order.size(0), gated ? W.size(1) / 2 : W.size(1)}, at::kBFloat16);
}

void experts_bf16_out(const at::Tensor& W, const at::Tensor& x, const at::Tensor& order, const at::Tensor& offsets,
                      const OptTensor& bias, bool gated, at::Tensor& out)
{
    TORCH_CHECK(W.dim() == 3 && is_bf16(W) && W.is_contiguous(), "W must be contiguous bfloat16 [experts, N, K]");
    const Call c = call_of(W, W.size(2), x, order, offsets, bias, gated, out);
    c10::DeviceGuard g(W.device());
    check_rc(paia_experts_bf16(W.data_ptr(), x.data_ptr(), stride_of(x, 0), c.x_rows, order.data_ptr(), offsets.data_ptr(),
                               c.bias, out.data_ptr(), stride_of(out, 0), to_int(c.E, "experts"), to_int(c.N, "N"),
                               to_int(c.K, "K"), c.pairs, gated, stream_of(W)),
             "paia_experts_bf16");
}
void experts_fp8_out(const at::Tensor& Wq, const at::Tensor& scale, const at::Tensor& x, const at::Tensor& order,
                     const at::Tensor& offsets, const OptTensor& bias, bool gated, at::Tensor& out)
{
    TORCH_CHECK(Wq.dim() == 3 && (Wq.scalar_type() == at::kByte || Wq.scalar_type() == at::kFloat8_e4m3fn) &&
                    Wq.is_contiguous(), "Wq must be contiguous e4m3 (float8_e4m3fn or uint8) [experts, N, K]");
    const Call c = call_of(Wq, Wq.size(2), x, order, offsets, bias, gated, out);
    check_meta(Wq, scale, at::kFloat, c.E * c.N, "scale");
    c10::DeviceGuard g(Wq.device());
    check_rc(paia_experts_fp8(Wq.data_ptr(), scale.data_ptr(), x.data_ptr(), stride_of(x, 0), c.x_rows, order.data_ptr(),
                              offsets.data_ptr(), c.bias, out.data_ptr(), stride_of(out, 0), to_int(c.E, "experts"),
                              to_int(c.N, "N"), to_int(c.K, "K"), c.pairs, gated, stream_of(Wq)),
             "paia_experts_fp8");
}
int64_t int4_columns(const at::Tensor& Wq)
{
    TORCH_CHECK(Wq.dim() == 3 && (Wq.scalar_type() == at::kByte || Wq.scalar_type() == at::kInt) && Wq.is_contiguous(),
                "Wq must be contiguous uint8 [experts, N, K/2] or int32 [experts, N, K/8]");
    return Wq.size(2) * (Wq.scalar_type() == at::kByte ? 2 : 8);
}
void experts_int4_out(const at::Tensor& Wq, const at::Tensor& scales, const at::Tensor& x, const at::Tensor& order,
                      const at::Tensor& offsets, bool gated, at::Tensor& out)
{
    const Call c = call_of(Wq, int4_columns(Wq), x, order, offsets, {}, gated, out);
    check_meta(Wq, scales, at::kHalf, c.E * c.N * (c.K / 128), "scales");
    c10::DeviceGuard g(Wq.device());
    check_rc(paia_experts_int4(Wq.data_ptr(), scales.data_ptr(), x.data_ptr(), stride_of(x, 0), c.x_rows, order.data_ptr(),
                               offsets.data_ptr(), out.data_ptr(), stride_of(out, 0), to_int(c.E, "experts"),
                               to_int(c.N, "N"), to_int(c.K, "K"), c.pairs, gated, stream_of(Wq)),
             "paia_experts_int4");
}
void experts_int4_zp_out(const at::Tensor& Wq, const at::Tensor& scales, const at::Tensor& zeros, const at::Tensor& x,
                         const at::Tensor& order, const at::Tensor& offsets, const OptTensor& bias, bool gated,
                         at::Tensor& out)
{
    const Call c = call_of(Wq, int4_columns(Wq), x, order, offsets, bias, gated, out);
    const int64_t G = c.K / 128;
    check_meta(Wq, scales, at::kBFloat16, c.E * c.N * G, "scales");
    check_meta(Wq, zeros, at::kByte, c.E * c.N * ((G + 1) / 2), "zeros");
    c10::DeviceGuard g(Wq.device());
    check_rc(paia_experts_int4_zp(Wq.data_ptr(), scales.data_ptr(), zeros.data_ptr(), x.data_ptr(), stride_of(x, 0),
                                  c.x_rows, order.data_ptr(), offsets.data_ptr(), c.bias, out.data_ptr(), stride_of(out, 0),
                                  to_int(c.E, "experts"), to_int(c.N, "N"), to_int(c.K, "K"), c.pairs, gated, stream_of(Wq)),
             "paia_experts_int4_zp");
}
at::Tensor experts_bf16(const at::Tensor& W, const at::Tensor& x, const at::Tensor& order, const at::Tensor& offsets,
                        const OptTensor& bias, bool gated)
{
    at::Tensor out = experts_new(W, x, order, gated);
    experts_bf16_out(W, x, order, offsets, bias, gated, out);
    return out;
}
at::Tensor experts_fp8(const at::Tensor& Wq, const at::Tensor& scale, const at::Tensor& x, const at::Tensor& order,
                       const at::Tensor& offsets, const OptTensor& bias, bool gated)
{
    at::Tensor out = experts_new(Wq, x, order, gated);
    experts_fp8_out(Wq, scale, x, order, offsets, bias, gated, out);
    return out;
}
at::Tensor experts_int4(const at::Tensor& Wq, const at::Tensor& scales, const at::Tensor& x, const at::Tensor& order,
                        const at::Tensor& offsets, bool gated)
{
    at::Tensor out = experts_new(Wq, x, order, gated);
    experts_int4_out(Wq, scales, x, order, offsets, gated, out);
    return out;
}
at::Tensor experts_int4_zp(const at::Tensor& Wq, const at::Tensor& scales, const at::Tensor& zeros, const at::Tensor& x,
                           const at::Tensor& order, const at::Tensor& offsets, const OptTensor& bias, bool gated)
{
    at::Tensor out = experts_new(Wq, x, order, gated);
    experts_int4_zp_out(Wq, scales, zeros, x, order, offsets, bias, gated, out);
    return out;
}

// ---- Meta (shape-only) kernels ------------------------------------------------------------------------------
std::tuple<at::Tensor, at::Tensor> add_norm_meta(const at::Tensor& x, const OptTensor& residual, const at::Tensor&,
                                                 const OptTensor&, const OptTensor&, const OptTensor&, double, double, bool)
{
    return add_norm_new(x, residual);
}
void add_norm_out_meta(const at::Tensor&, const OptTensor&, const at::Tensor&, const OptTensor&, const OptTensor&,
                       const OptTensor&, double, double, bool, const at::Tensor&, const at::Tensor&) {}
Route route_experts_meta(const at::Tensor& logits, int64_t k, const OptTensor&, c10::string_view scoring, bool, double,
                         const OptTensor&)
{
    by_sigmoid(scoring);
    return route_new(logits, k);
}
Order expert_order_meta(const at::Tensor& ids, int64_t experts, const OptTensor&) { return order_new(ids, experts); }
at::Tensor experts_bf16_meta(const at::Tensor& W, const at::Tensor& x, const at::Tensor& order, const at::Tensor&,
                             const OptTensor&, bool gated)
{
    return experts_new(W, x, order, gated);
}
at::Tensor experts_fp8_meta(const at::Tensor& Wq, const at::Tensor&, const at::Tensor& x, const at::Tensor& order,
                            const at::Tensor&, const OptTensor&, bool gated)
{
    return experts_new(Wq, x, order, gated);
}
at::Tensor experts_int4_meta(const at::Tensor& Wq, const at::Tensor&, const at::Tensor& x, const at::Tensor& order,
                             const at::Tensor&, bool gated)
{
    return experts_new(Wq, x, order, gated);
}
at::Tensor experts_int4_zp_meta(const at::Tensor& Wq, const at::Tensor&, const at::Tensor&, const at::Tensor& x,
                                const at::Tensor& order, const at::Tensor&, const OptTensor&, bool gated)
{
    return experts_new(Wq, x, order, gated);
}
void experts_bf16_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&, bool,
                           at::Tensor&) {}
void experts_fp8_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                          const OptTensor&, bool, at::Tensor&) {}
void experts_int4_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, bool,
                           at::Tensor&) {}
void experts_int4_zp_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                              const at::Tensor&, const OptTensor&, bool, at::Tensor&) {}

}  // namespace

TORCH_LIBRARY_FRAGMENT(paia_gemv, m)
{
    m.def("add_norm(Tensor x, Tensor? residual, Tensor norm, Tensor? post_norm=None, Tensor? gate=None, Tensor? weights=None, "
          "float scale=1.0, float eps=1e-6, bool plus_one=False) -> (Tensor, Tensor)");
    m.def("add_norm_out(Tensor x, Tensor? residual, Tensor norm, Tensor? post_norm, Tensor? gate, Tensor? weights, "
          "float scale, float eps, bool plus_one, Tensor(a!) out, Tensor(b!) residual_out) -> ()");
    m.def("route_experts(Tensor logits, int k, Tensor? bias=None, str scoring=\"softmax\", bool renormalize=True, "
          "float scale=1.0, Tensor(a!)? workspace=None) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("route_experts_workspace(int M, int experts, int k) -> int", &route_experts_workspace);
    m.def("expert_order(Tensor ids, int experts, Tensor(a!)? workspace=None) -> (Tensor, Tensor)");
    m.def("experts_bf16(Tensor W, Tensor x, Tensor order, Tensor offsets, Tensor? bias=None, bool gated=False) -> Tensor");
    m.def("experts_bf16_out(Tensor W, Tensor x, Tensor order, Tensor offsets, Tensor? bias, bool gated, Tensor(a!) out) -> ()");
    m.def("experts_fp8(Tensor Wq, Tensor scale, Tensor x, Tensor order, Tensor offsets, Tensor? bias=None, bool gated=False) "
          "-> Tensor");
    m.def("experts_fp8_out(Tensor Wq, Tensor scale, Tensor x, Tensor order, Tensor offsets, Tensor? bias, bool gated, "
          "Tensor(a!) out) -> ()");
    m.def("experts_int4(Tensor Wq, Tensor scales, Tensor x, Tensor order, Tensor offsets, bool gated=False) -> Tensor");
    m.def("experts_int4_out(Tensor Wq, Tensor scales, Tensor x, Tensor order, Tensor offsets, bool gated, Tensor(a!) out) "
          "-> ()");
    m.def("experts_int4_zp(Tensor Wq, Tensor scales, Tensor zeros, Tensor x, Tensor order, Tensor offsets, "
          "Tensor? bias=None, bool gated=False) -> Tensor");
    m.def("experts_int4_zp_out(Tensor Wq, Tensor scales, Tensor zeros, Tensor x, Tensor order, Tensor offsets, Tensor? bias, "
          "bool gated, Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(paia_gemv, CUDA, m)
{
    m.impl("add_norm", &add_norm);
    m.impl("add_norm_out", &add_norm_out);
    m.impl("route_experts", &route_experts);
    m.impl("expert_order", &expert_order);
    m.impl("experts_bf16", &experts_bf16);
    m.impl("experts_bf16_out", &experts_bf16_out);
    m.impl("experts_fp8", &experts_fp8);
    m.impl("experts_fp8_out", &experts_fp8_out);
    m.impl("experts_int4", &experts_int4);
    m.impl("experts_int4_out", &experts_int4_out);
    m.impl("experts_int4_zp", &experts_int4_zp);
    m.impl("experts_int4_zp_out", &experts_int4_zp_out);
}

TORCH_LIBRARY_IMPL(paia_gemv, Meta, m)
{
    m.impl("add_norm", &add_norm_meta);
    m.impl("add_norm_out", &add_norm_out_meta);
    m.impl("route_experts", &route_experts_meta);
    m.impl("expert_order", &expert_order_meta);
    m.impl("experts_bf16", &experts_bf16_meta);
    m.impl("experts_bf16_out", &experts_bf16_out_meta);
    m.impl("experts_fp8", &experts_fp8_meta);
    m.impl("experts_fp8_out", &experts_fp8_out_meta);
    m.impl("experts_int4", &experts_int4_meta);
    m.impl("experts_int4_out", &experts_int4_out_meta);
    m.impl("experts_int4_zp", &experts_int4_zp_meta);
    m.impl("experts_int4_zp_out", &experts_int4_zp_out_meta);
}
