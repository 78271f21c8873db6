// torch.library custom ops for what lies between and beside the projections of a decode step: rotation with the write into
// the paged cache, attention over that cache, low-rank adapters. Same conduct as torch_ops.cpp: tensors are checked here, the
// C ABI is called on torch's current HIP stream of the operands' device, Meta kernels give shapes.
//
// A cache is two tensors [pages, kv_heads, page_size, head_dim], bf16 or e4m3 (float8_e4m3fn or uint8), whose last
// dimension is contiguous; the other three may have any strides that are multiples of 16 bytes, so a cache laid out as
// [pages, page_size, kv_heads, head_dim] is passed as its transpose(1, 2).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>

#include "paia_gemv.h"

namespace {

void check_rc(int rc, const char* what)
{
    TORCH_CHECK(rc == 0, what, " failed with code ", rc, " (-2 bad shape/alignment, >0 hipError_t)");
}

void* stream_of(const at::Tensor& t)
{
    return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// Every operand must live on the GPU the kernel runs on: `on` is the tensor whose device counts.
void on_device_of(const at::Tensor& on, const at::Tensor& t, const char* name)
{
    TORCH_CHECK(t.device() == on.device(), name, " must be on ", on.device(), ", found ", t.device());
}

// The data of an optional operand of the given type and length, null where there is none.
const void* opt_ptr(const std::optional<at::Tensor>& t, at::ScalarType type, int64_t n, const at::Tensor& on,
                    const char* name)
{
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->scalar_type() == type && t->is_contiguous() && t->numel() == n, name, " must be a contiguous ",
                at::toString(type), " tensor of ", n, " elements");
    on_device_of(on, *t, name);
    return t->data_ptr();
}

int to_int(int64_t v, const char* name)
{
    TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, name, " must fit in 32 bits");
    return (int)v;
}

void check_index(const at::Tensor& t, at::ScalarType type, int64_t n, const at::Tensor& on, const char* name)
{
    TORCH_CHECK(t.dim() == 1 && t.scalar_type() == type && t.is_contiguous() && t.numel() == n, name,
                " must be a contiguous ", at::toString(type), " tensor [", n, "]");
    on_device_of(on, t, name);
}

paia_kv_cache cache_of(const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& k_scale,
                       const std::optional<at::Tensor>& v_scale, const at::Tensor& on)
{
    const auto is_code = [](const at::Tensor& t) {
        return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte;
    };
    TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(),
                "k_cache and v_cache must both be [pages, kv_heads, page_size, head_dim]");
    TORCH_CHECK(k.scalar_type() == v.scalar_type() && (k.scalar_type() == at::kBFloat16 || is_code(k)),
                "k_cache and v_cache must both be bfloat16 or both e4m3 (float8_e4m3fn or uint8)");
    TORCH_CHECK(k.numel() > 0, "the cache must not be empty");
    TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, "the cache's last dimension must be contiguous");
    on_device_of(on, k, "k_cache");
    on_device_of(on, v, "v_cache");
    TORCH_CHECK(is_code(k) || (!k_scale.has_value() && !v_scale.has_value()), "k_scale and v_scale go with an e4m3 cache");
    paia_kv_cache c;
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.pages = to_int(k.size(0), "pages");
    c.kv_heads = to_int(k.size(1), "kv_heads");
    c.page_size = to_int(k.size(2), "page_size");
    c.head_dim = to_int(k.size(3), "head_dim");
    c.fp8 = is_code(k);
    c.k_scale = static_cast<const float*>(opt_ptr(k_scale, at::kFloat, c.kv_heads, on, "k_scale"));
    c.v_scale = static_cast<const float*>(opt_ptr(v_scale, at::kFloat, c.kv_heads, on, "v_scale"));
    for (int i = 0; i < 3; ++i) {
        c.k_strides[i] = k.stride(i);
        c.v_strides[i] = v.stride(i);
    }
    return c;
}

// -------------------------------------------------------------------------------------------------------------
void rope_append_out(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& cos_sin, at::Tensor& k_cache,
                     at::Tensor& v_cache, const at::Tensor& slots, int64_t num_heads,
                     const std::optional<at::Tensor>& q_norm, const std::optional<at::Tensor>& k_norm, double eps,
                     bool interleaved, const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                     at::Tensor& out)
{
    TORCH_CHECK(qkv.is_cuda(), "qkv must be on a GPU, found ", qkv.device());
    TORCH_CHECK(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 && (qkv.stride(1) == 1 || qkv.size(0) == 0),
                "qkv must be bfloat16 [M, (heads + 2 kv_heads) * head_dim] with contiguous rows");
    const paia_kv_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, qkv);
    const int64_t M = qkv.size(0), D = c.head_dim;
    TORCH_CHECK(num_heads > 0 && qkv.size(1) == (num_heads + 2 * (int64_t)c.kv_heads) * D, "qkv has ", qkv.size(1),
                " columns, (", num_heads, " + 2 * ", c.kv_heads, ") * ", D, " are wanted");
    check_index(positions, at::kLong, M, qkv, "positions");
    check_index(slots, at::kLong, M, qkv, "slots");
    TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous(),
                "cos_sin must be contiguous fp32 [context, rotary dims]");
    on_device_of(qkv, cos_sin, "cos_sin");
    TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.numel() == M * num_heads * D,
                "out must be a contiguous bfloat16 tensor [M, num_heads, head_dim]");
    on_device_of(qkv, out, "out");
    c10::DeviceGuard g(qkv.device());
    check_rc(paia_rope_append(qkv.data_ptr(), qkv.stride(0), positions.data_ptr(), cos_sin.data_ptr(),
                              to_int(cos_sin.size(0), "context"), to_int(cos_sin.size(1), "rotary dims"), interleaved,
                              opt_ptr(q_norm, at::kBFloat16, D, qkv, "q_norm"),
                              opt_ptr(k_norm, at::kBFloat16, D, qkv, "k_norm"), (float)eps, slots.data_ptr(), &c,
                              out.data_ptr(), to_int(M, "M"), to_int(num_heads, "num_heads"), stream_of(qkv)),
             "paia_rope_append");
}
at::Tensor rope_append(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& cos_sin, at::Tensor& k_cache,
                       at::Tensor& v_cache, const at::Tensor& slots, int64_t num_heads,
                       const std::optional<at::Tensor>& q_norm, const std::optional<at::Tensor>& k_norm, double eps,
                       bool interleaved, const std::optional<at::Tensor>& k_scale,
                       const std::optional<at::Tensor>& v_scale)
{
    TORCH_CHECK(qkv.dim() == 2 && k_cache.dim() == 4 && num_heads > 0, "qkv must be 2-D, k_cache 4-D, num_heads positive");
    at::Tensor out = at::empty({qkv.size(0), num_heads, k_cache.size(3)}, qkv.options());
    rope_append_out(qkv, positions, cos_sin, k_cache, v_cache, slots, num_heads, q_norm, k_norm, eps, interleaved, k_scale,
                    v_scale, out);
    return out;
}

// ---- Meta (shape-only) kernels ------------------------------------------------------------------------------
at::Tensor rope_append_meta(const at::Tensor& qkv, const at::Tensor&, const at::Tensor&, at::Tensor& k_cache, at::Tensor&,
                            const at::Tensor&, int64_t num_heads, const std::optional<at::Tensor>&,
                            const std::optional<at::Tensor>&, double, bool, const std::optional<at::Tensor>&,
                            const std::optional<at::Tensor>&)
{
    return at::empty({qkv.size(0), num_heads, k_cache.size(3)}, qkv.options());
}
void rope_append_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, at::Tensor&,
                          const at::Tensor&, int64_t, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                          double, bool, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, at::Tensor&) {}

}  // namespace

TORCH_LIBRARY_FRAGMENT(paia_gemv, m)
{
    m.def("rope_append(Tensor qkv, Tensor positions, Tensor cos_sin, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, "
          "int num_heads, Tensor? q_norm=None, Tensor? k_norm=None, float eps=1e-6, bool interleaved=False, "
          "Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
    m.def("rope_append_out(Tensor qkv, Tensor positions, Tensor cos_sin, Tensor(a!) k_cache, Tensor(b!) v_cache, "
          "Tensor slots, int num_heads, Tensor? q_norm, Tensor? k_norm, float eps, bool interleaved, Tensor? k_scale, "
          "Tensor? v_scale, Tensor(c!) out) -> ()");
}

TORCH_LIBRARY_IMPL(paia_gemv, CUDA, m)
{
    m.impl("rope_append", &rope_append);
    m.impl("rope_append_out", &rope_append_out);
}

TORCH_LIBRARY_IMPL(paia_gemv, Meta, m)
{
    m.impl("rope_append", &rope_append_meta);
    m.impl("rope_append_out", &rope_append_out_meta);
}
