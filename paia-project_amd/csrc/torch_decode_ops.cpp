// torch.library custom ops for what lies between and beside the projections of a decode step: rotation with the write into
// the paged cache, attention over that cache, low-rank adapters. Same conduct as torch_ops.cpp: tensors are checked here, the
// C ABI is called on torch's current HIP stream of the operands' device, Meta kernels give shapes.
//
// A cache is two tensors [pages, kv_heads, page_size, head_dim], bf16 or e4m3 (float8_e4m3fn or uint8), whose last
// dimension is contiguous; the other three may have any strides that are multiples of 16 bytes, so a cache laid out as
// [pages, page_size, kv_heads, head_dim] is passed as its transpose(1, 2).
#include <torch/library.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <tuple>

#include "paia_gemv.h"
#include "torch_operands.h"

namespace {

// A cache's sizes, type and strides, which tracing has too; no addresses.
paia_kv_cache shape_of(const at::Tensor& k, const at::Tensor& v)
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
    paia_kv_cache c{};
    c.pages = to_int(k.size(0), "pages");
    c.kv_heads = to_int(k.size(1), "kv_heads");
    c.page_size = to_int(k.size(2), "page_size");
    c.head_dim = to_int(k.size(3), "head_dim");
    c.fp8 = is_code(k);
    for (int i = 0; i < 3; ++i) {
        c.k_strides[i] = stride_of(k, i);
        c.v_strides[i] = stride_of(v, i);
    }
    return c;
}
paia_kv_cache cache_of(const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& k_scale,
                       const std::optional<at::Tensor>& v_scale, const at::Tensor& on)
{
    paia_kv_cache c = shape_of(k, v);
    on_device_of(on, k, "k_cache");
    on_device_of(on, v, "v_cache");
    TORCH_CHECK(c.fp8 || (!k_scale.has_value() && !v_scale.has_value()), "k_scale and v_scale go with an e4m3 cache");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.k_scale = static_cast<const float*>(opt_ptr(k_scale, at::kFloat, c.kv_heads, on, "k_scale"));
    c.v_scale = static_cast<const float*>(opt_ptr(v_scale, at::kFloat, c.kv_heads, on, "v_scale"));
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
    check_rc(paia_rope_append(qkv.data_ptr(), stride_of(qkv, 0), positions.data_ptr(), cos_sin.data_ptr(),
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

// -------------------------------------------------------------------------------------------------------------
// q [B, heads, D] (one token a sequence) or [B, T, heads, D]: its sizes as the C ABI takes them.
struct Query {
    int64_t B, T, heads;
    long long strides[3];
};
Query query_of(const at::Tensor& q)
{
    TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && q.scalar_type() == at::kBFloat16,
                "q must be bfloat16 [B, heads, head_dim] or [B, T, heads, head_dim]");
    TORCH_CHECK(q.numel() == 0 || q.stride(-1) == 1, "q's last dimension must be contiguous");
    const int64_t d = q.dim();
    return {q.size(0), d == 4 ? q.size(1) : 1, q.size(d - 2),
            {stride_of(q, 0), d == 4 ? stride_of(q, 1) : 0, stride_of(q, d - 2)}};
}

// lse may be an undefined tensor: not wanted.
void paged_attention_run(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                         const at::Tensor& block_table, const at::Tensor& lens, std::optional<double> scale, int64_t window,
                         const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                         const at::Tensor& out, const at::Tensor& lse, const std::optional<at::Tensor>& workspace)
{
    TORCH_CHECK(q.is_cuda(), "q must be on a GPU, found ", q.device());
    const Query y = query_of(q);
    const paia_kv_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, q);
    TORCH_CHECK(q.size(-1) == c.head_dim, "q and the cache must have the same head_dim");
    TORCH_CHECK(y.T > 0 && y.heads > 0 && y.heads % c.kv_heads == 0, "q's heads (", y.heads,
                ") must be a multiple of the cache's (", c.kv_heads, "), its tokens at least one");
    check_index(lens, at::kInt, y.B, q, "lens");
    TORCH_CHECK(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) == y.B &&
                    (block_table.size(1) <= 1 || block_table.numel() == 0 || block_table.stride(1) == 1),
                "block_table must be int32 [B, pages of a sequence] with contiguous rows");
    on_device_of(q, block_table, "block_table");
    TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.numel() == y.B * y.T * y.heads * c.head_dim,
                "out must be a contiguous bfloat16 tensor of q's shape");
    on_device_of(q, out, "out");
    TORCH_CHECK(window >= 0, "window must not be negative");
    const int B = to_int(y.B, "B"), T = to_int(y.T, "T"), heads = to_int(y.heads, "heads");
    const int width = to_int(block_table.size(1), "the block table's width");
    c10::DeviceGuard g(q.device());
    const long long need = paia_paged_attention_workspace(&c, width, B, T, heads);
    check_rc(need < 0 ? (int)need : 0, "paia_paged_attention");
    const Workspace space(workspace, need, q);
    const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)c.head_dim);
    check_rc(paia_paged_attention(q.data_ptr(), y.strides, &c, block_table.data_ptr(), stride_of(block_table, 0), width,
                                  lens.data_ptr(), (float)s, to_int(window, "window"), out.data_ptr(),
                                  lse.defined() ? lse.data_ptr() : nullptr, B, T, heads, space.data, space.bytes,
                                  stream_of(q)),
             "paia_paged_attention");
}
at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_table, const at::Tensor& lens, std::optional<double> scale,
                           int64_t window, const std::optional<at::Tensor>& k_scale,
                           const std::optional<at::Tensor>& v_scale, const std::optional<at::Tensor>& workspace)
{
    at::Tensor out = at::empty(q.sizes(), q.options());
    paged_attention_run(q, k_cache, v_cache, block_table, lens, scale, window, k_scale, v_scale, out, {}, workspace);
    return out;
}
at::Tensor new_lse(const at::Tensor& q)
{
    return at::empty(q.sizes().slice(0, q.dim() > 0 ? q.dim() - 1 : 0), q.options().dtype(at::kFloat));
}
std::tuple<at::Tensor, at::Tensor> paged_attention_lse(const at::Tensor& q, const at::Tensor& k_cache,
                                                       const at::Tensor& v_cache, const at::Tensor& block_table,
                                                       const at::Tensor& lens, std::optional<double> scale, int64_t window,
                                                       const std::optional<at::Tensor>& k_scale,
                                                       const std::optional<at::Tensor>& v_scale,
                                                       const std::optional<at::Tensor>& workspace)
{
    at::Tensor out = at::empty(q.sizes(), q.options()), lse = new_lse(q);
    paged_attention_run(q, k_cache, v_cache, block_table, lens, scale, window, k_scale, v_scale, out, lse, workspace);
    return {out, lse};
}
void paged_attention_out(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                         const at::Tensor& block_table, const at::Tensor& lens, std::optional<double> scale, int64_t window,
                         const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                         const std::optional<at::Tensor>& workspace, at::Tensor& out)
{
    paged_attention_run(q, k_cache, v_cache, block_table, lens, scale, window, k_scale, v_scale, out, {}, workspace);
}
// On tensors without memory too (tracing): the sizes alone count, so the addresses only have to be ones that the C ABI takes.
int64_t paged_attention_workspace(const at::Tensor& k_cache, int64_t table_width, int64_t B, int64_t T, int64_t num_heads)
{
    paia_kv_cache c = shape_of(k_cache, k_cache);
    c.k = c.v = reinterpret_cast<void*>(16);
    c10::OptionalDeviceGuard g;
    if (k_cache.is_cuda()) g.reset_device(k_cache.device());
    const long long need = paia_paged_attention_workspace(&c, to_int(table_width, "table_width"), to_int(B, "B"),
                                                          to_int(T, "T"), to_int(num_heads, "num_heads"));
    check_rc(need < 0 ? (int)need : 0, "paia_paged_attention_workspace");
    return need;
}

// -------------------------------------------------------------------------------------------------------------
void lora_add_out(const at::Tensor& y, const at::Tensor& x, const at::Tensor& A, const at::Tensor& B, const at::Tensor& ids,
                  const std::optional<at::Tensor>& scaling, at::OptionalIntArrayRef splits,
                  const std::optional<at::Tensor>& workspace, at::Tensor& out)
{
    TORCH_CHECK(A.is_cuda(), "A must be on a GPU, found ", A.device());
    const auto bf16 = [](const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; };
    TORCH_CHECK(A.dim() == 3 && bf16(A) && A.is_contiguous(), "A must be contiguous bfloat16 [adapters, slices * rank, K]");
    TORCH_CHECK(B.dim() == 3 && bf16(B) && B.is_contiguous(), "B must be contiguous bfloat16 [adapters, N, rank]");
    const int64_t L = A.size(0), K = A.size(2), N = B.size(1), R = B.size(2);
    TORCH_CHECK(B.size(0) == L && L > 0, "A and B must hold the same adapters, at least one");
    TORCH_CHECK(bf16(x) && rows_of(x) && x.size(1) == K, "x must be bfloat16 [M, K] with contiguous rows");
    const int64_t M = x.size(0);
    TORCH_CHECK(bf16(y) && rows_of(y) && y.size(0) == M && y.size(1) == N, "y must be bfloat16 [M, N] with contiguous rows");
    TORCH_CHECK(bf16(out) && rows_of(out) && out.sizes() == y.sizes(), "out must be bfloat16 [M, N] with contiguous rows");
    check_index(ids, at::kInt, M, A, "ids");
    on_device_of(A, B, "B");
    on_device_of(A, x, "x");
    on_device_of(A, y, "y");
    on_device_of(A, out, "out");
    int parts[8], slices = 0;
    int64_t sum = 0;
    if (splits.has_value()) {
        TORCH_CHECK(splits->size() >= 1 && splits->size() <= 8, "splits must name 1 to 8 slices");
        for (const int64_t n : *splits) parts[slices++] = to_int(n, "a slice"), sum += n;
    } else {
        parts[slices++] = to_int(N, "N"), sum = N;
    }
    TORCH_CHECK(sum == N, "splits must sum to N (", N, "), found ", sum);
    TORCH_CHECK(A.size(1) == slices * R, "A must hold rank rows (", R, ") for each of ", slices, " slices");
    c10::DeviceGuard g(A.device());
    const long long need = paia_lora_add_workspace(to_int(M, "M"), to_int(K, "K"), to_int(R, "rank"), parts, slices);
    check_rc(need < 0 ? (int)need : 0, "paia_lora_add");
    const Workspace space(workspace, need, A);
    check_rc(paia_lora_add(y.data_ptr(), stride_of(y, 0), x.data_ptr(), stride_of(x, 0), A.data_ptr(), B.data_ptr(),
                           ids.data_ptr(), opt_ptr(scaling, at::kFloat, L, A, "scaling"), out.data_ptr(), stride_of(out, 0),
                           (int)M, (int)K, (int)R, parts, slices, to_int(L, "adapters"), space.data, space.bytes,
                           stream_of(A)),
             "paia_lora_add");
}
at::Tensor lora_add(const at::Tensor& y, const at::Tensor& x, const at::Tensor& A, const at::Tensor& B,
                    const at::Tensor& ids, const std::optional<at::Tensor>& scaling, at::OptionalIntArrayRef splits,
                    const std::optional<at::Tensor>& workspace)
{
    at::Tensor out = at::empty(y.sizes(), y.options());
    lora_add_out(y, x, A, B, ids, scaling, splits, workspace, out);
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

at::Tensor paged_attention_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                const at::Tensor&, std::optional<double>, int64_t, const std::optional<at::Tensor>&,
                                const std::optional<at::Tensor>&, const std::optional<at::Tensor>&)
{
    return at::empty(q.sizes(), q.options());
}
std::tuple<at::Tensor, at::Tensor> paged_attention_lse_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                            const at::Tensor&, const at::Tensor&, std::optional<double>,
                                                            int64_t, const std::optional<at::Tensor>&,
                                                            const std::optional<at::Tensor>&,
                                                            const std::optional<at::Tensor>&)
{
    return {at::empty(q.sizes(), q.options()), new_lse(q)};
}
void paged_attention_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                              std::optional<double>, int64_t, const std::optional<at::Tensor>&,
                              const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, at::Tensor&) {}

at::Tensor lora_add_meta(const at::Tensor& y, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                         const std::optional<at::Tensor>&, at::OptionalIntArrayRef, const std::optional<at::Tensor>&)
{
    return at::empty(y.sizes(), y.options());
}
void lora_add_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                       const std::optional<at::Tensor>&, at::OptionalIntArrayRef, const std::optional<at::Tensor>&,
                       at::Tensor&) {}

}  // namespace

TORCH_LIBRARY_FRAGMENT(paia_gemv, m)
{
    m.def("rope_append(Tensor qkv, Tensor positions, Tensor cos_sin, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, "
          "int num_heads, Tensor? q_norm=None, Tensor? k_norm=None, float eps=1e-6, bool interleaved=False, "
          "Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
    m.def("rope_append_out(Tensor qkv, Tensor positions, Tensor cos_sin, Tensor(a!) k_cache, Tensor(b!) v_cache, "
          "Tensor slots, int num_heads, Tensor? q_norm, Tensor? k_norm, float eps, bool interleaved, Tensor? k_scale, "
          "Tensor? v_scale, Tensor(c!) out) -> ()");
    m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor lens, float? scale=None, "
          "int window=0, Tensor? k_scale=None, Tensor? v_scale=None, Tensor(a!)? workspace=None) -> Tensor");
    m.def("paged_attention_lse(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor lens, "
          "float? scale=None, int window=0, Tensor? k_scale=None, Tensor? v_scale=None, Tensor(a!)? workspace=None) "
          "-> (Tensor, Tensor)");
    m.def("paged_attention_out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor lens, float? scale, "
          "int window, Tensor? k_scale, Tensor? v_scale, Tensor(a!)? workspace, Tensor(b!) out) -> ()");
    m.def("lora_add(Tensor y, Tensor x, Tensor A, Tensor B, Tensor ids, Tensor? scaling=None, int[]? splits=None, "
          "Tensor(a!)? workspace=None) -> Tensor");
    m.def("lora_add_out(Tensor y, Tensor x, Tensor A, Tensor B, Tensor ids, Tensor? scaling, int[]? splits, "
          "Tensor(a!)? workspace, Tensor(b!) out) -> ()");
    m.def("paged_attention_workspace(Tensor k_cache, int table_width, int B, int T, int num_heads) -> int");
}

TORCH_LIBRARY_IMPL(paia_gemv, CUDA, m)
{
    m.impl("rope_append", &rope_append);
    m.impl("rope_append_out", &rope_append_out);
    m.impl("paged_attention", &paged_attention);
    m.impl("paged_attention_lse", &paged_attention_lse);
    m.impl("paged_attention_out", &paged_attention_out);
    m.impl("paged_attention_workspace", &paged_attention_workspace);
    m.impl("lora_add", &lora_add);
    m.impl("lora_add_out", &lora_add_out);
}

TORCH_LIBRARY_IMPL(paia_gemv, Meta, m)
{
    m.impl("rope_append", &rope_append_meta);
    m.impl("rope_append_out", &rope_append_out_meta);
    m.impl("paged_attention", &paged_attention_meta);
    m.impl("paged_attention_lse", &paged_attention_lse_meta);
    m.impl("paged_attention_out", &paged_attention_out_meta);
    m.impl("paged_attention_workspace", &paged_attention_workspace);
    m.impl("lora_add", &lora_add_meta);
    m.impl("lora_add_out", &lora_add_out_meta);
}
