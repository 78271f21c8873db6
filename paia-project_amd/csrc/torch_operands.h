// Checks and operands that the torch ops around the projections share.
#pragma once
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <optional>

namespace {

inline void check_rc(int rc, const char* what)
{
    TORCH_CHECK(rc == 0, what, " failed with code ", rc, " (-2 bad shape/alignment, >0 hipError_t)");
}

inline void* stream_of(const at::Tensor& t)
{
    return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// Every operand must live on the GPU the kernel runs on: `on` is the tensor whose device counts.
inline void on_device_of(const at::Tensor& on, const at::Tensor& t, const char* name)
{
    TORCH_CHECK(t.device() == on.device(), name, " must be on ", on.device(), ", found ", t.device());
}

// The stride of a dimension as the C ABI takes it: 0 where there is only one element, whose stride may be anything.
inline int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

// The data of an optional operand of the given type and length, null where there is none.
inline const void* opt_ptr(const std::optional<at::Tensor>& t, at::ScalarType type, int64_t n, const at::Tensor& on,
                    const char* name)
{
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->scalar_type() == type && t->is_contiguous() && t->numel() == n, name, " must be a contiguous ",
                at::toString(type), " tensor of ", n, " elements");
    on_device_of(on, *t, name);
    return t->data_ptr();
}

inline int to_int(int64_t v, const char* name)
{
    TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, name, " must fit in 32 bits");
    return (int)v;
}

inline void check_index(const at::Tensor& t, at::ScalarType type, int64_t n, const at::Tensor& on, const char* name)
{
    TORCH_CHECK(t.dim() == 1 && t.scalar_type() == type && t.is_contiguous() && t.numel() == n, name,
                " must be a contiguous ", at::toString(type), " tensor [", n, "]");
    on_device_of(on, t, name);
}

// A call's workspace: the caller's tensor, or memory of torch's allocator for as long as the call is made (its next user on
// this stream comes behind the call's kernels, as with a tensor that goes out of scope).
struct Workspace {
    c10::DataPtr held;
    void* data = nullptr;
    long long bytes = 0;
    Workspace(const std::optional<at::Tensor>& given, long long need, const at::Tensor& on)
    {
        if (given.has_value()) {
            TORCH_CHECK(given->is_contiguous() && (int64_t)given->nbytes() >= need,
                        "workspace must be contiguous and hold ", need, " bytes");
            on_device_of(on, *given, "workspace");
            data = given->data_ptr();
            bytes = (long long)given->nbytes();
        } else if (need > 0) {
            held = c10::hip::HIPCachingAllocator::get()->allocate((size_t)need);
            data = held.get();
            bytes = need;
        }
    }
};

// Rows of contiguous values, any distance apart.
inline bool rows_of(const at::Tensor& t) { return t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1); }

}  // namespace
