// The paged key-value cache as the kernels see it (paia_kv_cache of the C ABI), and its checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "divisor.h"
#include "gemv_kernel.h"
#include "paia_gemv.h"

namespace paia {

struct CacheView {
    uint8_t *k, *v;
    const float *k_scale, *v_scale;         // fp32 [kv_heads] or null
    int64_t kp, kh, kr, vp, vh, vr;         // strides of page, head and position, in bytes
    int pages, page_size, kv_heads;
    Divisor by_page;                        // by page_size
};

// Fills `c` from the caller's description; false where it is outside the contract.
inline bool cache_view(const paia_kv_cache* d, CacheView* c)
{
    if (d == nullptr || d->pages <= 0 || d->page_size <= 0 || d->kv_heads <= 0 || (d->fp8 != 0 && d->fp8 != 1)) return false;
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return false;
    if (d->k == nullptr || d->v == nullptr || !aligned(d->k, 16) || !aligned(d->v, 16)) return false;
    if (!aligned(d->k_scale, 4) || !aligned(d->v_scale, 4)) return false;
    const int size = d->fp8 ? 1 : 2;
    for (int i = 0; i < 3; ++i)
        if (d->k_strides[i] < 0 || d->v_strides[i] < 0 || (d->k_strides[i] * size) % 16 || (d->v_strides[i] * size) % 16)
            return false;
    c->k = static_cast<uint8_t*>(d->k);
    c->v = static_cast<uint8_t*>(d->v);
    c->k_scale = d->k_scale;
    c->v_scale = d->v_scale;
    c->kp = d->k_strides[0] * size, c->kh = d->k_strides[1] * size, c->kr = d->k_strides[2] * size;
    c->vp = d->v_strides[0] * size, c->vh = d->v_strides[1] * size, c->vr = d->v_strides[2] * size;
    c->pages = d->pages;
    c->page_size = d->page_size;
    c->by_page = Divisor((uint32_t)d->page_size);
    c->kv_heads = d->kv_heads;
    return true;
}

}  // namespace paia
