// Head norm, position rotation and cache write of a decode step's (or a prompt's) tokens, in one pass over the fused
// projection's output.
//
//   q, k:  x <- x * rsqrt(mean(x^2) + eps) * w      (where a norm weight is given)
//          (a, b) <- (a cos - b sin, b cos + a sin) over the pairs (i, i + rot/2) or (2i, 2i+1) of the first rot dims
//   q -> bf16;  k, v -> the token's slot of the cache, bf16 or e4m3 of value / scale[head]
//
// Few operations per byte: bound by the bytes for a prompt, by latency (one load, one store) for a decode step.
//   * A head is D/16 lanes with two 16-byte pieces each, taken so that a lane holds both halves of its pairs: pieces i and
//     i + rot/16 of the rotating part, or two neighbours. No exchange between lanes but the norm's sum (DPP).
//   * A wave is one token (its position and slot are scalar) and 1024/D heads. All its loads but the cosines (whose address
//     waits for the position) are on their way before the first use: a token waits for memory twice, not four times.
//     8001 tokens of 32 + 16 heads: 39.8 us without that, 35.4 with it (198 MB, 5.6 TB/s; a plain copy of as many bytes
//     reaches 4.9). Two or three groups of heads a wave, which read the cosines once: 36.1; streaming loads or stores: 38.3
//     and 42.2.
// All arithmetic is fp32; each output is rounded once, to its stored type.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemv_kernel.h"
#include "kv_cache.h"
#include "paia_gemv.h"

namespace paia {

struct RopeParams {
    const uint8_t* qkv;
    int64_t row_bytes;
    const int64_t *positions, *slots;
    const float* cos_sin;
    const uint16_t *q_norm, *k_norm;
    uint16_t* q_out;
    CacheView cache;
    uint32_t tokens;
    Divisor by_units;        // by the waves per token
    int context, rotary, heads;
    float eps;
};

__device__ __forceinline__ void unpack8(const u32x4 w, float v[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_to_f32(w[i] & 0xFFFFu);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

// value / scale, clamped to the type's largest (a NaN stays one)
__device__ __forceinline__ float e4m3_clamp(float v, float s)
{
    v = v / s;
    return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}

// Eight values to 16 bytes of bf16 or 8 bytes of e4m3.
template <bool FP8>
__device__ __forceinline__ void store8(uint8_t* p, const float v[8], float s)
{
    if constexpr (FP8) {
        uint2 w;
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = e4m3_clamp(v[i], s);
        int a = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        w.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], a, true);
        a = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
        w.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], a, true);
        *reinterpret_cast<uint2*>(p) = w;
    } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<u32x4*>(p) = w;
    }
}

constexpr int kRopeBlock = 256;
// A launch has less than 2^32 threads: tokens beyond kRopeMaxBlocks blocks go into a further one.
constexpr int64_t kRopeMaxBlocks = 1 << 23;

// PAIRS: pairs (2i, 2i+1) instead of halves; NORM: at least one norm weight is given
template <int D, bool FP8, bool PAIRS, bool NORM>
__global__ void __launch_bounds__(kRopeBlock) rope_append_kernel(const RopeParams p)
{
    constexpr int kLanes = D / 16, kHeads = kWave / kLanes;      // lanes of a head, heads of a wave
    const uint32_t w = blockIdx.x * (kRopeBlock / kWave) + (uint32_t)wave_id();
    const uint32_t m = p.by_units.of(w);
    if (m >= p.tokens) return;
    const int hkv = p.cache.kv_heads, all = p.heads + 2 * hkv;
    // lanes past the last head repeat it up to the stores (a branch here would keep the compiler from moving loads up)
    const int asked = (int)(w - m * p.by_units.d) * kHeads + lane_id() / kLanes, i = lane_id() % kLanes;
    const int head = min(asked, all - 1);
    const bool is_q = head < p.heads, is_v = head >= p.heads + hkv;
    const int h = is_q ? 0 : head - p.heads - (is_v ? hkv : 0);      // of the cache
    const int turning = p.rotary / 16;       // lanes of a head whose pieces turn
    const int c0 = !PAIRS && i < turning ? i : 2 * i, c1 = !PAIRS && i < turning ? i + turning : 2 * i + 1;

    const int64_t pos = p.positions[m], slot = p.slots[m];
    const uint8_t* src = p.qkv + (int64_t)m * p.row_bytes + (int64_t)head * (2 * D);
    const u32x4 r0 = *reinterpret_cast<const u32x4*>(src + 16 * c0);
    const u32x4 r1 = *reinterpret_cast<const u32x4*>(src + 16 * c1);
    const uint16_t* weight = NORM && !is_v ? (is_q ? p.q_norm : p.k_norm) : nullptr;
    u32x4 w0 = {0, 0, 0, 0}, w1 = {0, 0, 0, 0};
    if (weight != nullptr) {
        w0 = *reinterpret_cast<const u32x4*>(weight + 8 * c0);
        w1 = *reinterpret_cast<const u32x4*>(weight + 8 * c1);
    }
    const float* scale = is_v ? p.cache.v_scale : p.cache.k_scale;
    const float factor = FP8 && scale != nullptr ? scale[h] : 1.0f;
    const int64_t page = slot >> 31 == 0 ? (int64_t)p.cache.by_page.of((uint32_t)slot) : slot / p.cache.page_size;
    const int64_t at = slot - page * p.cache.page_size;
    const bool bad = pos < 0 || pos >= p.context;
    const float* cs = p.cos_sin + (bad ? 0 : pos) * p.rotary + 8 * (i < turning ? i : 0);
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(cs + 4 * e), y = *reinterpret_cast<const f32x4*>(cs + p.rotary / 2 + 4 * e);
#pragma unroll
        for (int j = 0; j < 4; ++j) c[4 * e + j] = bad ? __builtin_nanf("") : x[j], s[4 * e + j] = y[j];
    }
    // Named here, or the compiler moves these loads into the branches that use them, behind the first wait (prompt 39.5 us).
    asm volatile("" ::"v"(c[0]), "v"(c[4]), "v"(s[0]), "v"(s[4]));
    if constexpr (FP8) asm volatile("" ::"v"(factor));

    float a[8], b[8];
    unpack8(r0, a);
    unpack8(r1, b);
    if constexpr (NORM) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(a[e], a[e], __builtin_fmaf(b[e], b[e], ss));
        ss = quad_sum(ss);
        if constexpr (kLanes >= 8) ss += dpp_f32<0x141>(ss);    // row_half_mirror: the other quad of eight lanes
        if constexpr (kLanes >= 16) ss += dpp_f32<0x140>(ss);   // row_mirror: the other half of the row
        if (weight != nullptr) {
            const float r = rsqrtf(ss * (1.0f / D) + p.eps);
            float wa[8], wb[8];
            unpack8(w0, wa);
            unpack8(w1, wb);
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = a[e] * r * wa[e], b[e] = b[e] * r * wb[e];
        }
    }
    if (i < turning && !is_v) {
        if constexpr (PAIRS) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float u = a[2 * e], v = a[2 * e + 1], x = b[2 * e], y = b[2 * e + 1];
                a[2 * e] = u * c[e] - v * s[e], a[2 * e + 1] = v * c[e] + u * s[e];
                b[2 * e] = x * c[4 + e] - y * s[4 + e], b[2 * e + 1] = y * c[4 + e] + x * s[4 + e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float u = a[e], v = b[e];
                a[e] = u * c[e] - v * s[e], b[e] = v * c[e] + u * s[e];
            }
        }
    }
    if (asked >= all) return;
    if (is_q) {
        uint8_t* q = reinterpret_cast<uint8_t*>(p.q_out) + ((int64_t)m * p.heads + head) * (2 * D);
        store8<false>(q + 16 * c0, a, 1.0f);
        store8<false>(q + 16 * c1, b, 1.0f);
        return;
    }
    if (slot < 0 || slot >= (int64_t)p.cache.pages * p.cache.page_size) return;
    uint8_t* dst = is_v ? p.cache.v + page * p.cache.vp + h * p.cache.vh + at * p.cache.vr
                        : p.cache.k + page * p.cache.kp + h * p.cache.kh + at * p.cache.kr;
    constexpr int kPiece = FP8 ? 8 : 16;
    store8<FP8>(dst + kPiece * c0, a, factor);
    store8<FP8>(dst + kPiece * c1, b, factor);
}

template <int D, bool FP8>
int launch_rope(RopeParams p, bool pairs, int64_t M, hipStream_t st)
{
    constexpr int kHeads = kWave / (D / 16), kWaves = kRopeBlock / kWave;
    const uint32_t units = ((uint32_t)p.heads + 2u * (uint32_t)p.cache.kv_heads + kHeads - 1) / kHeads;    // waves a token
    p.by_units = Divisor(units);
    const bool norm = p.q_norm != nullptr || p.k_norm != nullptr;
    const int64_t step = kRopeMaxBlocks * kWaves / units;
    for (int64_t m = 0; m < M; m += step) {
        RopeParams s = p;
        s.tokens = (uint32_t)(M - m < step ? M - m : step);
        s.qkv += m * p.row_bytes;
        s.positions += m;
        s.slots += m;
        s.q_out += m * p.heads * (int64_t)D;
        const uint32_t blocks = (uint32_t)(((int64_t)s.tokens * units + kWaves - 1) / kWaves);
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kRopeBlock), 0, st, s); };
        if (pairs) norm ? go(rope_append_kernel<D, FP8, true, true>) : go(rope_append_kernel<D, FP8, true, false>);
        else norm ? go(rope_append_kernel<D, FP8, false, true>) : go(rope_append_kernel<D, FP8, false, false>);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    }
    return 0;
}
}  // namespace paia

extern "C" {

int paia_rope_append(const void* qkv, long long qkv_stride, const void* positions, const void* cos_sin, int context,
                     int rotary, int interleaved, const void* q_norm, const void* k_norm, float eps, const void* slots,
                     const paia_kv_cache* cache, void* q_out, int M, int heads, void* stream)
{
    using namespace paia;
    RopeParams p;
    if (!cache_view(cache, &p.cache) || M < 0 || heads <= 0 || heads > (1 << 20) || cache->kv_heads > (1 << 20)) return -2;
    if (context <= 0 || rotary <= 0 || rotary % 16 || rotary > cache->head_dim) return -2;
    if (M == 0) return 0;
    if (qkv == nullptr || positions == nullptr || cos_sin == nullptr || slots == nullptr || q_out == nullptr) return -2;
    if (q_out == qkv || !aligned(qkv, 16) || !aligned(cos_sin, 16) || !aligned(q_out, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16) ||
        !aligned(positions, 8) || !aligned(slots, 8) || qkv_stride % 8)
        return -2;
    p.qkv = static_cast<const uint8_t*>(qkv);
    p.row_bytes = qkv_stride * 2;
    p.positions = static_cast<const int64_t*>(positions);
    p.slots = static_cast<const int64_t*>(slots);
    p.cos_sin = static_cast<const float*>(cos_sin);
    p.q_norm = static_cast<const uint16_t*>(q_norm);
    p.k_norm = static_cast<const uint16_t*>(k_norm);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.context = context, p.rotary = rotary, p.heads = heads, p.eps = eps;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool pairs = interleaved != 0;
    switch (cache->head_dim * 2 + cache->fp8) {
    case 128: return launch_rope<64, false>(p, pairs, M, st);
    case 129: return launch_rope<64, true>(p, pairs, M, st);
    case 256: return launch_rope<128, false>(p, pairs, M, st);
    case 257: return launch_rope<128, true>(p, pairs, M, st);
    case 512: return launch_rope<256, false>(p, pairs, M, st);
    default: return launch_rope<256, true>(p, pairs, M, st);
    }
}

}  // extern "C"
