// Residual and norms between the halves of a layer.
//
//   y = x[m], or sum_j weights[m, j] x[m, j]            (a token's experts)
//   y = y rsqrt(mean(y^2) + eps) post                   (a norm behind the block, where `post` is given)
//   r = residual[m] + scale gate y                      (gate a factor per channel, or per token and channel)
//   h = r rsqrt(mean(r^2) + eps) norm
//
// fp32 throughout; h is made of r as it is in fp32, and both are rounded once on their way out. One pass: a block has a row, its
// threads hold the row's values in registers from the first load to the last store. Bound by bytes where there are many rows
// and by latency (the loads, then one or two sums over the block) where there is one: every load is on its way ahead of the
// first sum. Measured: 8001 tokens of two pairs of 4096 56 to 58 us (5.7 TB/s; a copy moves 4.9), 13 tokens of eight pairs of 3584 with
// a norm behind the block 5.0, one token 2.7, of which the launch is 1.6. Four pieces a thread with pairs (D beyond 16384) keep 46 and more
// registers in memory: 2000 tokens of two pairs of 18944 143 us (2.6 TB/s), of 16384 68 (4.8), of 18944 without pairs 58 (5.2).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gemv_kernel.h"
#include "paia_gemv.h"

namespace paia {

struct AddNormParams {
    const uint16_t *x, *gate, *post, *norm;
    const void* residual;                // bf16, or fp32
    const float* weights;                // [M][pairs]
    uint16_t* h;
    void* r;                             // of the residual's type, or null
    int64_t x_stride, pair_stride, residual_stride, gate_stride, h_stride, r_stride;
    int pieces, pairs;                   // 8-value pieces of a row; 0: x has no pairs
    float scale, eps, inverse, plus;     // inverse: 1 / D; plus: 1 where the norms' weights are kept less 1
};

constexpr int kNormMaxWaves = 16;

// A block's sum of one value a thread, the same in every thread: the waves' sums added in order.
__device__ __forceinline__ float block_sum(float v, float* part, int waves)
{
    v = wave_sum(v);
    if (waves == 1) return v;
    if (lane_id() == 0) part[wave_id()] = v;
    __syncthreads();
    float sum = part[0];
    for (int w = 1; w < waves; ++w) sum += part[w];
    return sum;
}

__device__ __forceinline__ void unpack8(const u32x4 v, float f[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
}
__device__ __forceinline__ u32x4 pack8(const float f[8])
{
    return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
}

// NV: 16-byte pieces of a row that a thread holds. R32: the residual is fp32. PAIRS: x has pairs.
template <int NV, bool R32, bool PAIRS>
__global__ void __launch_bounds__(1024) add_norm_kernel(const AddNormParams p)
{
    __shared__ float part[2][kNormMaxWaves];
    const int64_t m = blockIdx.x;
    const int waves = (int)blockDim.x / kWave;
    const u32x4 none = {0, 0, 0, 0};
    const auto load = [&](const uint16_t* row, int c) { return c < p.pieces ? reinterpret_cast<const u32x4*>(row)[c] : none; };

    // the loads that nothing has to be known for
    constexpr int kAhead = PAIRS ? 8 / NV : 1;       // rows of x whose loads are on their way together
    const int rows = PAIRS ? p.pairs : 1;
    const uint16_t* x = p.x + m * p.x_stride;
    u32x4 in[kAhead][NV], gate[NV], post[NV], norm[NV], res[NV][R32 ? 2 : 1];
    float w[kAhead];
    const auto load_rows = [&](int j) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (j + a < rows) {
                w[a] = PAIRS ? p.weights[m * p.pairs + j + a] : 1.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    in[a][i] = load(x + (j + a) * p.pair_stride, (int)(threadIdx.x + i * blockDim.x));
            }
    };
    load_rows(0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (int)(threadIdx.x + i * blockDim.x);
        res[i][0] = none;
        if constexpr (R32) {
            res[i][1] = none;
            const u32x4* row = reinterpret_cast<const u32x4*>(static_cast<const float*>(p.residual) + m * p.residual_stride);
            if (p.residual != nullptr && c < p.pieces) res[i][0] = row[2 * c], res[i][1] = row[2 * c + 1];
        } else if (p.residual != nullptr) {
            res[i][0] = load(static_cast<const uint16_t*>(p.residual) + m * p.residual_stride, c);
        }
        gate[i] = p.gate != nullptr ? load(p.gate + m * p.gate_stride, c) : none;
        post[i] = p.post != nullptr ? load(p.post, c) : none;
        norm[i] = load(p.norm, c);
    }

    float y[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = 0.0f;
    for (int j = 0;;) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (j + a >= rows || w[a] == 0.0f) continue;     // a pair of weight 0 adds nothing, whatever its row holds
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[8];
                unpack8(in[a][i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] = __builtin_fmaf(w[a], f[e], y[i][e]);
            }
        }
        j += kAhead;
        if (j >= rows) break;
        load_rows(j);
    }
    const auto squares = [&]() {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __builtin_fmaf(y[i][e], y[i][e], s);
        return s;
    };
    if (p.post != nullptr) {
        const float by = 1.0f / sqrtf(block_sum(squares(), part[0], waves) * p.inverse + p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[8];
            unpack8(post[i], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * by * (f[e] + p.plus);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (int)(threadIdx.x + i * blockDim.x);
        float f[8];
        if (p.gate != nullptr) {
            unpack8(gate[i], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] *= f[e];
        }
        if constexpr (R32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(res[i][e / 4][e % 4]);
        } else {
            unpack8(res[i][0], f);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = p.residual != nullptr ? __builtin_fmaf(p.scale, y[i][e], f[e]) : p.scale * y[i][e];
        if (c >= p.pieces) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = 0.0f;
        } else if (p.r != nullptr) {
            if constexpr (R32) {
                f32x4* row = reinterpret_cast<f32x4*>(static_cast<float*>(p.r) + m * p.r_stride);
                row[2 * c] = f32x4{y[i][0], y[i][1], y[i][2], y[i][3]};
                row[2 * c + 1] = f32x4{y[i][4], y[i][5], y[i][6], y[i][7]};
            } else {
                reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.r) + m * p.r_stride)[c] = pack8(y[i]);
            }
        }
    }
    const float by = 1.0f / sqrtf(block_sum(squares(), part[1], waves) * p.inverse + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (int)(threadIdx.x + i * blockDim.x);
        if (c >= p.pieces) continue;
        float f[8];
        unpack8(norm[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = y[i][e] * by * (f[e] + p.plus);
        reinterpret_cast<u32x4*>(p.h + m * p.h_stride)[c] = pack8(f);
    }
}

}  // namespace paia

extern "C" {

int paia_add_norm(const void* x, long long x_stride, const void* weights, long long pair_stride, int pairs,
                  const void* residual, long long residual_stride, int residual_fp32, const void* post_norm,
                  const void* gate, long long gate_stride, float scale, const void* norm, int plus_one, float eps, void* out,
                  long long out_stride, void* residual_out, long long residual_out_stride, int M, int D, void* stream)
{
    using namespace paia;
    if (M < 0 || D <= 0 || D % 8 || D > 32768 || pairs < 0 || (residual_fp32 != 0 && residual_fp32 != 1) ||
        (plus_one != 0 && plus_one != 1) || !(eps >= 0.0f))
        return -2;
    if (M == 0) return 0;
    if (x == nullptr || norm == nullptr || out == nullptr || (pairs > 0) != (weights != nullptr)) return -2;
    for (const void* ptr : {x, residual, post_norm, gate, norm, static_cast<const void*>(out),
                            static_cast<const void*>(residual_out)})
        if (!aligned(ptr, 16)) return -2;
    if (!aligned(weights, 4)) return -2;
    for (const long long s : {x_stride, pair_stride, residual_stride, gate_stride, out_stride, residual_out_stride})
        if (s < 0 || s % 8) return -2;
    if (M > 1 && (out_stride < D || (residual_out != nullptr && residual_out_stride < D))) return -2;
    AddNormParams p{};
    p.post = static_cast<const uint16_t*>(post_norm);
    p.norm = static_cast<const uint16_t*>(norm);
    p.x_stride = x_stride, p.pair_stride = pair_stride, p.residual_stride = residual_stride, p.gate_stride = gate_stride;
    p.h_stride = out_stride, p.r_stride = residual_out_stride;
    p.pieces = D / 8, p.pairs = pairs;
    p.scale = scale, p.eps = eps, p.inverse = 1.0f / (float)D, p.plus = plus_one ? 1.0f : 0.0f;
    const size_t width = residual_fp32 ? 4 : 2;
    // threads: one piece each up to 1024 (two each, us: 16 tokens of two pairs of 4096 3.14 -> 3.44, 8001 56.4 -> 58.2; 2000 tokens
    // of 8192 the same)
    int threads = kWave;
    while (threads < 1024 && threads < p.pieces) threads *= 2;
    const int nv = (p.pieces + threads - 1) / threads;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int rows = 1 << 21;                    // of a launch: a grid has fewer than 2^32 threads
    for (int m = 0; m < M; m += rows) {
        p.x = static_cast<const uint16_t*>(x) + m * x_stride;
        p.weights = weights != nullptr ? static_cast<const float*>(weights) + (int64_t)m * pairs : nullptr;
        p.residual = residual != nullptr ? static_cast<const uint8_t*>(residual) + m * residual_stride * width : nullptr;
        p.gate = gate != nullptr ? static_cast<const uint16_t*>(gate) + m * gate_stride : nullptr;
        p.h = static_cast<uint16_t*>(out) + m * out_stride;
        p.r = residual_out != nullptr ? static_cast<uint8_t*>(residual_out) + m * residual_out_stride * width : nullptr;
        const dim3 grid((uint32_t)(M - m < rows ? M - m : rows)), block((uint32_t)threads);
        auto go = [&](auto narrow, auto wide) { hipLaunchKernelGGL(residual_fp32 ? wide : narrow, grid, block, 0, st, p); };
        const auto go_nv = [&](auto n) {
            constexpr int NV = decltype(n)::value;
            if (pairs > 0) go(add_norm_kernel<NV, false, true>, add_norm_kernel<NV, true, true>);
            else go(add_norm_kernel<NV, false, false>, add_norm_kernel<NV, true, false>);
        };
        if (nv == 1) go_nv(std::integral_constant<int, 1>{});
        else if (nv == 2) go_nv(std::integral_constant<int, 2>{});
        else go_nv(std::integral_constant<int, 4>{});
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
        if (M - m <= rows) break;
    }
    return 0;
}

}  // extern "C"
