// Each token's experts, and the pairs of token and expert in the experts' order.
//
//   key[m, e] = logits[m, e]                     softmax, whose order is that of the logits
//             = sigmoid(logits[m, e]) + bias[e]  sigmoid; the bias decides the choice, not the weight
//   ids[m, :] = the k experts of the largest keys, the lower index first among equal ones
//   weights[m, j] = scale * s(m, ids[m, j]) (/ their sum),  s = softmax over the row's experts, or sigmoid
//
// Experts whose logit (or bias) is -inf or NaN are closed to the token; where fewer than k are open the rest of ids is -1, of
// weight 0. A wave has a token, a lane every 64th expert of it: the largest key comes of one DPP maximum, its lowest index of
// the lanes' ballots, k times; a bf16 logit and its index are one key (8001 tokens, eight of 256 22.0 -> 19.4 us). Keys that are
// computed (sigmoid), and all weights, are so in 64 bits: neighbouring keys decide which experts run, and there are few of them.
//
// order: the pairs m * k + j sorted by expert, in their own order within one, those without an expert at the end. A block counts
// its pairs by wave and expert in LDS and gives each its place: the lanes with the same expert find each other by one ballot
// a bit of the id. Few tokens are one launch of one block. Otherwise each block leaves its counts in the workspace and the second
// launch's blocks add up those before their own (integers: the order of sums does not matter, nothing is atomic across blocks).
// Bound by its dependent steps, k maxima and two walks over the pairs; two tokens a wave overlap theirs. Measured: one token, eight
// of 64 experts 4.0 us; 61 tokens, six of 160 by sigmoid 13.1, 8.6 of it the choice (16 tokens a block, four waves a SIMD with their
// sigmoids in 64 bits on 4 of 256 CUs); 8001 tokens, eight of 256 19.4, 9 of it the second launch. The order alone, from ids, of these:
// 3.3, 7.0 and 12.4.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemv_kernel.h"
#include "paia_gemv.h"

namespace paia {

constexpr int kRouteBlock = 1024, kRouteWaves = kRouteBlock / kWave;
constexpr int kRouteExperts = 1024;      // experts at most: a thread each in the scan
constexpr int kRouteBlocks = 256;        // blocks at most that share the tokens
constexpr int kRouteTokens = 32;         // tokens up to which one block does all of it (61 at a block: 11.8 us, in two launches 9.1)

struct RouteParams {
    const void* logits;                  // bf16 or fp32 [M][E]
    const float* bias;                   // [E] or null
    int32_t *ids, *order, *offsets;
    float* weights;
    int32_t* counts;                     // workspace: [block][count_stride], E + 1 of them used
    int64_t stride;                      // elements
    int M, E, k, tokens;                 // tokens: of a block
    int count_stride;                    // E + 1 rounded up to 4
    int id_bits;
    bool fp32, renormalize;
    float scale;
};

// Bits whose order is that of the values, 0 below all of them; -0 counts as 0.
__device__ __forceinline__ uint32_t sortable(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t sortable(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// The sum over the wave in every lane, by the steps of wave_sum.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_add(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROW_MASK, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROW_MASK, 0xF, false);
    return v + __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_add(double v)
{
    v = dpp_add<0xB1, 0xF>(v);
    v = dpp_add<0x4E, 0xF>(v);
    v = dpp_add<0x124, 0xF>(v);
    v = dpp_add<0x128, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    v = dpp_add<0x143, 0xC>(v);
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// The largest key of the wave: its lowest index (lane + 64 i), -1 where all keys are 0. The key found is set to 0.
template <int NE>
__device__ __forceinline__ int take_largest(uint32_t (&key)[NE])
{
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) most = max(most, key[i]);
    most = wave_max_u32(most);
    int at = -1;
#pragma unroll
    for (int i = NE - 1; i >= 0; --i) {
        const uint64_t here = __ballot(key[i] == most);
        if (here != 0) at = 64 * i + __builtin_ctzll(here);
    }
    if (most == 0) at = -1;
#pragma unroll
    for (int i = 0; i < NE; ++i)
        if (at == 64 * i + lane_id()) key[i] = 0;
    return at;
}
template <int NE>
__device__ __forceinline__ int take_largest(uint64_t (&key)[NE])
{
    uint32_t high = 0, low = 0;          // open keys are sums above -2^1024: their upper halves are not 0
#pragma unroll
    for (int i = 0; i < NE; ++i) high = max(high, (uint32_t)(key[i] >> 32));
    high = wave_max_u32(high);
#pragma unroll
    for (int i = 0; i < NE; ++i)
        if ((uint32_t)(key[i] >> 32) == high) low = max(low, (uint32_t)key[i]);
    low = wave_max_u32(low);
    const uint64_t most = (uint64_t)high << 32 | low;
    int at = -1;
#pragma unroll
    for (int i = NE - 1; i >= 0; --i) {
        const uint64_t here = __ballot(key[i] == most);
        if (here != 0) at = 64 * i + __builtin_ctzll(here);
    }
    if (high == 0) at = -1;
#pragma unroll
    for (int i = 0; i < NE; ++i)
        if (at == 64 * i + lane_id()) key[i] = 0;
    return at;
}

// A bf16 logit's 16 sortable bits above its index from the far end: the largest is the largest logit at its lowest index, all that
// a choice by softmax needs to know. 0: closed.
__device__ __forceinline__ uint32_t packed_key(uint32_t b, int e)
{
    if ((b & 0x7FFFu) > 0x7F80u || b == 0xFF80u) return 0;       // NaN, -inf
    if (b == 0x8000u) b = 0;
    return (b >> 15 ? ~b & 0xFFFFu : b | 0x8000u) << 16 | (0xFFFFu - (uint32_t)e);
}
__device__ __forceinline__ float packed_logit(uint32_t key)
{
    return __uint_as_float(key >> 31 ? (key & 0x7FFF0000u) : ~key & 0xFFFF0000u);
}

// The choices of T tokens m, m + step, .. by one wave, whose chains of dependent steps overlap. The lanes j < k write them.
template <int NE, bool SIGMOID, bool PACKED, int T>
__device__ __forceinline__ void choose(const RouteParams& p, int m, int step)
{
    const int lane = lane_id();
    float v[T][NE];
#pragma unroll
    for (int u = 0; u < T; ++u)
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = lane + 64 * i;
            v[u][i] = -__builtin_inff();
            if (e < p.E) {
                const int64_t at = (int64_t)(m + u * step) * p.stride + e;
                v[u][i] = !PACKED && p.fp32 ? static_cast<const float*>(p.logits)[at] : bf16_to_f32(static_cast<const uint16_t*>(p.logits)[at]);
            }
        }
    int id[T];
    float top[T], mine[T];               // the largest logit, and that of the lane's expert
#pragma unroll
    for (int u = 0; u < T; ++u) id[u] = -1, top[u] = mine[u] = 0.0f;
    if constexpr (PACKED) {
        uint32_t key[T][NE], first[T], own[T];
#pragma unroll
        for (int u = 0; u < T; ++u) {
            first[u] = own[u] = 0;
#pragma unroll
            for (int i = 0; i < NE; ++i) key[u][i] = packed_key(__float_as_uint(v[u][i]) >> 16, lane + 64 * i);
        }
        for (int j = 0; j < p.k; ++j) {
#pragma unroll
            for (int u = 0; u < T; ++u) {
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < NE; ++i) most = max(most, key[u][i]);
                most = wave_max_u32(most);
#pragma unroll
                for (int i = 0; i < NE; ++i) key[u][i] = key[u][i] == most ? 0u : key[u][i];
                if (j == 0) first[u] = most;
                if (lane == j) own[u] = most;
            }
        }
#pragma unroll
        for (int u = 0; u < T; ++u)
            if (own[u] != 0) id[u] = (int)(0xFFFFu - (own[u] & 0xFFFFu)), mine[u] = packed_logit(own[u]);
#pragma unroll
        for (int u = 0; u < T; ++u)
            if (first[u] != 0) top[u] = packed_logit(first[u]);
    } else {
        using Key = typename std::conditional<SIGMOID, uint64_t, uint32_t>::type;
        Key key[T][NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            double b = 0.0;
            if constexpr (SIGMOID)
                if (p.bias != nullptr && lane + 64 * i < p.E) b = (double)p.bias[lane + 64 * i];
#pragma unroll
            for (int u = 0; u < T; ++u) {
                const bool open = v[u][i] > -__builtin_inff();
                if constexpr (SIGMOID) {
                    key[u][i] = open && b > -__builtin_inf() ? sortable(1.0 / (1.0 + exp(-(double)v[u][i])) + b) : 0;
                } else {
                    key[u][i] = open ? sortable(v[u][i]) : 0;
                }
            }
        }
        for (int j = 0; j < p.k; ++j) {
#pragma unroll
            for (int u = 0; u < T; ++u) {
                const int e = take_largest<NE>(key[u]);
                float logit = 0.0f;
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (e >> 6 == i) logit = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v[u][i]), e & 63));
                if (j == 0) top[u] = logit;
                if (lane == j) id[u] = e, mine[u] = logit;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < T; ++u) {
        double w = 0.0, all = 1.0;
        if constexpr (SIGMOID) {
            if (id[u] >= 0) w = 1.0 / (1.0 + exp(-(double)mine[u]));
            if (p.renormalize) all = wave_add(w);
        } else {
            if (id[u] >= 0) w = exp((double)mine[u] - (double)top[u]);
            if (p.renormalize) {
                all = wave_add(w);
            } else {
                all = 0.0;
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (v[u][i] > -__builtin_inff()) all += exp((double)v[u][i] - (double)top[u]);
                all = wave_add(all);
            }
        }
        if (lane < p.k) {
            const int at = (m + u * step) * p.k + lane;
            p.ids[at] = id[u];
            p.weights[at] = (float)(all > 0.0 || all != all ? w / all * (double)p.scale : 0.0);
        }
    }
}

__device__ __forceinline__ int inclusive(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// Counts or places of a wave's pairs by expert, 64 at a time in their order. at[e]: the count so far, or the next place.
struct SortSpace {
    int32_t at[kRouteWaves][kRouteExperts + 1];
    int32_t sums[kRouteWaves];
};
template <bool PLACE>
__device__ __forceinline__ void walk(const RouteParams& p, int32_t* at, int first, int last)
{
    const int lane = lane_id();
    for (int q0 = first; q0 < last; q0 += kWave) {
        const int q = q0 + lane;
        const bool in = q < last;
        int id = in ? p.ids[q] : -1;
        if ((uint32_t)id >= (uint32_t)p.E) id = p.E;
        uint64_t same = __ballot(in);
        for (int b = 0; b < p.id_bits; ++b) {
            const uint64_t set = __ballot(id >> b & 1);
            same &= id >> b & 1 ? set : ~set;
        }
        if (in) {
            const int before = __popcll(same & ((1ull << lane) - 1)), base = at[id];
            if (PLACE) p.order[base + before] = q;
            wave_lds_order();
            if (before == 0) at[id] = base + __popcll(same);
        }
        wave_lds_order();
    }
}

// An exclusive scan over the block's threads; total in every thread.
__device__ __forceinline__ int block_scan(int v, int32_t* sums, int* total)
{
    const int upto = inclusive(v);
    if (lane_id() == 63) sums[wave_id()] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) {
        before += w < wave_id() ? sums[w] : 0;
        all += sums[w];
    }
    *total = all;
    return before + upto - v;
}

// A block's pairs [first, last) by wave: each wave takes a range of whole 64s.
__device__ __forceinline__ void wave_range(int first, int last, int* from, int* to)
{
    const int steps = (last - first + kWave - 1) / kWave, wave = wave_id();
    *from = first + steps * wave / kRouteWaves * kWave;
    *to = min(last, first + steps * (wave + 1) / kRouteWaves * kWave);
}

// ONE: the only block, which does the order too. SELECT: choose the experts first (else ids are given).
template <int NE, bool SIGMOID, bool SELECT, bool ONE>
__global__ void __launch_bounds__(kRouteBlock) route_kernel(const RouteParams p)
{
    __shared__ SortSpace s;
    const int wave = wave_id(), t = (int)threadIdx.x;
    const int m0 = (int)blockIdx.x * p.tokens, m1 = min(p.M, m0 + p.tokens);
    if constexpr (SELECT) {
        const auto all = [&](auto packed) __attribute__((always_inline)) {
            constexpr bool PACKED = decltype(packed)::value;
            int m = m0 + wave;
            if constexpr (NE <= 4)
                for (; m + kRouteWaves < m1; m += 2 * kRouteWaves) choose<NE, SIGMOID, PACKED, 2>(p, m, kRouteWaves);
            for (; m < m1; m += kRouteWaves) choose<NE, SIGMOID, PACKED, 1>(p, m, kRouteWaves);
        };
        if (SIGMOID || p.fp32) all(std::false_type{});
        else all(std::bool_constant<!SIGMOID>{});
    }
    for (int e = t; e <= p.E; e += kRouteBlock)
#pragma unroll
        for (int w = 0; w < kRouteWaves; ++w) s.at[w][e] = 0;
    __threadfence_block();
    __syncthreads();
    int from, to;
    wave_range(m0 * p.k, m1 * p.k, &from, &to);
    walk<false>(p, s.at[wave], from, to);
    __syncthreads();
    if constexpr (!ONE) {
        for (int e = t; e < p.count_stride; e += kRouteBlock) {
            int sum = 0;
            if (e <= p.E)
#pragma unroll
                for (int w = 0; w < kRouteWaves; ++w) sum += s.at[w][e];
            p.counts[(int64_t)blockIdx.x * p.count_stride + e] = sum;
        }
    } else {
        int own = 0, total;
        if (t < p.E)
#pragma unroll
            for (int w = 0; w < kRouteWaves; ++w) own += s.at[w][t];
        int at = block_scan(own, s.sums, &total);
        const auto places = [&](int e, int place) {
#pragma unroll
            for (int w = 0; w < kRouteWaves; ++w) {
                const int n = s.at[w][e];
                s.at[w][e] = place;
                place += n;
            }
        };
        if (t < p.E) p.offsets[t] = at, places(t, at);
        if (t == 0) p.offsets[p.E] = total, places(p.E, total);
        __syncthreads();
        walk<true>(p, s.at[wave], from, to);
    }
}

// The second launch: block b's places follow from all blocks' counts, four experts a thread and load; where there are fewer
// such quads than threads, groups of threads share the blocks.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__global__ void __launch_bounds__(kRouteBlock) route_order_kernel(const RouteParams p)
{
    __shared__ SortSpace s;
    __shared__ i32x4 sum[2][kRouteBlock];            // [before this block, in all][group][quad]
    const int wave = wave_id(), t = (int)threadIdx.x, bins = p.E + 1;
    const int m0 = (int)blockIdx.x * p.tokens, m1 = min(p.M, m0 + p.tokens);
    const int quads = p.count_stride / 4, groups = min(kRouteBlock / quads, 16), group = t / quads, quad = t - group * quads;
    i32x4 before = {0, 0, 0, 0}, all = {0, 0, 0, 0};
    if (group < groups) {
        const i32x4* counts = reinterpret_cast<const i32x4*>(p.counts) + quad;
        const int last = (int)gridDim.x - 1, own = (int)blockIdx.x;
        constexpr int kAhead = 8;
        for (int b = group; b <= last; b += kAhead * groups) {
            i32x4 n[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) n[i] = counts[(int64_t)min(b + i * groups, last) * quads];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (b + i * groups <= last) all += n[i];
                if (b + i * groups < own) before += n[i];
            }
        }
        sum[0][t] = before, sum[1][t] = all;
    }
    for (int b = t; b < bins; b += kRouteBlock)
#pragma unroll
        for (int w = 0; w < kRouteWaves; ++w) s.at[w][b] = 0;
    __syncthreads();
    int from, to;
    wave_range(m0 * p.k, m1 * p.k, &from, &to);
    walk<false>(p, s.at[wave], from, to);
    const auto total_of = [&](int what, int bin) {
        int n = 0;
        for (int g = 0; g < groups; ++g) n += reinterpret_cast<const int32_t*>(sum[what])[g * p.count_stride + bin];
        return n;
    };
    int total;
    const int at = block_scan(t < p.E ? total_of(1, t) : 0, s.sums, &total);
    __syncthreads();
    const auto places = [&](int bin, int place) {
#pragma unroll
        for (int w = 0; w < kRouteWaves; ++w) {
            const int n = s.at[w][bin];
            s.at[w][bin] = place;
            place += n;
        }
    };
    if (t < p.E) {
        if (blockIdx.x == 0) p.offsets[t] = at;
        places(t, at + total_of(0, t));
    }
    if (t == 0) {
        if (blockIdx.x == 0) p.offsets[p.E] = total;
        places(p.E, total + total_of(0, p.E));
    }
    __syncthreads();
    walk<true>(p, s.at[wave], from, to);
}

// Tokens that a block takes, and the blocks.
static int route_blocks(int M, int* tokens)
{
    *tokens = M <= kRouteTokens ? M : (M + kRouteBlocks - 1) / kRouteBlocks;
    if (M > kRouteTokens && *tokens < kRouteWaves) *tokens = kRouteWaves;
    return (M + *tokens - 1) / *tokens;
}
static bool route_sizes(int M, int E, int k)
{
    return M >= 0 && E > 0 && E <= kRouteExperts && k > 0 && k <= kWave && (int64_t)M * k < 1 << 26;
}
static int64_t route_workspace(int M, int E)
{
    int tokens;
    return M <= kRouteTokens ? 0 : (int64_t)route_blocks(M, &tokens) * ((E + 4) / 4 * 4) * (int64_t)sizeof(int32_t);
}

template <bool SIGMOID, bool SELECT, bool ONE>
static void launch_route(const RouteParams& p, int blocks, hipStream_t st)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kRouteBlock), 0, st, p); };
    if constexpr (!SELECT) {
        go(route_kernel<1, SIGMOID, SELECT, ONE>);           // holds no logits
    } else {
        if (p.E <= 64) go(route_kernel<1, SIGMOID, SELECT, ONE>);
        else if (p.E <= 128) go(route_kernel<2, SIGMOID, SELECT, ONE>);
        else if (p.E <= 256) go(route_kernel<4, SIGMOID, SELECT, ONE>);
        else if (p.E <= 512) go(route_kernel<8, SIGMOID, SELECT, ONE>);
        else go(route_kernel<16, SIGMOID, SELECT, ONE>);
    }
}

static int run_route(RouteParams& p, bool select, bool sigmoid, void* workspace, long long bytes, hipStream_t st)
{
    const int64_t need = route_workspace(p.M, p.E);
    if (need > 0 && (workspace == nullptr || !aligned(workspace, 16) || bytes < need)) return -2;
    p.counts = static_cast<int32_t*>(workspace);
    p.count_stride = (p.E + 4) / 4 * 4;
    p.id_bits = 0;
    while (p.E >> p.id_bits) ++p.id_bits;        // ids 0 .. E
    const int blocks = route_blocks(p.M, &p.tokens);
    const bool one = need == 0;
    if (!select) one ? launch_route<false, false, true>(p, 1, st) : launch_route<false, false, false>(p, blocks, st);
    else if (sigmoid) one ? launch_route<true, true, true>(p, 1, st) : launch_route<true, true, false>(p, blocks, st);
    else one ? launch_route<false, true, true>(p, 1, st) : launch_route<false, true, false>(p, blocks, st);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess || one) return (int)e;
    hipLaunchKernelGGL(route_order_kernel, dim3((uint32_t)blocks), dim3(kRouteBlock), 0, st, p);
    return (int)hipGetLastError();
}

// No tokens: every expert has none.
__global__ void __launch_bounds__(kRouteBlock) route_nothing_kernel(int32_t* offsets, int E)
{
    for (int e = (int)threadIdx.x; e <= E; e += kRouteBlock) offsets[e] = 0;
}
static int route_nothing(void* offsets, int E, hipStream_t st)
{
    hipLaunchKernelGGL(route_nothing_kernel, dim3(1), dim3(kRouteBlock), 0, st, static_cast<int32_t*>(offsets), E);
    return (int)hipGetLastError();
}

}  // namespace paia

extern "C" {

long long paia_route_experts_workspace(int M, int experts, int k)
{
    return paia::route_sizes(M, experts, k) ? paia::route_workspace(M, experts) : -2;
}

int paia_route_experts(const void* logits, int logits_fp32, long long logits_stride, const void* bias, int sigmoid,
                       int renormalize, float scale, void* ids, void* weights, void* order, void* offsets, int M, int experts,
                       int k, void* workspace, long long workspace_bytes, void* stream)
{
    using namespace paia;
    if (!route_sizes(M, experts, k) || k > experts || (logits_fp32 != 0 && logits_fp32 != 1) ||
        (sigmoid != 0 && sigmoid != 1) || (renormalize != 0 && renormalize != 1) || (bias != nullptr && !sigmoid))
        return -2;
    if (offsets == nullptr || !aligned(offsets, 4)) return -2;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (M == 0) return route_nothing(offsets, experts, st);
    if (logits == nullptr || ids == nullptr || weights == nullptr || order == nullptr ||
        !aligned(logits, logits_fp32 ? 4 : 2) || !aligned(bias, 4) || !aligned(ids, 4) || !aligned(weights, 4) ||
        !aligned(order, 4) || logits_stride < 0)
        return -2;
    RouteParams p{};
    p.logits = logits;
    p.bias = static_cast<const float*>(bias);
    p.ids = static_cast<int32_t*>(ids);
    p.weights = static_cast<float*>(weights);
    p.order = static_cast<int32_t*>(order);
    p.offsets = static_cast<int32_t*>(offsets);
    p.stride = logits_stride;
    p.M = M, p.E = experts, p.k = k;
    p.fp32 = logits_fp32, p.renormalize = renormalize, p.scale = scale;
    return run_route(p, true, sigmoid, workspace, workspace_bytes, st);
}

int paia_expert_order(const void* ids, void* order, void* offsets, int M, int experts, int k, void* workspace,
                      long long workspace_bytes, void* stream)
{
    using namespace paia;
    if (!route_sizes(M, experts, k) || offsets == nullptr || !aligned(offsets, 4)) return -2;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (M == 0) return route_nothing(offsets, experts, st);
    if (ids == nullptr || order == nullptr || !aligned(ids, 4) || !aligned(order, 4)) return -2;
    RouteParams p{};
    p.ids = static_cast<int32_t*>(const_cast<void*>(ids));
    p.order = static_cast<int32_t*>(order);
    p.offsets = static_cast<int32_t*>(offsets);
    p.M = M, p.E = experts, p.k = k;
    return run_route(p, false, false, workspace, workspace_bytes, st);
}

}  // extern "C"
