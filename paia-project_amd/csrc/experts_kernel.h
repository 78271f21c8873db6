// Products of rows with the matrices of the experts that they chose, grouped by expert, for gfx950.
//
//   out[p, n] = bf16_rn( act( sum_k deq(W[e, n, k]) x[row(p), k] + bias[e, n] ) ),   e the expert of pair p
//
// The pairs come ordered by expert (`order`, `offsets`), as many each as the tokens happened to choose; what a call has to do
// is known on the device alone. So the host launches the most blocks that these sizes can need, and a block finds from the
// offsets which expert, which of its chunks of at most BM pairs and which columns are its own, or that there is nothing left
// (unit_of: one load a lane and a scan, no list has to be made beforehand). Units of one expert and columns follow each
// other, and each of the 8 XCDs takes a contiguous range of them: its chunks read the weights from one L2.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "divisor.h"
#include "gemv_tile.h"

namespace paia {

struct ExpertsParams {
    const uint8_t* W;        // [E][N] weight rows of row_bytes
    const uint8_t* meta;     // FP8: fp32 scale [E][N]; INT4: fp16 scale [E][N][G]; INT4ZP: bf16 scale [E][N][G]
    const uint8_t* zeros;    // INT4ZP: [E][N][zbytes]
    const uint16_t* x;
    const uint16_t* bias;    // bf16 [E][N] or null
    uint16_t* out;
    const int32_t *order, *offsets;
    int64_t x_stride, out_stride;    // elements
    int E, N, K, R;          // R: pairs
    int cols;                // outputs of a pair: N, or N / 2 where gated
    int tiles;               // units of columns
    int lane_experts;        // experts a lane counts: ceil(E / 64)
    int most;                // chunks that the launch has blocks for
    uint32_t row_bytes, zbytes;
    int G;                   // groups of a row
    Divisor by_tiles, by_pairs;      // by `tiles`; by the pairs that share a row of x
};

struct ExpertUnit {
    int expert;              // E: pairs without an expert; -1: no unit
    int first, held, tile;   // its pairs are order[first .. first + held)
};

__device__ __forceinline__ int wave_inclusive(int v)
{
    // row-wise shifts, then the row ends carried on: lane 63 holds the sum
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// The unit of this block, the same in every lane. Offsets are taken as they are but for their range: whatever they hold, first
// and held stay within the pairs.
template <int BM>
__device__ __forceinline__ ExpertUnit unit_of(const ExpertsParams& p)
{
    const int lane = lane_id(), e0 = lane * p.lane_experts;
    const auto place = [&](int e) { return min(max(p.offsets[min(e, p.E)], 0), p.R); };
    const int rest_at = place(p.E);
    int from = place(e0), own = 0;
    const int from0 = from;
    for (int i = 1; i <= p.lane_experts; ++i) {
        const int to = place(e0 + i);
        own += (max(to - from, 0) + BM - 1) / BM;
        from = to;
    }
    own = min(own, p.most);                  // no more than that in all, unless the offsets are not in order
    const int upto = wave_inclusive(own);
    const int chunks = min(__builtin_amdgcn_readlane(upto, 63), p.most);
    const int units = min(chunks + (p.R - rest_at + BM - 1) / BM, p.most) * p.tiles;
    int u = (int)blockIdx.x;
    if (u >= units) return {-1, 0, 0, 0};
    {
        const int xcd = u % 8, per = units / 8, rem = units % 8;
        u = xcd * per + min(xcd, rem) + u / 8;
    }
    const int c = (int)p.by_tiles.of((uint32_t)u);
    if (c >= chunks) {
        const int first = rest_at + (c - chunks) * BM;
        return {p.E, first, min(BM, p.R - first), u - c * p.tiles};
    }
    const int owner = __builtin_ctzll(__ballot(upto > c));
    int e = 0, begin = 0, lo = 0, hi = 0, n = 1, at = upto - own;
    from = from0;
    for (int i = 1; i <= p.lane_experts; ++i) {
        const int to = place(e0 + i), k = (max(to - from, 0) + BM - 1) / BM;
        if (c >= at && c < at + k) e = e0 + i - 1, begin = at, lo = from, hi = to, n = k;
        at += k;
        from = to;
    }
    e = __builtin_amdgcn_readlane(e, owner), begin = __builtin_amdgcn_readlane(begin, owner);
    lo = __builtin_amdgcn_readlane(lo, owner), hi = __builtin_amdgcn_readlane(hi, owner);
    n = __builtin_amdgcn_readlane(n, owner);
    const int local = u - begin * p.tiles, tile = local / n, first = lo + (local - tile * n) * BM;
    return {e, first, min(BM, hi - first), tile};
}

__device__ __forceinline__ int pair_at(const ExpertsParams& p, const ExpertUnit& u, int i)
{
    return p.order[u.first + min(i, u.held - 1)];
}
// A pair's row of x; a number that is no pair reads row 0, and is not written.
__device__ __forceinline__ const uint8_t* x_row(const ExpertsParams& p, int pair)
{
    const uint32_t q = (uint32_t)pair < (uint32_t)p.R ? (uint32_t)pair : 0u;
    return reinterpret_cast<const uint8_t*>(p.x) + (int64_t)p.by_pairs.of(q) * p.x_stride * 2;
}

// 16 bytes from each lane's address to LDS, at the wave's base + 16 * lane.
__device__ __forceinline__ void lds_copy16(uint8_t* base, const uint8_t* p)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                     (__attribute__((address_space(3))) void*)base, 16, 0, 0);
}
// Until at most N of the wave's loads are on their way: what the others brought to LDS can be read. The compiler does not see that
// such a load writes all of what its lanes cover, so neither its own waits nor its order of accesses are relied on: the fences
// (no instructions come of them) keep every access on its side.
template <int N>
__device__ __forceinline__ void wait_loads()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// Until the wave's reads of LDS are done: what they read can be overwritten.
__device__ __forceinline__ void wait_reads()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Rows of outputs without an expert are 0.
__device__ __forceinline__ void zero_rows(const ExpertsParams& p, const ExpertUnit& u, int c0, int c1)
{
    const int width = c1 - c0;
    for (int i = (int)threadIdx.x; i < u.held * width; i += (int)blockDim.x) {
        const int r = i / width, pair = p.order[u.first + r];
        if ((uint32_t)pair < (uint32_t)p.R) p.out[(int64_t)pair * p.out_stride + c0 + (i - r * width)] = 0;
    }
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

// Eight nibbles of a word (k .. k + 7) as bf16 in their order, times 2^-9 and the power of two of `f`.
__device__ __forceinline__ u32x4 i4_frag(uint32_t v, float f)
{
    const uint32_t lo = v & 0x0F0F0F0Fu, hi = (v >> 4) & 0x0F0F0F0Fu;
    const uint32_t a = __builtin_amdgcn_perm(hi, lo, 0x05010400u), b = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
    return u32x4{i4x2_to_bf16x2<false>(a, f), i4x2_to_bf16x2<true>(a, f), i4x2_to_bf16x2<false>(b, f),
                 i4x2_to_bf16x2<true>(b, f)};
}
__device__ __forceinline__ u32x4 fp8_frag(uint32_t d0, uint32_t d1)
{
    return u32x4{fp8x2_to_bf16x2<false>(d0), fp8x2_to_bf16x2<true>(d0), fp8x2_to_bf16x2<false>(d1),
                 fp8x2_to_bf16x2<true>(d1)};
}

// INT4 metadata of one row and group as gemv_tile.h's words.
template <int F>
__device__ __forceinline__ uint32_t i4_word_of(uint32_t scale, uint32_t zero)
{
    const uint32_t s = scale << 16;
    const float up = (F == kI4 ? f16_to_f32(scale) : __uint_as_float(s)) * kI4Up;
    if constexpr (F == kI4) return __float_as_uint(up);
    return fabsf(up) > kF32Max ? i4zp_word_big(s, zero) : i4zp_word(up, zero);
}
template <int F>
__device__ __forceinline__ uint32_t i4_meta(const ExpertsParams& p, int64_t row, int g)
{
    const uint32_t s = reinterpret_cast<const uint16_t*>(p.meta)[row * p.G + g];
    const uint32_t z = F == kI4ZP ? (uint32_t)p.zeros[row * p.zbytes + (g >> 1)] >> (4 * (g & 1)) & 15u : 8u;
    return i4_word_of<F>(s, z);
}
template <int F> __device__ __forceinline__ float i4_factor(uint32_t m) { return __uint_as_float(F == kI4 ? kI4Exp << 23 : (m & 0xFF00u) << 15); }
template <int F> __device__ __forceinline__ float i4_scale(uint32_t m) { return __uint_as_float(F == kI4 ? m : m & 0xFFFF0000u); }
template <int F> __device__ __forceinline__ float i4_zero(uint32_t m) { return F == kI4 ? 8.0f : (float)(m & 0xFFu); }

// The sum of a row and column on its way out: scale, bias.
template <int F>
__device__ __forceinline__ float finish(float v, float scale, float bias)
{
    if constexpr (F == kI4 || F == kI4ZP) v = v * kI4Back;
    if constexpr (F == kFP8) v = v * scale;
    return v + bias;
}

// Which weight row the columns of a unit's 16-row tile i are: gated units take gate and up tiles in turn.
template <bool GATED, int TILES>
__device__ __forceinline__ int tile_row(const ExpertsParams& p, int unit_tile, int i)
{
    if constexpr (GATED) return (i & 1 ? p.cols : 0) + (unit_tile * (TILES / 2) + i / 2) * kTileRows;
    return (unit_tile * TILES + i) * kTileRows;
}
// Rows of that tile within its half (or within N).
template <bool GATED, int TILES>
__device__ __forceinline__ int tile_rows(const ExpertsParams& p, int unit_tile, int i)
{
    return min(kTileRows, p.cols - (unit_tile * (GATED ? TILES / 2 : TILES) + (GATED ? i / 2 : i)) * kTileRows);
}

template <int F>
struct StreamFmt {
    static constexpr bool kI4F = F == kI4 || F == kI4ZP;
    static constexpr int kCols = F == kBF16 ? 64 : 128;          // columns of a stage
    static constexpr int kRowBytes = kI4F ? 64 : 128;            // weight bytes of a row and stage
    static constexpr int kSteps = kCols / 32;
    static constexpr int kXRowBytes = 2 * kCols;
};

// ---------------------------------------------------------------------------------------------------------------
// Few rows an expert: bound by reading the weights. A unit is up to MT pairs and P tiles of 16 weight rows; the WAVES waves of
// its block take the stages of K in turn, each through two wave-private places in LDS that are filled straight from memory
// (no registers, no block barrier), and add their partial sums in LDS at the end, in order.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kStreamGroups = 160;       // INT4: groups of a row whose metadata the block keeps (K <= 20480)
template <int F, int P, int WAVES, int MT, bool GATED>
struct StreamShape {
    using T = StreamFmt<F>;
    static constexpr int kXRows = MT > kChunkBytes / T::kXRowBytes ? MT : kChunkBytes / T::kXRowBytes;
    static constexpr int kWBytes = P * kTileRows * T::kRowBytes, kXBytes = kXRows * T::kXRowBytes;
    static constexpr int kSlot = kWBytes + kXBytes > P * 1024 ? kWBytes + kXBytes : P * 1024;
};

template <int F, int P, int WAVES, int MT, bool GATED>
__global__ void __launch_bounds__(WAVES * kWave) experts_stream_kernel(const ExpertsParams p)
{
    using T = StreamFmt<F>;
    using S = StreamShape<F, P, WAVES, MT, GATED>;
    constexpr bool I4 = T::kI4F;
    constexpr int C = T::kCols, RB = T::kRowBytes, X = T::kSteps, L = RB * kTileRows / kChunkBytes;
    constexpr int WP = RB / 16, WR = kWave / WP, XP = T::kXRowBytes / 16, XR = kWave / XP, XL = S::kXRows / XR;
    __shared__ __attribute__((aligned(16))) uint8_t slot0[WAVES][S::kSlot];
    __shared__ __attribute__((aligned(16))) uint8_t slot1[WAVES][S::kSlot];
    constexpr int kMdStride = P * kTileRows + 1;
    __shared__ uint32_t md[I4 ? kStreamGroups * kMdStride : 1];      // INT4: metadata words [group][row]

    const ExpertUnit u = unit_of<MT>(p);
    if (u.expert < 0) return;
    const int lane = lane_id(), wave = wave_id(), ln = lane & 15, lh = lane >> 4;
    constexpr int kOutCols = (GATED ? P / 2 : P) * kTileRows;
    const int c0 = u.tile * kOutCols;
    if (u.expert == p.E) {
        zero_rows(p, u, c0, min(c0 + kOutCols, p.cols));
        return;
    }
    const int64_t row0 = (int64_t)u.expert * p.N;

    // addresses: one base a tile and load for the weights, one a load for x
    const uint8_t* wt[P];
    uint32_t wo[P][L], wpiece;
    const uint8_t* xp[XL];
    uint32_t xpiece[XL];
    {
        const int r = lane / WP, at = lane % WP;
        wpiece = (uint32_t)(RB == 128 ? at ^ (r & 7) : at ^ (r >> 1 & 3)) * 16u;
#pragma unroll
        for (int t = 0; t < P; ++t) {
            const int n0 = tile_row<GATED, P>(p, u.tile, t), rows = max(1, tile_rows<GATED, P>(p, u.tile, t));
            wt[t] = p.W + (row0 + min(n0, p.N - 1)) * p.row_bytes;
#pragma unroll
            for (int i = 0; i < L; ++i) wo[t][i] = (uint32_t)min(i * WR + r, rows - 1) * p.row_bytes;
        }
    }
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int r = i * XR + lane / XP;
        xp[i] = x_row(p, pair_at(p, u, r));
        xpiece[i] = (uint32_t)((lane % XP) ^ (r & 7)) * 16u;
    }
    const int stages = (p.K + C - 1) / C, n = (stages - wave + WAVES - 1) / WAVES;
    const auto issue = [&](uint8_t* slot, int t) {
        if (t >= n) return;
        const uint32_t s = (uint32_t)(wave + t * WAVES);
        // bytes past the row's end are read from its last piece, and dropped in the last stage
        const uint32_t wc = min(s * RB + wpiece, p.row_bytes - 16u);
#pragma unroll
        for (int t2 = 0; t2 < P; ++t2)
#pragma unroll
            for (int i = 0; i < L; ++i) lds_copy16(slot + (t2 * L + i) * 1024, wt[t2] + (wo[t2][i] + wc));
#pragma unroll
        for (int i = 0; i < XL; ++i)
            lds_copy16(slot + S::kWBytes + i * 1024, xp[i] + min(s * (2 * C) + xpiece[i], (uint32_t)p.K * 2u - 16u));
    };
    issue(slot0[wave], 0);
    issue(slot1[wave], 1);

    if constexpr (I4) {
        for (int i = (int)threadIdx.x; i < P * kTileRows * p.G; i += WAVES * kWave) {
            const int r = i / p.G, g = i - r * p.G, t = r / kTileRows;
            const int rows = max(1, tile_rows<GATED, P>(p, u.tile, t));
            const int row = min(tile_row<GATED, P>(p, u.tile, t), p.N - 1) + min(r % kTileRows, rows - 1);
            md[g * kMdStride + r] = i4_meta<F>(p, row0 + row, g);
        }
        __syncthreads();
    }
    const uint32_t one2 = (uint32_t)__builtin_amdgcn_readfirstlane((int)kI4Ones);
    const u32x4 ones = {one2, one2, one2, one2};
    f32x4 acc[P];
#pragma unroll
    for (int t = 0; t < P; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto use = [&](uint8_t* slot, int t) {
        const int s = wave + t * WAVES, left = p.K - s * C;
        if (t + 1 < n) wait_loads<P * L + XL>();     // the next stage's may be on their way
        else wait_loads<0>();
        u32x4 a[X], w[P][L];
#pragma unroll
        for (int j = 0; j < X; ++j) {
            const int piece = F == kBF16 ? 4 * j + lh : (F == kFP8 ? 8 * (j >> 1) + 2 * lh + (j & 1) : 4 * lh + j);
            const int r = ln & (S::kXRows - 1);
            a[j] = *reinterpret_cast<const u32x4*>(slot + S::kWBytes + r * T::kXRowBytes + ((piece ^ (r & 7)) << 4));
        }
#pragma unroll
        for (int t2 = 0; t2 < P; ++t2)
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int piece = 4 * i + lh;
                const int at = RB == 128 ? ln * 128 + ((piece ^ (ln & 7)) << 4) : ln * 64 + ((piece ^ (ln >> 1 & 3)) << 4);
                w[t2][i] = *reinterpret_cast<const u32x4*>(slot + t2 * kTileRows * RB + at);
            }
        wait_reads();
        issue(slot, t + 2);
        __builtin_amdgcn_sched_barrier(0);
        if (!I4 && left < C) {                       // the row's end: both operands are 0 past it
#pragma unroll
            for (int j = 0; j < X; ++j)
                if (step_col<F>(j, lh) >= left) a[j] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int t2 = 0; t2 < P; ++t2)
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (step_col<F>(F == kFP8 ? 2 * i : i, lh) >= left) w[t2][i] = u32x4{0, 0, 0, 0};
        }
        f32x4 xs = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (I4) {
#pragma unroll
            for (int j = 0; j < X; ++j) xs = mfma_16x16x32(a[j], ones, xs);
        }
#pragma unroll
        for (int t2 = 0; t2 < P; ++t2) {
            if constexpr (F == kBF16) {
#pragma unroll
                for (int j = 0; j < X; ++j) acc[t2] = mfma_16x16x32(a[j], w[t2][j], acc[t2]);
            } else if constexpr (F == kFP8) {
#pragma unroll
                for (int j = 0; j < X; ++j) {
                    const u32x4 v = w[t2][j >> 1];
                    acc[t2] = mfma_16x16x32(a[j], j & 1 ? fp8_frag(v.z, v.w) : fp8_frag(v.x, v.y), acc[t2]);
                }
            } else {
                const uint32_t m = md[s * kMdStride + t2 * kTileRows + ln];
                const float f = i4_factor<F>(m), sc = i4_scale<F>(m), z = i4_zero<F>(m);
                f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < X; ++j) g = mfma_16x16x32(a[j], i4_frag(w[t2][0][j], f), g);
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[t2][v] = __builtin_fmaf(sc, __builtin_fmaf(-z, xs[v], g[v]), acc[t2][v]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    for (int t = 0; t < n; t += 2) {
        use(slot0[wave], t);
        if (t + 1 < n) use(slot1[wave], t + 1);
    }

    // partial tiles to the wave's own place, then the first waves add them in order and finish
#pragma unroll
    for (int t = 0; t < P; ++t) *reinterpret_cast<f32x4*>(slot0[wave] + t * 1024 + lane * 16) = acc[t];
    __syncthreads();
    constexpr int kOuts = GATED ? P / 2 : P;
    for (int q = wave; q < kOuts; q += WAVES) {
        f32x4 v[GATED ? 2 : 1];
        const int col = c0 + q * kTileRows + ln;
        if (col >= p.cols) continue;
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h) {
            const int t = GATED ? 2 * q + h : q;
            const int64_t row = row0 + (GATED ? h * p.cols : 0) + col;
            f32x4 sum = *reinterpret_cast<const f32x4*>(slot0[0] + t * 1024 + lane * 16);
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += *reinterpret_cast<const f32x4*>(slot0[w] + t * 1024 + lane * 16);
            const float scale = F == kFP8 ? reinterpret_cast<const float*>(p.meta)[row] : 1.0f;
            const float bias = p.bias != nullptr ? bf16_to_f32(p.bias[row]) : 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) v[h][c] = finish<F>(sum[c], scale, bias);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int m = 4 * lh + c;
            const int pair = m < u.held ? p.order[u.first + m] : -1;
            if ((uint32_t)pair >= (uint32_t)p.R) continue;
            const float o = GATED ? silu(v[0][c]) * v[GATED ? 1 : 0][c] : v[0][c];
            p.out[(int64_t)pair * p.out_stride + col] = (uint16_t)f32_to_bf16_out(o);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// More rows an expert: a block is BM pairs by 16 tiles of weight rows, its 8 waves 2 x 4 (or 1 x 8) parts of that. Two places
// in LDS are filled straight from memory in turn: while one stage is multiplied the next is on its way, one barrier a stage.
// ---------------------------------------------------------------------------------------------------------------
template <int F, int BM>
struct TileShape {
    static constexpr bool kI4F = F == kI4 || F == kI4ZP;
    static constexpr int kCols = F == kBF16 || (F == kFP8 && BM == 256) ? 64 : 128;
    static constexpr int kRowBytes = F == kBF16 ? 2 * kCols : (F == kFP8 ? kCols : kCols / 2);
    static constexpr int kXRowBytes = 2 * kCols, kSteps = kCols / 32;
    static constexpr int kTiles = 16;                            // of 16 weight rows
    static constexpr int kM = BM >= 128 ? 2 : 1, kN = 8 / kM;    // the waves' parts
    static constexpr int kTM = BM / 16 / kM, kTN = kTiles / kN;
    static constexpr int kWBytes = kTiles * kTileRows * kRowBytes, kXBytes = BM * kXRowBytes;
};

template <int F, int BM, bool GATED>
__global__ void __launch_bounds__(512) experts_tile_kernel(const ExpertsParams p)
{
    using T = TileShape<F, BM>;
    constexpr bool I4 = T::kI4F;
    constexpr int C = T::kCols, RB = T::kRowBytes, XB = T::kXRowBytes, X = T::kSteps, TM = T::kTM, TN = T::kTN;
    constexpr int WP = RB / 16, WR = kWave / WP, WL = T::kWBytes / 8192, XP = XB / 16, XR = kWave / XP;
    constexpr int XL = (T::kXBytes + 8191) / 8192, XW = T::kXBytes / 1024 < 8 ? T::kXBytes / 1024 : 8;   // XW: waves that load x
    __shared__ __attribute__((aligned(16))) uint8_t slot0[T::kWBytes + T::kXBytes];
    __shared__ __attribute__((aligned(16))) uint8_t slot1[T::kWBytes + T::kXBytes];

    const ExpertUnit u = unit_of<BM>(p);
    if (u.expert < 0) return;
    const int lane = lane_id(), wave = wave_id(), ln = lane & 15, lh = lane >> 4;
    const int wm = wave / T::kN, wn = wave % T::kN;
    constexpr int kOutCols = (GATED ? T::kTiles / 2 : T::kTiles) * kTileRows;
    const int c0 = u.tile * kOutCols;
    if (u.expert == p.E) {
        zero_rows(p, u, c0, min(c0 + kOutCols, p.cols));
        return;
    }
    const int64_t row0 = (int64_t)u.expert * p.N;
    const uint8_t* We = p.W + row0 * p.row_bytes;

    // A load of weights lies within a 16-row tile: its base is the wave's, an offset the lane's. x has an address a row.
    const auto w_piece = [](int r) { return RB == 128 ? r & 7 : r >> 1 & 3; };
    const uint8_t* wp[WL];
    uint32_t wo[WL];
    const int wr = lane / WP, xr = lane / XP;
    const uint32_t wpiece = (uint32_t)((lane % WP) ^ w_piece(wr)) * 16u;         // a load's first row is a multiple of 8
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int r0 = (wave * WL + i) * WR, t = r0 / kTileRows;
        const int rows = max(1, tile_rows<GATED, T::kTiles>(p, u.tile, t));
        wp[i] = We + (int64_t)min(tile_row<GATED, T::kTiles>(p, u.tile, t), p.N - 1) * p.row_bytes;
        wo[i] = (uint32_t)min(r0 % kTileRows + wr, rows - 1) * p.row_bytes;
    }
    const uint8_t* xp[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) xp[i] = x_row(p, pair_at(p, u, (wave * XL + i) * XR + xr));
    const int stages = (p.K + C - 1) / C;
    const auto issue = [&](uint8_t* slot, int s) {
        if (s >= stages) return;
        const uint32_t wc = min((uint32_t)s * RB + wpiece, p.row_bytes - 16u);
#pragma unroll
        for (int i = 0; i < WL; ++i) lds_copy16(slot + (wave * WL + i) * 1024, wp[i] + (wo[i] + wc));
        if (XW == 8 || wave < XW) {
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                const int r = (wave * XL + i) * XR + xr;
                const uint32_t c = (uint32_t)s * XB + (uint32_t)((lane % XP) ^ (r & 7)) * 16u;
                lds_copy16(slot + T::kWBytes + (wave * XL + i) * 1024, xp[i] + min(c, (uint32_t)p.K * 2u - 16u));
            }
        }
    };
    // INT4: the words of the stage's group for the wave's columns, a stage ahead
    int64_t mrow[I4 ? TN : 1];
    uint32_t word[I4 ? TN : 1];
    if constexpr (I4) {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            const int i = wn * TN + t, rows = max(1, tile_rows<GATED, T::kTiles>(p, u.tile, i));
            mrow[t] = row0 + min(tile_row<GATED, T::kTiles>(p, u.tile, i), p.N - 1) + min(ln, rows - 1);
            word[t] = i4_meta<F>(p, mrow[t], 0);
        }
    }
    const uint32_t one2 = (uint32_t)__builtin_amdgcn_readfirstlane((int)kI4Ones);
    const u32x4 ones = {one2, one2, one2, one2};
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const bool busy = wm * TM * 16 < u.held;         // a part without pairs waits at the barriers only

    const auto get_x = [&](const uint8_t* slot, int i, int j) {
        const int r = (wm * TM + i) * 16 + ln;
        const int piece = F == kBF16 ? 4 * j + lh : (F == kFP8 ? 8 * (j >> 1) + 2 * lh + (j & 1) : 4 * lh + j);
        return *reinterpret_cast<const u32x4*>(slot + T::kWBytes + r * XB + ((piece ^ (r & 7)) << 4));
    };
    const auto get_w = [&](const uint8_t* slot, int t, int i) {
        const int r = (wn * TN + t) * 16 + ln;
        return *reinterpret_cast<const u32x4*>(slot + r * RB + (((4 * i + lh) ^ w_piece(r)) << 4));
    };
    const auto use = [&](const uint8_t* slot) {
        if constexpr (I4) {
            u32x4 a[TM][X], w[TN];
            f32x4 xs[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < X; ++j) a[i][j] = get_x(slot, i, j);
#pragma unroll
            for (int t = 0; t < TN; ++t) w[t] = get_w(slot, t, 0);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                xs[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < X; ++j) xs[i] = mfma_16x16x32(a[i][j], ones, xs[i]);
            }
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const float f = i4_factor<F>(word[t]), sc = i4_scale<F>(word[t]), z = i4_zero<F>(word[t]);
                f32x4 g[TM];
#pragma unroll
                for (int i = 0; i < TM; ++i) g[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < X; ++j) {
                    const u32x4 b = i4_frag(w[t][j], f);
#pragma unroll
                    for (int i = 0; i < TM; ++i) g[i] = mfma_16x16x32(a[i][j], b, g[i]);
                }
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        acc[i][t][v] = __builtin_fmaf(sc, __builtin_fmaf(-z, xs[i][v], g[i][v]), acc[i][t][v]);
            }
        } else {
            constexpr int kWSteps = F == kFP8 ? 2 : 1;     // steps that a 16-byte piece of a weight row holds
#pragma unroll
            for (int j0 = 0; j0 < X; j0 += kWSteps) {
                u32x4 w[TN];
#pragma unroll
                for (int t = 0; t < TN; ++t) w[t] = get_w(slot, t, j0 / kWSteps);
#pragma unroll
                for (int k = 0; k < kWSteps; ++k) {
                    u32x4 b[TN];
#pragma unroll
                    for (int t = 0; t < TN; ++t)
                        b[t] = F == kBF16 ? w[t] : (k ? fp8_frag(w[t].z, w[t].w) : fp8_frag(w[t].x, w[t].y));
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        const u32x4 a = get_x(slot, i, j0 + k);
#pragma unroll
                        for (int t = 0; t < TN; ++t) acc[i][t] = mfma_16x16x32(a, b[t], acc[i][t]);
                    }
                }
            }
        }
    };
    // The last stage of a K that is no multiple of its columns: what lies past the rows' ends is 0 in both operands.
    const auto clear_past = [&](uint8_t* slot, int left) {
        constexpr int kWCols = F == kFP8 ? 16 : 8;
        const u32x4 none = {0, 0, 0, 0};
        for (int e = (int)threadIdx.x; e < T::kTiles * kTileRows * WP; e += 512) {
            const int r = e / WP, at = e % WP;
            if ((at ^ w_piece(r)) * kWCols >= left) *reinterpret_cast<u32x4*>(slot + r * RB + at * 16) = none;
        }
        for (int e = (int)threadIdx.x; e < BM * XP; e += 512) {
            const int r = e / XP, at = e % XP;
            if ((at ^ (r & 7)) * 8 >= left) *reinterpret_cast<u32x4*>(slot + T::kWBytes + r * XB + at * 16) = none;
        }
        __syncthreads();
    };
    const auto stage = [&](uint8_t* mine, uint8_t* next, int s) {
        wait_loads<0>();
        __syncthreads();                             // this stage has arrived, the other place is read
        issue(next, s + 1);
        uint32_t ahead[I4 ? TN : 1];
        if constexpr (I4) {
#pragma unroll
            for (int t = 0; t < TN; ++t) ahead[t] = i4_meta<F>(p, mrow[t], min(s + 1, p.G - 1));
        }
        if (!I4 && p.K - s * C < C) clear_past(mine, p.K - s * C);
        if (busy) use(mine);
        if constexpr (I4) {
#pragma unroll
            for (int t = 0; t < TN; ++t) word[t] = ahead[t];
        }
    };
    issue(slot0, 0);
    for (int s = 0; s < stages; s += 2) {
        stage(slot0, slot1, s);
        if (s + 1 < stages) stage(slot1, slot0, s + 1);
    }
    if (!busy) return;

    float scale[TN], bias[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) {
        const int i = wn * TN + t, rows = max(1, tile_rows<GATED, T::kTiles>(p, u.tile, i));
        const int64_t row = row0 + min(tile_row<GATED, T::kTiles>(p, u.tile, i), p.N - 1) + min(ln, rows - 1);
        scale[t] = F == kFP8 ? reinterpret_cast<const float*>(p.meta)[row] : 1.0f;
        bias[t] = p.bias != nullptr ? bf16_to_f32(p.bias[row]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int m = (wm * TM + i) * 16 + 4 * lh + c;
            const int pair = m < u.held ? p.order[u.first + m] : -1;
            if ((uint32_t)pair >= (uint32_t)p.R) continue;
            uint16_t* out = p.out + (int64_t)pair * p.out_stride;
#pragma unroll
            for (int t = 0; t < TN; t += GATED ? 2 : 1) {
                const int i0 = wn * TN + t, col = c0 + (GATED ? i0 / 2 : i0) * kTileRows + ln;
                float o = finish<F>(acc[i][t][c], scale[t], bias[t]);
                if constexpr (GATED) o = silu(o) * finish<F>(acc[i][t + (GATED ? 1 : 0)][c], scale[t + (GATED ? 1 : 0)],
                                                             bias[t + (GATED ? 1 : 0)]);
                if (col < p.cols) out[col] = (uint16_t)f32_to_bf16_out(o);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------

// Launches of a format's kernels; p as the entry point fills it but for tiles and most. 0, -2 (more blocks than a launch has)
// or a hipError_t.
constexpr int kMostBlocks = 1 << 22;
template <typename K>
int launch_experts(K kernel, ExpertsParams p, int BM, int tiles_cols, int threads, hipStream_t st)
{
    p.tiles = (p.cols + tiles_cols - 1) / tiles_cols;
    p.by_tiles = Divisor((uint32_t)p.tiles);
    const int64_t bins = p.R < p.E + 1 ? p.R : p.E + 1;
    const int64_t most = ((int64_t)p.R + bins * (BM - 1)) / BM;
    if (most * p.tiles > kMostBlocks) return -2;
    p.most = (int)most;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(most * p.tiles)), dim3((uint32_t)threads), 0, st, p);
    return (int)hipGetLastError();
}
template <int F, int MT, bool GATED>
int launch_stream(const ExpertsParams& p, hipStream_t st)
{
    constexpr int P = 2, WAVES = 8;
    return launch_experts(experts_stream_kernel<F, P, WAVES, MT, GATED>, p, MT, (GATED ? P / 2 : P) * kTileRows,
                          WAVES * kWave, st);
}
template <int F, int BM, bool GATED>
int launch_tiles(const ExpertsParams& p, hipStream_t st)
{
    using T = TileShape<F, BM>;
    return launch_experts(experts_tile_kernel<F, BM, GATED>, p, BM, (GATED ? T::kTiles / 2 : T::kTiles) * kTileRows, 512, st);
}
template <int F, bool GATED>
int launch_format(const ExpertsParams& p, hipStream_t st)
{
    constexpr bool kI4F = F == kI4 || F == kI4ZP;
    const int64_t R = p.R, E = p.E;
    if (R <= 12 * E && (!kI4F || p.G <= kStreamGroups)) {
        if (3 * R <= 4 * E) return launch_stream<F, 4, GATED>(p, st);
        if (3 * R <= 8 * E) return launch_stream<F, 8, GATED>(p, st);
        return launch_stream<F, 16, GATED>(p, st);
    }
    if (R <= 32 * E) return launch_tiles<F, 32, GATED>(p, st);
    if (R <= 64 * E) return launch_tiles<F, 64, GATED>(p, st);
    if (kI4F || R <= 160 * E) return launch_tiles<F, 128, GATED>(p, st);
    return launch_tiles<F, kI4F ? 128 : 256, GATED>(p, st);
}
template <int F>
int launch_experts_format(const ExpertsParams& p, bool gated, hipStream_t st)
{
    return gated ? launch_format<F, true>(p, st) : launch_format<F, false>(p, st);
}

// The formats' launches, one source each.
int launch_experts_bf16(const ExpertsParams& p, bool gated, hipStream_t st);
int launch_experts_fp8(const ExpertsParams& p, bool gated, hipStream_t st);
int launch_experts_int4(const ExpertsParams& p, bool gated, hipStream_t st);
int launch_experts_int4_zp(const ExpertsParams& p, bool gated, hipStream_t st);

}  // namespace paia
