// Products of rows with the matrices of the experts that they chose, grouped by expert, for gfx950.
//
//   out[p, n] = bf16_rn( act( sum_k deq(W[e, n, k]) x[row(p), k] + bias[e, n] ) ),   e the expert of pair p
//
// The pairs come ordered by expert (`order`, `offsets`), as many each as the tokens happened to choose; what a call has to do
// is known on the device alone. So the host launches the most blocks that these sizes can need, and a block finds from the
// offsets which expert, which of its chunks of at most BM pairs and which columns are its own, or that there is nothing left
// (unit_of: one load a lane and a scan, no list has to be made beforehand; the arithmetic is in expert_units.h). Units of one
// expert and columns follow each other, and each of the 8 XCDs takes a contiguous range of them: its chunks read the weights from one L2.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "divisor.h"
#include "expert_units.h"
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
    uint32_t x_bytes;        // of x, first row's start to last row's end (streaming: below 2^31)
    int lane_experts;        // experts a lane counts: ceil(E / 64)
    int most;                // chunks that the launch has blocks for
    uint32_t row_bytes, zbytes;
    int G;                   // groups of a row
    Divisor by_tiles, by_pairs;      // by `tiles`; by the pairs that share a row of x
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

// How many chunks of BM pairs the experts have, and which one is which; the same in every lane but `upto` and `mine`. What a
// lane does by itself is in expert_units.h.
template <int BM>
struct Chunks {
    int count, rest_at, rest;            // rest: chunks of the pairs without an expert, order[rest_at ..]
    int upto;                            // chunks of the experts up to the lane's last
    LaneChunks mine;
    int order;                           // of up to 64 pairs the lane's, loaded beside the offsets

    __device__ __forceinline__ explicit Chunks(const ExpertsParams& p)
    {
        order = p.order[min(lane_id(), p.R - 1)];
        rest_at = pairs_begin(p.offsets, p.E, p.E, p.R);
        mine = lane_chunks(p.offsets, p.E, p.R, BM, lane_id() * p.lane_experts, p.lane_experts, p.most);
        upto = wave_inclusive(mine.own);
        count = min(__builtin_amdgcn_readlane(upto, 63), p.most);
        rest = min(chunks_of(p.R - rest_at, BM), p.most - count);
    }
    // That of chunk c < count.
    __device__ __forceinline__ ChunkExpert of(const ExpertsParams& p, int c) const
    {
        const int owner = __builtin_ctzll(__ballot(upto > c));
        const ChunkExpert x = expert_of(p.offsets, p.E, p.R, BM, lane_id() * p.lane_experts, p.lane_experts, mine, upto - mine.own, c);
        return {__builtin_amdgcn_readlane(x.expert, owner), __builtin_amdgcn_readlane(x.lo, owner), __builtin_amdgcn_readlane(x.hi, owner),
                __builtin_amdgcn_readlane(x.begin, owner), __builtin_amdgcn_readlane(x.n, owner)};
    }
};

// The unit of this block.
template <int BM>
__device__ __forceinline__ ExpertUnit unit_of(const ExpertsParams& p)
{
    const Chunks<BM> chunks(p);
    const int units = chunks.count * p.tiles, b = (int)blockIdx.x;
    if (b >= units + chunks.rest * p.tiles) return {-1, 0, 0, 0, 0};
    // units without an expert come last: dealt out with the others they left one XCD almost nothing to do
    const int u = b < units ? xcd_contiguous(b, units) : b;
    const int c = (int)p.by_tiles.of((uint32_t)u);
    if (c >= chunks.count) return unit_without<BM>(p.E, p.R, chunks.rest_at, c - chunks.count, u - c * p.tiles);
    return unit_in<BM>(chunks.of(p, c), u, p.tiles);
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
// A barrier for the block's LDS alone: loads from memory stay on their way.
__device__ __forceinline__ void block_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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
// The same in the order of i4_pair_x's values: (k, k + 2), (k + 4, k + 6), (k + 1, k + 3), (k + 5, k + 7).
__device__ __forceinline__ u32x4 i4_frag_paired(uint32_t v, float f)
{
    const uint32_t lo = v & 0x0F0F0F0Fu, hi = (v >> 4) & 0x0F0F0F0Fu;
    return u32x4{i4x2_to_bf16x2<false>(lo, f), i4x2_to_bf16x2<true>(lo, f), i4x2_to_bf16x2<false>(hi, f),
                 i4x2_to_bf16x2<true>(hi, f)};
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
// The words of a stage's H groups, the stage's number as odd as `stage`, from scales (two where H is 2) and zero points as stored.
template <int F, int H>
__device__ __forceinline__ void i4_words_of(uint32_t scales, uint32_t zeros, int stage, uint32_t (&word)[H])
{
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const uint32_t zero = F == kI4ZP ? zeros >> (4 * ((stage * H + h) & 1)) & 15u : 8u;
        word[h] = i4_word_of<F>(h ? scales >> 16 : scales & 0xFFFFu, zero);
    }
}
// Two bf16 whose products with x sum up to what a group's zero points take: -8 in the nibbles' scale, so that the group's sum begins
// with it; with zero points of their own 1, and each row takes its multiple (8 of 200 instructions of a stage more).
template <int F> constexpr uint32_t kI4Take = F == kI4 ? (kI4Ones + 0x01800180u) | 0x80008000u : kI4Ones;
template <int F> __device__ __forceinline__ float i4_factor(uint32_t m) { return __uint_as_float(F == kI4 ? kI4Exp << 23 : (m & 0xFF00u) << 15); }
template <int F> __device__ __forceinline__ float i4_scale(uint32_t m) { return __uint_as_float(F == kI4 ? m : m & 0xFFFF0000u); }
template <int F> __device__ __forceinline__ float i4_zero(uint32_t m) { return (float)(m & 0xFFu); }

// Where piece (16 bytes, 8 columns) `piece` of a row of x of XB bytes lies among the row's, before the XOR with the row's lowest
// three bits. A 16-byte read takes 16 lanes at a time: eight rows (all values of those bits) of one column group of the
// matrix instruction and eight of the next one, which differ in the lowest bit of the lane group lh. Their places are
// disjoint where that bit decides the half of the 256 bytes of a cycle's banks: through the row's parity for rows of 128
// bytes (the place's bit 0), as bit 3 of the place for longer ones. E4M3 by plain pieces had 118 conflict cycles for 182 of reads.
template <int F, int XB>
__device__ __forceinline__ int x_place(int piece)
{
    if constexpr (F == kBF16) return piece;                                    // 4 j + lh
    else if constexpr (F == kFP8 && XB == 128) return piece >> 1 | (piece & 1) << 2;      // 2 lh + j
    else if constexpr (F == kFP8) return (piece >> 1 & 1) << 3 | (piece >> 3 & 1) << 2 | (piece >> 2 & 1) << 1 | (piece & 1);
    else return (piece & ~12) | (piece >> 2 & 1) << 3 | (piece >> 3 & 1) << 2;            // 16 h + 4 lh + j
}
// The piece at a place.
template <int F, int XB>
__device__ __forceinline__ int x_piece_at(int at)
{
    if constexpr (F == kBF16) return at;
    else if constexpr (F == kFP8 && XB == 128) return (at & 3) << 1 | at >> 2;
    else if constexpr (F == kFP8) return (at >> 3 & 1) << 1 | (at >> 2 & 1) << 3 | (at >> 1 & 1) << 2 | (at & 1);
    else return (at & ~12) | (at >> 2 & 1) << 3 | (at >> 3 & 1) << 2;
}

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

// ---------------------------------------------------------------------------------------------------------------
// Few rows an expert: bound by reading the weights. An item is up to MT pairs and P tiles of 16 weight rows; the items, chunk by
// chunk, are shared out evenly among as many blocks as are resident, so that none waits for another's second round. The WAVES
// waves of a block share K, a range each, and add their partial sums in LDS, in order, at an item's end. A wave's stages of all
// items of a chunk are one stream with D stages of loads in flight in registers (they hold several times what LDS
// could), which pass through wave-private LDS into the matrix layout: every load is row-contiguous, no barrier within an item.
// Waves with items of their own, without the sums in LDS, were slower (us, 16 tokens, two of 8 experts 28672x4096 bf16 285 -> 316,
// e4m3 145 -> 176). Measured (us, of the weights' bytes TB/s): 4 tokens, two of 8 experts 28672x4096 bf16 140, 6.7; e4m3 72, 6.5; INT4
// 44.5, 5.4 (weights alone 39, the rest scales, x and decode); one token, eight of 64 experts 2048x2048 e4m3 8.8, 3.8.
// ---------------------------------------------------------------------------------------------------------------
// WIDE (INT4 of an even number of groups): stages of 256 columns, whole 128-byte lines of the weights.
template <int F, int MT, bool WIDE>
struct StreamShape {
    static constexpr bool kI4F = F == kI4 || F == kI4ZP;
    static constexpr int kTiles = 2;                             // P
    static constexpr int kWaves = 4, kBlocks = 3;                // of a block, of a CU
    static constexpr int kAhead = 2;                             // D
    static constexpr int kCols = F == kBF16 ? 64 : (WIDE ? 256 : 128);          // columns of a stage
    static constexpr int kRowBytes = F == kBF16 ? 2 * kCols : (F == kFP8 ? kCols : kCols / 2);      // its bytes of a weight row
    static constexpr int kSteps = kCols / 32, kXRowBytes = 2 * kCols;
    static constexpr int kXLoadRows = kWave * 16 / kXRowBytes, kXRows = MT > kXLoadRows ? MT : kXLoadRows;
    static constexpr int kWBytes = kTiles * kTileRows * kRowBytes, kWaveBytes = kWBytes + kXRows * kXRowBytes;
};
template <int F, int MT, bool WIDE>
struct StreamSpace {
    using T = StreamShape<F, MT, WIDE>;
    __attribute__((aligned(16))) uint8_t place[T::kWaves][T::kWaveBytes];
    f32x4 part[T::kWaves][T::kTiles][kWave];
};

// `groups` items from column group `group0` on, of the pairs order[first .. first + held) of one expert.
template <int F, int MT, bool WIDE, bool PAST, bool GATED>
__device__ __forceinline__ void stream_items(const ExpertsParams& p, StreamSpace<F, MT, WIDE>& space, int expert, int first, int held,
                                             int order, int group0, int groups)
{
    using T = StreamShape<F, MT, WIDE>;
    constexpr bool I4 = T::kI4F;
    constexpr int P = T::kTiles, WAVES = T::kWaves, D = T::kAhead;
    constexpr int C = T::kCols, RB = T::kRowBytes, X = T::kSteps, L = RB * kTileRows / kChunkBytes;
    constexpr int H = I4 ? C / 128 : 1;               // INT4: groups of a stage
    constexpr int WP = RB / 16, WR = kWave / WP, XP = T::kXRowBytes / 16, XR = T::kXLoadRows, XL = T::kXRows / XR;
    constexpr int kOuts = GATED ? P / 2 : P, kOutCols = kOuts * kTileRows;

    const int lane = lane_id(), wave = wave_id(), ln = lane & 15, lh = lane >> 4;
    const int stages = (p.K + C - 1) / C, k0 = wave_begin(stages, wave, WAVES);      // this wave's stages; where there are none,
    const int mine_n = wave_begin(stages, wave + 1, WAVES) - k0;                     // one that reads nothing
    const int n = max(1, mine_n);
    const int columns = mine_n > 0 ? p.K : 0;
    const int64_t row0 = (int64_t)expert * p.N;
    uint8_t* mine = space.place[wave];

    struct Stage {
        u32x4 w[P][L], x[XL];
        // INT4: scales (WIDE: two) and zero points. Lane group lh loads those of the lh-th of four stages, in the first of the
        // four that the wave has: a stage of its own at a time brought the lines of 32 rows four times, most of them from
        // beyond the L2 by then (us, 4 tokens, two of 8 experts 4096x14336: 28.9 -> 26.7).
        uint32_t m[I4 ? P : 1], z[F == kI4ZP ? P : 1];
    };
    // the stream's next stage: stage `it` of item `ig`, the descriptors of whose tiles end with their rows
    int ig = 0, it = 0;
    __amdgpu_buffer_rsrc_t rw[P], rm[I4 ? P : 1], rz[F == kI4ZP ? P : 1];
    const auto aim = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < P; ++t) {
            const int rows = ig < groups ? max(0, tile_rows<GATED, P>(p, group0 + ig, t)) : 0;
            const uint32_t in = (uint32_t)__builtin_amdgcn_readfirstlane(rows);
            const int64_t row = row0 + (rows ? tile_row<GATED, P>(p, group0 + ig, t) : 0);
            rw[t] = make_rsrc(p.W + row * p.row_bytes, in * p.row_bytes);
            if constexpr (I4) rm[t] = make_rsrc(p.meta + row * p.G * 2, in * (uint32_t)p.G * 2u);
            if constexpr (F == kI4ZP) rz[t] = make_rsrc(p.zeros + row * p.zbytes, in * p.zbytes);
        }
    };
    // Unconditional loads (under a branch the compiler would wait for all that are on their way), out of range past the end.
    const uint32_t lw = (uint32_t)(lane / WP) * p.row_bytes + (uint32_t)(lane % WP) * 16u, wstep = (uint32_t)WR * p.row_bytes;
    const int cw = (lane % WP) * (C / WP), cx = (lane % XP) * 8;     // first column of the lane's 16 bytes
    const auto issue_w = [&](Stage& B) __attribute__((always_inline)) {
        const int kb = k0 + it, left = ig < groups ? columns - kb * C : 0;
        const uint32_t wo = cw < left ? lw + (uint32_t)kb * (uint32_t)RB : kOOB;
#pragma unroll
        for (int t = 0; t < P; ++t) {
#pragma unroll
            for (int i = 0; i < L; ++i) B.w[t][i] = ld16<PAST ? 2 : 0>(rw[t], wo + wstep * (uint32_t)i, 0u);
            if constexpr (I4) {
                const int at = ((kb & ~3) + lh) * H;
                const bool in = (it == 0 || (kb & 3) == 0) && left > 0 && at < p.G;
                const uint32_t lm = in ? ((uint32_t)ln * (uint32_t)p.G + (uint32_t)at) * 2u : kOOB;
                if constexpr (WIDE) B.m[t] = __builtin_amdgcn_raw_buffer_load_b32(rm[t], lm, 0u, 0);
                else B.m[t] = ld_u16(rm[t], lm, 0u);
                if constexpr (F == kI4ZP) B.z[t] = ld_u8(rz[t], in ? (uint32_t)ln * p.zbytes + (uint32_t)(at >> 1) : kOOB, 0u);
            }
        }
    };
    uint32_t xo[XL];
    const __amdgpu_buffer_rsrc_t xrs = make_rsrc(p.x, p.x_bytes);
    const auto issue_x = [&](Stage& B, int g, int t) __attribute__((always_inline)) {
        const int kb = k0 + t, left = g < groups ? columns - kb * C : 0;
#pragma unroll
        for (int i = 0; i < XL; ++i) B.x[i] = ld16<0>(xrs, cx < left ? xo[i] + (uint32_t)kb * (2u * C) : kOOB, 0u);
    };
    const auto next = [&]() __attribute__((always_inline)) {
        if (++it == n) it = 0, ++ig, aim();
    };

    const auto pair_of = [&](int i) { return p.R <= kWave ? __shfl(order, first + i, kWave) : p.order[first + i]; };
    // the weights' first loads go ahead of the chain order -> rows of x
    Stage buf[D];
    int pg[D], pt[D];
    aim();
#pragma unroll
    for (int d = 0; d < D; ++d) {
        pg[d] = ig, pt[d] = it;
        issue_w(buf[d]);
        next();
    }
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int r = i * XR + lane / XP, pair = pair_of(min(r, held - 1));
        const bool in = r < held && (uint32_t)pair < (uint32_t)p.R;
        xo[i] = in ? p.by_pairs.of((uint32_t)pair) * (uint32_t)(p.x_stride * 2) + (uint32_t)(lane % XP) * 16u : kOOB;
    }
#pragma unroll
    for (int d = 0; d < D; ++d) issue_x(buf[d], pg[d], pt[d]);
    const int last = pair_of(min(ln, held - 1)), pairs = ln < held ? last : -1;

    const auto w_at = [](int row, int piece) {
        return RB == 128 ? row * 128 + ((piece ^ (row & 7)) << 4) : row * 64 + ((piece ^ (row >> 1 & 3)) << 4);
    };
    const auto x_at = [](int row, int piece) {
        return T::kWBytes + row * T::kXRowBytes + ((x_place<F, T::kXRowBytes>(piece) ^ (row & 7)) << 4);
    };
    const uint32_t one2 = (uint32_t)__builtin_amdgcn_readfirstlane((int)kI4Take<F>);
    const u32x4 ones = {one2, one2, one2, one2};
    f32x4 acc[P];
#pragma unroll
    for (int t = 0; t < P; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t four[I4 ? P : 1][H];                    // the lane group's words of the four stages
    const auto consume = [&](const Stage& B, int kb, bool first_of_item) __attribute__((always_inline)) {
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < XL; ++i)
            *reinterpret_cast<u32x4*>(mine + x_at(i * XR + lane / XP, lane % XP)) = I4 ? i4_pair_x(B.x[i]) : B.x[i];
#pragma unroll
        for (int t = 0; t < P; ++t)
#pragma unroll
            for (int i = 0; i < L; ++i)
                *reinterpret_cast<u32x4*>(mine + t * kTileRows * RB + w_at(i * WR + lane / WP, lane % WP)) = B.w[t][i];
        wave_lds_order();
        const auto x_piece = [&](int piece) { return *reinterpret_cast<const u32x4*>(mine + x_at(ln & (T::kXRows - 1), piece)); };
        const auto w_piece = [&](int t, int piece) { return *reinterpret_cast<const u32x4*>(mine + t * kTileRows * RB + w_at(ln, piece)); };
        if constexpr (I4) {
            if (first_of_item || (kb & 3) == 0)
#pragma unroll
                for (int t = 0; t < P; ++t) i4_words_of<F, H>(B.m[t], F == kI4ZP ? B.z[F == kI4ZP ? t : 0] : 0u, lh, four[t]);
            const int from = (kb & 3) * 16 + ln;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                u32x4 a[4];
                f32x4 xs = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = x_piece(16 * h + 4 * lh + j);
#pragma unroll
                for (int j = 0; j < 4; ++j) xs = mfma_16x16x32(a[j], ones, xs);
#pragma unroll
                for (int t = 0; t < P; ++t) {
                    const u32x4 w = w_piece(t, 4 * h + lh);
                    const uint32_t m = (uint32_t)__shfl((int)four[t][h], from, kWave);
                    const float f = i4_factor<F>(m), sc = i4_scale<F>(m), z = i4_zero<F>(m);
                    f32x4 g = F == kI4 ? xs : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 4; ++j) g = mfma_16x16x32(a[j], i4_frag_paired(w[j], f), g);
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[t][v] = __builtin_fmaf(sc, F == kI4 ? g[v] : __builtin_fmaf(-z, xs[v], g[v]), acc[t][v]);
                }
                if (h + 1 < H) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            u32x4 a[X];
#pragma unroll
            for (int j = 0; j < X; ++j) a[j] = x_piece(F == kBF16 ? 4 * j + lh : 8 * (j >> 1) + 2 * lh + (j & 1));
#pragma unroll
            for (int t = 0; t < P; ++t) {
                u32x4 w[L];
#pragma unroll
                for (int i = 0; i < L; ++i) w[i] = w_piece(t, 4 * i + lh);
#pragma unroll
                for (int j = 0; j < X; ++j) {
                    const u32x4 v = w[F == kFP8 ? j >> 1 : j];
                    acc[t] = mfma_16x16x32(a[j], F == kBF16 ? v : (j & 1 ? fp8_frag(v.z, v.w) : fp8_frag(v.x, v.y)), acc[t]);
                }
            }
        }
    };

    // An item's end: partial tiles to LDS, then some of the waves add them and finish. Its operands are loaded an item ahead.
    uint32_t scale[P], bias[P];
    const __amdgpu_buffer_rsrc_t scales = make_rsrc(reinterpret_cast<const float*>(p.meta) + (F == kFP8 ? row0 : 0),
                                                    F == kFP8 ? (uint32_t)p.N * 4u : 0u);
    const __amdgpu_buffer_rsrc_t biases = make_rsrc(p.bias != nullptr ? p.bias + row0 : p.x,
                                                    p.bias != nullptr ? (uint32_t)p.N * 2u : 0u);
    const auto operands = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < P; ++t) {
            const uint32_t row = (uint32_t)(tile_row<GATED, P>(p, group0 + g, t) + ln);
            if constexpr (F == kFP8) scale[t] = __builtin_amdgcn_raw_buffer_load_b32(scales, row * 4u, 0u, 0);
            bias[t] = ld_u16(biases, row * 2u, 0u);
        }
    };
    operands(0);
    // column tile q of item g out of its finished sums
    const auto put = [&](int g, int q, const f32x4 (&sum)[GATED ? 2 : 1]) __attribute__((always_inline)) {
        const int col = (group0 + g) * kOutCols + q * kTileRows + ln;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int pair = __shfl(pairs, 4 * lh + c, kWave);
            float v[GATED ? 2 : 1];
#pragma unroll
            for (int h = 0; h < (GATED ? 2 : 1); ++h) {
                const int t = GATED ? 2 * q + h : q;
                v[h] = finish<F>(sum[h][c], F == kFP8 ? __uint_as_float(scale[t]) : 1.0f, bf16_to_f32(bias[t]));
            }
            const float o = GATED ? silu(v[0]) * v[GATED ? 1 : 0] : v[0];
            if ((uint32_t)pair < (uint32_t)p.R && col < p.cols)
                p.out[(int64_t)pair * p.out_stride + col] = (uint16_t)f32_to_bf16_out(o);
        }
    };
    const auto finish_item = [&](int g) __attribute__((always_inline)) {
        __syncthreads();                         // the last item's sums have been read
#pragma unroll
        for (int t = 0; t < P; ++t) space.part[wave][t][lane] = acc[t];
        __syncthreads();
        const int from = g * kOuts % WAVES;      // the items' finishes go round the waves
#pragma unroll
        for (int q = 0; q < kOuts; ++q) {
            if (wave != (from + q) % WAVES) continue;
            f32x4 sum[GATED ? 2 : 1];
#pragma unroll
            for (int h = 0; h < (GATED ? 2 : 1); ++h) {
                const int t = GATED ? 2 * q + h : q;
                sum[h] = space.part[0][t][lane];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) sum[h] += space.part[w][t][lane];
            }
            put(g, q, sum);
        }
#pragma unroll
        for (int t = 0; t < P; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        operands(g + 1);
    };

    const int all = groups * n;
    int g = 0, t = 0;                                // of the stage that is consumed next
    wait_loads<0>();                                 // the loop's waits then count its own order of loads alone
    for (int f = 0; f < all; f += D) {               // past the last stage the sums take zeros
#pragma unroll
        for (int d = 0; d < D; ++d) {
            consume(buf[d], k0 + t, t == 0);
            const int ng = ig, nt = it;
            issue_w(buf[d]);
            issue_x(buf[d], ng, nt);
            next();
            __builtin_amdgcn_sched_barrier(0);
            if (++t == n && f + d < all) finish_item(g), t = 0, ++g;
        }
    }
}

template <int F, int MT, bool WIDE, bool PAST, bool GATED>
__global__ void __launch_bounds__((StreamShape<F, MT, WIDE>::kWaves * kWave),
                                  (StreamShape<F, MT, WIDE>::kBlocks * StreamShape<F, MT, WIDE>::kWaves / 4))
experts_stream_kernel(const ExpertsParams p)
{
    __shared__ StreamSpace<F, MT, WIDE> space;
    const Chunks<MT> chunks(p);
    // below 2^32: at most kMostItems, and fewer than 2^12 blocks
    const uint32_t block = (uint32_t)xcd_contiguous((int)blockIdx.x, (int)gridDim.x), blocks = gridDim.x;
    const uint32_t items = (uint32_t)(chunks.count * p.tiles), end = share_begin(items, block + 1, blocks);
    for (uint32_t item = share_begin(items, block, blocks); item < end;) {
        const int chunk = (int)p.by_tiles.of(item), group0 = (int)item - chunk * p.tiles;
        const int groups = min(p.tiles - group0, (int)(end - item));
        const auto x = chunks.of(p, chunk);
        const int first = x.lo + (chunk - x.begin) * MT;
        stream_items<F, MT, WIDE, PAST, GATED>(p, space, x.expert, first, min(MT, x.hi - first), chunks.order,
                                                 group0, groups);
        item += (uint32_t)groups;
    }
    // rows of pairs without an expert, a block's width of columns at a time: as many as there are shared by all blocks (by one, the
    // four such pairs of 16 tokens were 10 of 85 us)
    const uint32_t width = StreamShape<F, MT, WIDE>::kWaves * kWave, pieces = ((uint32_t)p.cols + width - 1) / width;
    const uint64_t all = (uint64_t)(uint32_t)(p.R - chunks.rest_at) * pieces;
    const uint64_t last = share_begin<uint64_t>(all, block + 1, blocks);
    for (uint64_t i = share_begin<uint64_t>(all, block, blocks); i < last; ++i) {
        const uint32_t r = (uint32_t)i / pieces, col = ((uint32_t)i - r * pieces) * width + threadIdx.x;
        const int pair = p.order[chunks.rest_at + (int)r];
        if ((uint32_t)pair < (uint32_t)p.R && col < (uint32_t)p.cols) p.out[(int64_t)pair * p.out_stride + col] = 0;
    }
}

// ---------------------------------------------------------------------------------------------------------------
// More rows an expert: a block is BM pairs by 8 or 16 tiles of weight rows, its 4 or 8 waves 1 x 4, 2 x 2 or 2 x 4 parts of that. Two
// places in LDS are filled in turn, one barrier a stage. Up to 64 pairs (INT4 32), where reading the weights still counts, the
// stages come by way of registers with two of them in flight; larger blocks, whose sums take the registers, are filled straight
// from memory while the stage before is multiplied. A block is a unit, and chunks of one expert and columns are neighbours, so
// that they read the weights once: blocks that took several units, chunk by chunk, were slower (us, 64 tokens and two of 8
// experts 28672x4096 e4m3 169 -> 190). INT4 weights loaded by the lanes that use them, 64 bytes of a row at a time, without LDS
// were slower (16 tokens 86 -> 101). Measured, two of 8 experts 28672x4096: 4001 tokens e4m3 1635 us, 1150 TFLOP/s, bf16 1015 to 1055,
// INT4 840, with zero points 790 (a library bf16 product of 1000x28672x4096: 1156); 48 tokens e4m3 152, 64 bf16 290 (6.2 and
// 6.5 TB/s), 16 INT4 82 (5.9); 509 tokens, four of 64 experts 2816x2048 bf16 128 (5.8).
// ---------------------------------------------------------------------------------------------------------------
// SPLIT: two waves a part, which share the K of each stage. An INT4 wave has some 250 instructions a stage, as long as the stage's
// bytes take: alone on its SIMD, as where there are few blocks, it kept the loads waiting (us, 16 tokens, two of 8 experts
// 4096x14336: 57.3, two a part 48.2, without any products 43.4; 44.5 since the weights pass by the caches).
template <int F, int BM, bool WIDE, bool SPLIT>
struct TileShape {
    static constexpr bool kI4F = F == kI4 || F == kI4ZP;
    static constexpr int kCols = F == kBF16 || (F == kFP8 && BM >= 128) ? 64 : (WIDE ? 256 : 128);
    static constexpr int kRowBytes = F == kBF16 ? 2 * kCols : (F == kFP8 ? kCols : kCols / 2);
    static constexpr int kXRowBytes = 2 * kCols, kSteps = kCols / 32;
    static constexpr int kParts = BM == 256 ? 8 : 4, kTiles = 2 * kParts;     // of a block; its tiles of 16 weight rows
    static constexpr int kM = BM >= 128 ? 2 : 1, kN = kParts / kM;               // the parts' rows and columns
    static constexpr int kHalves = SPLIT ? 2 : 1, kWaves = kParts * kHalves;      // waves of a part, of a block
    static constexpr int kTM = BM / 16 / kM, kTN = kTiles / kN;
    static constexpr int kWBytes = kTiles * kTileRows * kRowBytes, kXBytes = BM * kXRowBytes;
    static constexpr bool kDirect = BM >= 128 || (kI4F && BM == 64);
    static constexpr int kBlocks = kParts == 8 ? 1 : (SPLIT || BM >= 64 || (WIDE && BM == 32) ? 2 : 3);      // of a CU
};

template <int F, int BM, bool WIDE, bool SPLIT, bool PAST, bool GATED>
__global__ void __launch_bounds__((TileShape<F, BM, WIDE, SPLIT>::kWaves * kWave),
                                  (TileShape<F, BM, WIDE, SPLIT>::kBlocks * TileShape<F, BM, WIDE, SPLIT>::kWaves / 4))
experts_tile_kernel(const ExpertsParams p)
{
    using T = TileShape<F, BM, WIDE, SPLIT>;
    constexpr bool I4 = T::kI4F;
    constexpr int C = T::kCols, RB = T::kRowBytes, XB = T::kXRowBytes, X = T::kSteps, TM = T::kTM, TN = T::kTN;
    constexpr int H = I4 ? C / 128 : 1;               // INT4: groups of a stage
    constexpr int WAVES = T::kWaves, WP = RB / 16, WR = kWave / WP, WL = T::kWBytes / (1024 * WAVES), XP = XB / 16, XR = kWave / XP;
    constexpr int XL = (T::kXBytes / 1024 + WAVES - 1) / WAVES;
    constexpr int XW = T::kXBytes / 1024 < WAVES ? T::kXBytes / 1024 : WAVES;    // waves that load x
    constexpr int kOutCols = (GATED ? T::kTiles / 2 : T::kTiles) * kTileRows;
    __shared__ __attribute__((aligned(16))) uint8_t slot0[T::kWBytes + T::kXBytes];
    __shared__ __attribute__((aligned(16))) uint8_t slot1[T::kWBytes + T::kXBytes];

    const int lane = lane_id(), wave = wave_id(), ln = lane & 15, lh = lane >> 4;
    constexpr int HALVES = T::kHalves, HW = H / HALVES;       // HW: groups of a stage that a wave has
    static_assert(!SPLIT || H == 2, "each half has a group");
    const int half = wave / (WAVES / HALVES), part = wave % (WAVES / HALVES);
    const int wm = part / T::kN, wn = part % T::kN;
    const int stages = (p.K + C - 1) / C;
    const auto w_piece = [](int r) { return RB == 128 ? r & 7 : r >> 1 & 3; };
    const int wr = lane / WP, xr = lane / XP;
    const uint32_t wpiece = (uint32_t)((lane % WP) ^ w_piece(wr)) * 16u;         // a load's first row is a multiple of 8
    const uint32_t one2 = (uint32_t)__builtin_amdgcn_readfirstlane((int)kI4Take<F>);
    const u32x4 ones = {one2, one2, one2, one2};

    const ExpertUnit u = unit_of<BM>(p);
    if (u.expert < 0) return;
    const int c0 = u.tile * kOutCols;
    if (u.expert == p.E) {
        zero_rows(p, u, c0, min(c0 + kOutCols, p.cols));
        return;
    }
    const int64_t row0 = (int64_t)u.expert * p.N;
    const bool busy = wm * TM * 16 < u.held;         // a part without pairs waits at the barriers only
    // A load of weights lies within a 16-row tile: its base is the wave's, an offset the lane's. x has an address a row.
    const uint8_t *wp[WL], *xp[XL];
    uint32_t wo[WL];
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int r0 = (wave * WL + i) * WR, t = r0 / kTileRows;
        const int rows = max(1, tile_rows<GATED, T::kTiles>(p, u.tile, t));
        wp[i] = p.W + (row0 + min(tile_row<GATED, T::kTiles>(p, u.tile, t), p.N - 1)) * p.row_bytes;
        wo[i] = (uint32_t)min(r0 % kTileRows + wr, rows - 1) * p.row_bytes;
    }
#pragma unroll
    for (int i = 0; i < XL; ++i) xp[i] = x_row(p, pair_at(p, u, (wave * XL + i) * XR + xr));
    // A stage's addresses; bytes past a row's end come from its last piece instead, and are cleared in the last stage.
    const auto w_from = [&](int s, int i) { return wp[i] + (wo[i] + min((uint32_t)s * RB + wpiece, p.row_bytes - 16u)); };
    const auto x_from = [&](int s, int i) {
        const int r = (wave * XL + i) * XR + xr;
        return xp[i] + min((uint32_t)s * XB + (uint32_t)x_piece_at<F, XB>((lane % XP) ^ (r & 7)) * 16u, (uint32_t)p.K * 2u - 16u);
    };
    // INT4: scales (WIDE: two) and zero points of four stages' groups for the wave's columns, as they are stored; lane group
    // lh has those of the lh-th. Loaded a round of four ahead: a stage at a time, one ahead, they came too late and each line of
    // theirs several times (us, zero points, two of 8 experts 4096x13696, 16 tokens 81.6 -> 62.7; 64 of 8 2048x1408, 32 tokens 27.6
    // -> 25.2; large calls -3 to 2%).
    struct Meta {
        uint32_t s[I4 ? TN : 1], z[F == kI4ZP ? TN : 1];
    };
    Meta ahead;
    // The lane group's words of the four stages; where there are no zero points scales as stored, cheaper to make words of again
    // and again than to keep and hand on two of them (us, 200 tokens, four of 60 experts 1003x3584: 34.0, 36.9 as words; with
    // zero points, words 39.7, as stored 41.0).
    constexpr int kWords = F == kI4ZP ? HW : 1;
    uint32_t four[I4 ? TN : 1][kWords];
    const auto meta_load = [&](Meta& m, int s) __attribute__((always_inline)) {
        if constexpr (I4) {
            s = min(s + lh, stages - 1);
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const int i = wn * TN + t, rows = max(1, tile_rows<GATED, T::kTiles>(p, u.tile, i));
                const int64_t first = row0 + min(tile_row<GATED, T::kTiles>(p, u.tile, i), p.N - 1);
                const uint32_t r = (uint32_t)min(ln, rows - 1);
                const uint8_t* at = p.meta + first * p.G * 2 + (r * (uint32_t)p.G + (uint32_t)(s * H)) * 2u;
                if constexpr (WIDE) m.s[t] = *reinterpret_cast<const uint32_t*>(at);
                else m.s[t] = *reinterpret_cast<const uint16_t*>(at);
                if constexpr (F == kI4ZP) m.z[t] = p.zeros[first * p.zbytes + (r * p.zbytes + (uint32_t)(s * H >> 1))];
            }
        }
    };
    const auto take_meta = [&]() __attribute__((always_inline)) {
        if constexpr (I4)
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const int g = SPLIT ? half : 0;                  // the first of the wave's groups
                if constexpr (F == kI4ZP) i4_words_of<F, HW>(ahead.s[t] >> 16 * g, ahead.z[t], lh * H + g, four[t]);
                else four[t][0] = ahead.s[t] >> 16 * g;
            }
    };
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto get_x = [&](const uint8_t* slot, int i, int j) {
        const int r = (wm * TM + i) * 16 + ln;
        const int piece = F == kBF16 ? 4 * j + lh : (F == kFP8 ? 8 * (j >> 1) + 2 * lh + (j & 1) : 16 * (j >> 2) + 4 * lh + (j & 3));
        return *reinterpret_cast<const u32x4*>(slot + T::kWBytes + r * XB + ((x_place<F, XB>(piece) ^ (r & 7)) << 4));
    };
    const auto get_w = [&](const uint8_t* slot, int t, int i) {
        const int r = (wn * TN + t) * 16 + ln;
        return *reinterpret_cast<const u32x4*>(slot + r * RB + (((4 * i + lh) ^ w_piece(r)) << 4));
    };
    const auto use = [&](const uint8_t* slot, int of_four) __attribute__((always_inline)) {
        if constexpr (I4) {
#pragma unroll
            for (int h = 0; h < HW; ++h) {
                const int hg = SPLIT ? half : h;
                u32x4 a[TM][4], w[TN];
                f32x4 xs[TM];
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[i][j] = get_x(slot, i, 4 * hg + j);
#pragma unroll
                for (int t = 0; t < TN; ++t) w[t] = get_w(slot, t, hg);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    xs[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 4; ++j) xs[i] = mfma_16x16x32(a[i][j], ones, xs[i]);
                }
#pragma unroll
                for (int t = 0; t < TN; ++t) {
                    uint32_t m = (uint32_t)__shfl((int)four[t][F == kI4ZP ? h : 0], of_four * 16 + ln, kWave);
                    if constexpr (F == kI4) m = i4_word_of<F>(h ? m >> 16 : m & 0xFFFFu, 8u);
                    const float f = i4_factor<F>(m), sc = i4_scale<F>(m), z = i4_zero<F>(m);
                    f32x4 g[TM];
#pragma unroll
                    for (int i = 0; i < TM; ++i) g[i] = F == kI4 ? xs[i] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const u32x4 b = T::kDirect ? i4_frag(w[t][j], f) : i4_frag_paired(w[t][j], f);     // x as it was stored
#pragma unroll
                        for (int i = 0; i < TM; ++i) g[i] = mfma_16x16x32(a[i][j], b, g[i]);
                    }
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            acc[i][t][v] = __builtin_fmaf(sc, F == kI4 ? g[i][v] : __builtin_fmaf(-z, xs[i][v], g[i][v]), acc[i][t][v]);
                }
                if (h + 1 < HW) __builtin_amdgcn_sched_barrier(0);
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
    // The last stage of a K that is no multiple of its columns: what lies past the rows' ends is 0 in both operands. (INT4
    // WIDE has whole stages.)
    const auto clear_past = [&](uint8_t* slot, int left) __attribute__((always_inline)) {
        constexpr int kWCols = F == kFP8 ? 16 : 8;
        const u32x4 none = {0, 0, 0, 0};
        for (int e = (int)threadIdx.x; e < T::kTiles * kTileRows * WP; e += WAVES * kWave) {
            const int r = e / WP, at = e % WP;
            if ((at ^ w_piece(r)) * kWCols >= left) *reinterpret_cast<u32x4*>(slot + r * RB + at * 16) = none;
        }
        for (int e = (int)threadIdx.x; e < BM * XP; e += WAVES * kWave) {
            const int r = e / XP, at = e % XP;
            if (x_piece_at<F, XB>(at ^ (r & 7)) * 8 >= left) *reinterpret_cast<u32x4*>(slot + T::kWBytes + r * XB + at * 16) = none;
        }
        __syncthreads();
    };
    constexpr int kRound = I4 ? 4 : 2;               // stages of a round of the loops
    const auto multiply = [&](uint8_t* slot, int s, int d, bool last) __attribute__((always_inline)) {
        if (!I4 && last && p.K - s * C < C) clear_past(slot, p.K - s * C);
        if (busy) {
            if constexpr (F == kFP8) __builtin_amdgcn_s_setprio(1);      // ahead of the blocks that fetch: 1674 -> 1646 us at 4001
            use(slot, d);                                                // tokens; INT4 1% slower so, BF16 even
            if constexpr (F == kFP8) __builtin_amdgcn_s_setprio(0);
        }
        if (I4 && d == kRound - 1) take_meta();
    };

    meta_load(ahead, 0);
    take_meta();
    if constexpr (T::kDirect) {
        static_assert(!T::kDirect || XW == WAVES, "every wave has a part of x");
        const auto issue = [&](uint8_t* slot, int s) __attribute__((always_inline)) {
            if (s >= stages) return;
#pragma unroll
            for (int i = 0; i < WL; ++i) lds_copy16(slot + (wave * WL + i) * 1024, w_from(s, i));
#pragma unroll
            for (int i = 0; i < XL; ++i) lds_copy16(slot + T::kWBytes + (wave * XL + i) * 1024, x_from(s, i));
        };
        const auto stage = [&](uint8_t* mine, uint8_t* next, int s, int d) __attribute__((always_inline)) {
            wait_loads<0>();
            __syncthreads();                         // this stage has arrived, the other place is read
            issue(next, s + 1);
            if (d == 0) meta_load(ahead, s + kRound);
            multiply(mine, s, d, true);
        };
        issue(slot0, 0);
        for (int s = 0; s < stages; s += kRound)
#pragma unroll
            for (int d = 0; d < kRound; ++d)
                if (s + d < stages) stage(d & 1 ? slot1 : slot0, d & 1 ? slot0 : slot1, s + d, d);
    } else {
        struct Stage {
            u32x4 w[WL], x[XL];
        };
        // Unconditional: past the last stage it reads that one again, waves without a part of x their neighbours' rows.
        const auto load = [&](auto once, Stage& B, int s) __attribute__((always_inline)) {
            s = min(s, stages - 1);
#pragma unroll
            for (int i = 0; i < WL; ++i) {
                const u32x4* from = reinterpret_cast<const u32x4*>(w_from(s, i));
                B.w[i] = decltype(once)::value ? __builtin_nontemporal_load(from) : *from;
            }
#pragma unroll
            for (int i = 0; i < XL; ++i) B.x[i] = *reinterpret_cast<const u32x4*>(x_from(s, i));
        };
        const auto store = [&](uint8_t* slot, const Stage& B) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < WL; ++i) *reinterpret_cast<u32x4*>(slot + (wave * WL + i) * 1024 + lane * 16) = B.w[i];
            if (XW == WAVES || wave < XW) {
#pragma unroll
                for (int i = 0; i < XL; ++i)
                    *reinterpret_cast<u32x4*>(slot + T::kWBytes + (wave * XL + i) * 1024 + lane * 16) = I4 ? i4_pair_x(B.x[i]) : B.x[i];
            }
        };
        const auto run = [&](auto once) __attribute__((always_inline)) {
            asm volatile("" ::"i"((int)decltype(once)::value) : "memory");
            Stage buf[2];
            load(once, buf[0], 0);
            load(once, buf[1], 1);
            int s = 0;
            wait_loads<0>();                             // the loop's waits then count its own order of loads alone
            for (; s + kRound < stages; s += kRound) {
#pragma unroll
                for (int d = 0; d < kRound; ++d) {
                    uint8_t* slot = d & 1 ? slot1 : slot0;
                    store(slot, buf[d & 1]);             // what was there is read: two stages ago, before the last barrier
                    if (d == 0) meta_load(ahead, s + kRound);      // ahead of the loads that stay on their way
                    load(once, buf[d & 1], s + d + 2);
                    block_lds_order();
                    multiply(slot, s + d, d, false);
                }
            }
#pragma unroll
            for (int d = 0; d < kRound; ++d)
                if (s + d < stages) {
                    uint8_t* slot = d & 1 ? slot1 : slot0;
                    store(slot, buf[d & 1]);
                    if (d + 2 < kRound && s + d + 2 < stages) load(once, buf[d & 1], s + d + 2);
                    block_lds_order();
                    multiply(slot, s + d, d, true);
                }
        };
        // Weights that no other block reads pass by the caches (us, two of 8 experts 28672x4096, 64 tokens bf16 323 -> 293, 48 e4m3
        // 170 -> 152; 509 tokens, four of 64 experts 2816x2048 bf16 145 -> 128), those of several chunks do not: bf16, 300 tokens
        // 429, past the caches 527. Nor do rows whose lines two stages share (INT4 of 11 groups, 32 tokens, eight of 64 experts
        // 2048x1408 24.7 -> 26.0). For INT4 the host decides (PAST): two loops would share too few registers.
        if (I4 ? PAST : __builtin_amdgcn_readfirstlane(u.chunks) == 1 && p.row_bytes % 128 == 0) run(std::true_type{});
        else run(std::false_type{});
    }
    if constexpr (HALVES == 2) {
        // the second half's sums go to the first's, by way of the places in LDS
        f32x4* sums = reinterpret_cast<f32x4*>(slot0) + part * (TM * TN * kWave) + lane;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < TN; ++t)
                if (half == 1) sums[(i * TN + t) * kWave] = acc[i][t];
        __syncthreads();
        if (half == 1) return;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < TN; ++t) acc[i][t] += sums[(i * TN + t) * kWave];
    }
    if (!busy) return;

    // out: the pairs of the wave's rows, the columns' scales and biases
    int pairs[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = (wm * TM + i) * 16 + ln;
        pairs[i] = m < u.held ? p.order[u.first + m] : -1;
    }
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
            const int pair = __shfl(pairs[i], 4 * lh + c, kWave);
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

// Launches of a format's kernels; p as the entry point fills it. 0, -2 (more blocks than a launch has) or a hipError_t.
// Sets what depends on the kernel's shape; the units that these sizes can need.
inline int64_t plan_experts(ExpertsParams& p, int BM, int unit_cols)
{
    p.tiles = (int)(((int64_t)p.cols + unit_cols - 1) / unit_cols);
    p.by_tiles = Divisor((uint32_t)p.tiles);
    const int64_t most = most_chunks(p.R, p.E, BM);
    p.most = (int)most;
    return most * p.tiles;
}
template <int F, int MT, bool WIDE, bool GATED>
int launch_stream(ExpertsParams p, hipStream_t st)
{
    using T = StreamShape<F, MT, WIDE>;
    const int64_t items = plan_experts(p, MT, (GATED ? T::kTiles / 2 : T::kTiles) * kTileRows);
    const int64_t resident = T::kBlocks * device_facts().cus;
    // Weights pass by the caches where a stage has whole lines; lines that two stages share are kept for the second (us, 4 tokens, two
    // of 8 experts 28672x4112 e4m3 96, past the caches 120; 28672x4096 83 and 76; INT4 of 33 groups 62 and 69). That an expert has
    // several chunks, which read its matrix again, the host cannot know; then kept lines are the better choice (us, kept / past: 12
    // pairs of one of 8 experts e4m3 28672x4096 55/62, 4096x14336 35/41; 40 of one bf16 100/116 and 71/98; 8 of one INT4 28.5/28.6 and
    // 17.2/17.5; spread evenly e4m3 167/146 and 83/73, bf16 318/278 and 157/139, INT4 92/81 and 44.3/44.1).
    const auto go = [&](auto past) {
        hipLaunchKernelGGL((experts_stream_kernel<F, MT, WIDE, decltype(past)::value, GATED>),
                           dim3((uint32_t)(items < resident ? items : resident)), dim3(T::kWaves * kWave), 0, st, p);
        return (int)hipGetLastError();
    };
    if constexpr (T::kI4F) return go(std::bool_constant<WIDE>{});
    else return p.row_bytes % 128 == 0 ? go(std::true_type{}) : go(std::false_type{});
}
// Where reading weights bounds a call: its items of two tiles fit the shares, a descriptor spans x, and a wave's quarter of a row
// is two lines or more.
inline bool streams(const ExpertsParams& p, int64_t pairs)
{
    return p.R <= pairs && p.x_bytes != 0 && p.row_bytes >= 1024 && most_chunks(p.R, p.E, 4) * ((p.cols + 15) / 16) <= kMostItems;
}
template <int F, int BM, bool WIDE, bool SPLIT, bool GATED>
int64_t tile_units(ExpertsParams& p)
{
    using T = TileShape<F, BM, WIDE, SPLIT>;
    return plan_experts(p, BM, (GATED ? T::kTiles / 2 : T::kTiles) * kTileRows);
}
template <int F, int BM, bool WIDE, bool SPLIT, bool GATED, bool PAST = false>
int launch_tiles(ExpertsParams p, hipStream_t st)
{
    using T = TileShape<F, BM, WIDE, SPLIT>;
    const int64_t units = tile_units<F, BM, WIDE, SPLIT, GATED>(p);
    if (units > kMostBlocks) {
        // the format's largest blocks, of which there are the fewest, are what the contract counts
        constexpr int kLargest = F == kBF16 ? 256 : 128;
        if constexpr (BM < kLargest) return launch_tiles<F, kLargest, false, false, GATED>(p, st);
        return -2;
    }
    hipLaunchKernelGGL((experts_tile_kernel<F, BM, WIDE, SPLIT, PAST, GATED>), dim3((uint32_t)units), dim3(T::kWaves * kWave), 0, st, p);
    return (int)hipGetLastError();
}
// The form of a call goes by the pairs an expert has on average, all that the host knows of them: it counts pairs without an expert
// too, and a call most of whose pairs are such (experts that lie on several GPUs) takes blocks that are too large for it (us, 8 experts
// of 32 pairs each, alone / beside seven times as many without one: e4m3 28672x4096 153/240, 4096x14336 96/190; bf16 299/441, 156/321;
// INT4 134/290, 65/160, with zero points 143/306, 79/169; of 4 pairs each e4m3 143/146, 69/94; bf16 288/289, 145/165; INT4 89/123,
// 51/64). Each side of a border measured, on these matrices alone
// (us a call; e8: two of 8 experts gated 28672x4096 a token, d8: 4096x14336, e64: eight of 64, gated 2816x2048, d64: 2048x1408; the
// pairs an expert in front):
//   E4M3  MT 4 / 16    0.25 e8 37/42 d8 21/48 e64 17.7/17.9, 0.5 e8 56/54 d8 31/50 e64 25.7/27.1, 0.75 e64 32.6/30.0,
//                      1 e8 72/79 d8 38/52 e64 34.6/29.6, 1.5 e8 91/96 d8 51/54, 2 e8 142/132 d8 75/62 e64 50/47
//         16 / 32      4 d8 69/70 e64 55/56, 5 e8 129/130 d8 63/65, 6 d8 109/81 d64 31/35, 16 e8 164/148; d64 10 38/41
//         32 / 64, few units: 16 d8 84/95, 20 121/98, 38 123/100, 50 120/152; many: 19 e64 65/74, 31 79/87
//         32 / 128     50 e64 99/97, 60 e8 260/265 d8 160/195, 64 e64 112/113, 75 e8 293/264, 88 e64 134/121
//   BF16  MT 8 / 16    0.25 e64 18.2/18.7, 1 e64 56.9/56.7       MT 16 / 32 2 e64 90/96,
//                      4 e8 281/284 d8 140/174 e64 109/122, 6 e8 328/285 d8 191/157 e64 120/115
//         32 / 64      few units: 16 d8 173/175, 20 223/175, 25 210/171; many: 19 e64 119/124, 25 e8 317/300 d64 63/70,
//                      31 e64 136/132
//         64 / 128     62 e64 155/162, 75 e8 428/388 d8 240/281, 88 e64 182/182, 100 e8 480/428
//         128 / 256    125 e64 199/211, 150 e8 539/483 d8 303/371, 187 e64 244/254, 250 e8 679/623
//   INT4  MT 4 / 16    0.5 e8 39.1/40.8 d8 24.0/56, 1 e8 47.7/53.0 e64 25.6/24.5, 2 e8 91.6/85.6 d8 50.9/54.4 e64 38.0/37.9
//         16 / 32      20 e8 157/164 d8 88/114 d64 (zp) 38/39, 25 e64 73/72 d64 (zp) 43.6/39.5, 28 e8 189/191
//         32 / 64      50 e8 240/259 e64 111/109, 64 e8 289/268 e64 128/123
//         blocks of 16, waves alone / two a part: d8 4 57.3/48.2, 13 of 60 1003x3584 33.7/32.6 (zp 39.5/34.6), 4096x3584 105/111 (zp
//                      121/115), 4 e8 89/91 (zp 98/95), 8 e64 42.3/43.8 (zp 48.6/45.4)
//         16, weights kept / past the caches: 4 e8 88/82 d8 48/45, 8 e64 42/38 (zp 45/43), 13 of 60 1003x3584 (zp) 35.1/34.1,
//                      20 e64 58/58 e8 143/149 d8 76/79
//         64 / 128     125 e8 418/433 e64 171/165 (zp 445/448, 188/175), 175 e8 533/546, 250 e8 746/706 d8 390/397 (zp 803/740,
//                      428/422), 1000 e8 2659/2287 (zp 2891/2441)
//   rows of 512 bytes, MT 4 / 16: E4M3 1024x512 11.4/7.9; of 704: INT4 d64 14.4/9.0; of 1024: INT4 e64 above; BF16 1024x512
//   12.4/11.8; of 1408: E4M3 d64 14.2/9.7
// Few units: three a CU or fewer by the most that these sizes can need, of which a usual call has one or two a CU, as many as
// blocks of 64 fit. An expert's second chunk is then another block on some of the CUs, and the call takes as long as those. Many units
// even that out.
template <int F, bool GATED>
int launch_format(ExpertsParams p, hipStream_t st)
{
    const int64_t R = p.R, E = p.E, few_units = 3 * device_facts().cus;
    if constexpr (F == kI4 || F == kI4ZP) {
        const auto few = [&](auto wide) {
            constexpr bool WIDE = decltype(wide)::value;
            if (streams(p, E)) return launch_stream<F, 4, WIDE, GATED>(p, st);
            const auto sixteen = [&](auto split) {
                constexpr bool SPLIT = decltype(split)::value;
                return WIDE && R <= 14 * E ? launch_tiles<F, 16, WIDE, SPLIT, GATED, WIDE>(p, st)
                                           : launch_tiles<F, 16, WIDE, SPLIT, GATED>(p, st);
            };
            if constexpr (WIDE) {
                const bool split = F == kI4ZP || tile_units<F, 16, true, true, GATED>(p) <= few_units;
                if (R <= 22 * E && split) return sixteen(std::true_type{});
            }
            if constexpr (!WIDE || F == kI4)
                if (R <= 22 * E) return sixteen(std::false_type{});
            return launch_tiles<F, 32, WIDE, false, GATED>(p, st);
        };
        if (R <= 56 * E) return p.G % 2 == 0 && aligned(p.meta, 4) ? few(std::true_type{}) : few(std::false_type{});
        if (R <= 192 * E) return launch_tiles<F, 64, false, false, GATED>(p, st);
        return launch_tiles<F, 128, false, false, GATED>(p, st);
    } else if constexpr (F == kFP8) {
        if (streams(p, p.row_bytes >= 4096 ? E * 3 / 2 : E / 2)) return launch_stream<F, 4, false, GATED>(p, st);
        if (R <= (p.row_bytes < 2048 ? 12 : 5) * E) return launch_tiles<F, 16, false, false, GATED>(p, st);
        if (R <= 64 * E) {
            if (R > 16 * E && R <= 40 * E && tile_units<F, 64, false, false, GATED>(p) <= few_units)
                return launch_tiles<F, 64, false, false, GATED>(p, st);
            return launch_tiles<F, 32, false, false, GATED>(p, st);
        }
        return launch_tiles<F, 128, false, false, GATED>(p, st);
    } else {
        if (streams(p, E)) return launch_stream<F, 8, false, GATED>(p, st);
        if (streams(p, 5 * E)) return launch_stream<F, 16, false, GATED>(p, st);
        const int64_t most32 = tile_units<F, 64, false, false, GATED>(p) <= few_units ? 16 : 28;
        if (R <= most32 * E) return launch_tiles<F, 32, false, false, GATED>(p, st);
        if (R <= 80 * E) return launch_tiles<F, 64, false, false, GATED>(p, st);
        if (R <= 192 * E) return launch_tiles<F, 128, false, false, GATED>(p, st);
        return launch_tiles<F, 256, false, false, GATED>(p, st);
    }
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
