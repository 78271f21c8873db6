// Low-rank adapters of many requests beside a shared projection.
//
//   out[m, n] = bf16( y[m, n] + s_a sum_r B_a[n, r] h[m, j(n) R + r] ),   h[m, :] = A_a x[m],   a = ids[m]
//
// j(n) is the slice of the projection that output n belongs to (q | k | v, gate | up): each slice has its own R rows of A.
// Rows without an adapter keep y. Every adapter in use is read once for each 16 rows that share it; the products are on
// v_mfma_f32_16x16x32_bf16 with the adapter's rows as one operand and the 16 rows as the other.
//   * Two launches: h has to be whole before any output. The first leaves partial sums of h over pieces of K in the workspace
//     (added in order by the second: no atomics), so that few rows and low ranks still fill the chip.
//   * The rows that share an adapter are found by each block from ids itself (row_chunks): ids are on the device, and
//     nothing has to be sorted or counted before the call.
//   * h goes to the second product as two bf16 terms (value and remainder, 16 bits together), so that out has the one
//     rounding at the end that matters.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "gemv_kernel.h"
#include "paia_gemv.h"

namespace paia {

constexpr int kLoraBlock = 256, kLoraWaves = kLoraBlock / kWave;
constexpr int kLoraRows = 256;           // rows of a launch
constexpr int kChunk = 16;               // rows that share a pass over an adapter
constexpr int kMaxSlices = 8, kMaxPieces = 8;
constexpr int kShrinkUnits = 512;        // blocks aimed at by the first product's split of K
constexpr int kShrinkAhead = 4;          // steps of K whose loads a wave has in flight
constexpr int kTilesPerWave = 4;         // tiles of 16 outputs a wave takes of a unit

struct LoraParams {
    const uint16_t *x, *A, *B, *y;
    uint16_t* out;
    const int32_t* ids;
    const float* scaling;                // fp32 [adapters] or null
    float* part;                         // [piece][row][h_stride]
    int64_t x_stride, y_stride, out_stride;
    int M, K, N, R, adapters, slices, h_rows, h_stride;     // h_rows: slices * R; h_stride: that rounded up to 16
    int first[kMaxSlices + 1];           // first output of each slice, N at the end
    int unit_first[kMaxSlices + 1];      // first expand unit of each slice within a chunk
    bool wide;                           // out and y take 8-byte accesses
};

// The rows in the order of their adapters, cut into chunks of at most kChunk rows of one adapter; rows without one last.
struct RowChunks {
    int key[kLoraRows];                  // adapter, INT_MAX without
    int order[kLoraRows];                // rows by (key, row)
    int start[kLoraRows + 1];            // first place in `order` of each chunk
    int marks[kLoraWaves];
    int count;
};
__device__ __forceinline__ void row_chunks(const LoraParams& p, RowChunks* s)
{
    const int t = (int)threadIdx.x;
    int key = INT_MAX;
    if (t < p.M) {
        const int id = p.ids[t];
        if (id >= 0 && id < p.adapters) key = id;
        s->key[t] = key;
    }
    __syncthreads();
    int place = 0, same = 0;
    for (int j = 0; j < p.M; ++j) {
        const int k = s->key[j];
        same += k == key && j < t;
        place += k < key;
    }
    place += same;
    if (t < p.M) s->order[place] = t | (same % kChunk == 0 ? 1 << 16 : 0);
    __syncthreads();
    const int row = t < p.M ? s->order[t] : 0;
    const bool begins = row >> 16;
    const uint64_t mark = __ballot(begins);
    if (lane_id() == 0) s->marks[wave_id()] = __popcll(mark);
    __syncthreads();
    int before = 0, count = 0;
#pragma unroll
    for (int w = 0; w < kLoraWaves; ++w) {
        before += w < wave_id() ? s->marks[w] : 0;
        count += s->marks[w];
    }
    if (begins) s->start[before + __popcll(mark & ((1ull << lane_id()) - 1))] = t;
    if (t < p.M) s->order[t] = row & 0xFFFF;
    if (t == 0) s->start[count] = p.M, s->count = count;
    __syncthreads();
}

// Pieces of K: as many as give the chip its blocks for the chunks at hand, each at least 256 columns.
__device__ __forceinline__ int k_pieces(const LoraParams& p, int chunks)
{
    const int units = chunks * (p.h_stride / 16);
    const int most = min(kMaxPieces, (p.K + 255) / 256);
    return max(1, min(most, kShrinkUnits / units));
}

__device__ __forceinline__ f32x4 lora_mfma(const u32x4 a, const u32x4 b, const f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ u32x4 load16_if(const uint16_t* p, bool take)
{
    return take ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
}

// What a value keeps beyond its bf16 rounding; nothing where that is not finite.
__device__ __forceinline__ float rest(float v, uint32_t rounded)
{
    return fabsf(__uint_as_float(rounded)) < 3.4e38f ? v - __uint_as_float(rounded) : 0.0f;
}

// h: a unit is (chunk, 16 rows of A, piece of K); the block's waves take its steps of 32 columns in turn.
__global__ void __launch_bounds__(kLoraBlock) lora_shrink_kernel(const LoraParams p)
{
    __shared__ RowChunks rows;
    __shared__ f32x4 sums[kLoraWaves][kWave];
    row_chunks(p, &rows);
    const int tiles = p.h_stride / 16, pieces = k_pieces(p, rows.count), steps = (p.K + 31) / 32;
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    for (int unit = (int)blockIdx.x; unit < rows.count * tiles * pieces; unit += (int)gridDim.x) {
        const int piece = unit % pieces, tile = unit / pieces % tiles, chunk = unit / pieces / tiles;
        const int start = rows.start[chunk], held = rows.start[chunk + 1] - start;
        const int m = rows.order[start + min(n, held - 1)], id = rows.key[rows.order[start]];
        if (id == INT_MAX) break;        // the last chunks: rows without an adapter
        const int r = tile * 16 + n;
        const uint16_t* a = p.A + ((int64_t)id * p.h_rows + min(r, p.h_rows - 1)) * p.K + 8 * g;
        const uint16_t* x = p.x + m * p.x_stride + 8 * g;
        const int s0 = (int)((int64_t)steps * piece / pieces), s1 = (int)((int64_t)steps * (piece + 1) / pieces);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = s0 + wave; s < s1; s += kShrinkAhead * kLoraWaves) {
            u32x4 u[kShrinkAhead], v[kShrinkAhead];
#pragma unroll
            for (int i = 0; i < kShrinkAhead; ++i) {
                const int at = s + i * kLoraWaves;
                const bool in = at < s1 && 32 * at + 8 * g < p.K;
                u[i] = load16_if(a + 32 * at, in && r < p.h_rows);
                v[i] = load16_if(x + 32 * at, in && n < held);
            }
#pragma unroll
            for (int i = 0; i < kShrinkAhead; ++i) acc = lora_mfma(u[i], v[i], acc);
        }
        sums[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && n < held) {
#pragma unroll
            for (int w = 1; w < kLoraWaves; ++w) acc += sums[w][lane];
            *reinterpret_cast<f32x4*>(p.part + ((int64_t)piece * p.M + m) * p.h_stride + tile * 16 + 4 * g) = acc;
        }
        __syncthreads();
    }
}

// out: a unit is (chunk, slice, kLoraWaves * kTilesPerWave tiles of 16 outputs of the slice). STEPS: 32-value steps of R.
template <int STEPS, bool WIDE>
__global__ void __launch_bounds__(kLoraBlock) lora_expand_kernel(const LoraParams p)
{
    __shared__ RowChunks rows;
    row_chunks(p, &rows);
    const int pieces = k_pieces(p, rows.count), per_chunk = p.unit_first[p.slices];
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    for (int unit = (int)blockIdx.x; unit < rows.count * per_chunk; unit += (int)gridDim.x) {
        const int chunk = unit / per_chunk, u = unit % per_chunk;
        int slice = 0;
        while (u >= p.unit_first[slice + 1]) ++slice;
        const int start = rows.start[chunk], held = rows.start[chunk + 1] - start;
        const int m = rows.order[start + min(n, held - 1)], id = rows.key[rows.order[start]];
        const bool live = n < held, bare = id == INT_MAX;
        if (bare && p.out == p.y && p.out_stride == p.y_stride) continue;
        const int end = p.first[slice + 1];
        const int n0 = p.first[slice] + ((u - p.unit_first[slice]) * kLoraWaves + wave) * kTilesPerWave * 16;
        if (n0 >= end) continue;

        u32x4 b[kTilesPerWave][STEPS];
        const uint16_t* B = p.B + ((int64_t)(bare ? 0 : id) * p.N) * p.R;
#pragma unroll
        for (int t = 0; t < kTilesPerWave; ++t)
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int row = n0 + 16 * t + n, r = 32 * s + 8 * g;
                b[t][s] = load16_if(B + (int64_t)min(row, end - 1) * p.R + r, !bare && row < end && r < p.R);
            }
        // the lane's values of h: the pieces' sums in order, times the adapter's factor, as value and remainder
        u32x4 hi[STEPS], lo[STEPS];
        const float factor = bare || p.scaling == nullptr ? 1.0f : p.scaling[id];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int r = 32 * s + 8 * g;
            float h[8] = {};
            if (live && !bare && r < p.R) {
                const float* src = p.part + (int64_t)m * p.h_stride + slice * p.R + r;
                for (int i = 0; i < pieces; ++i, src += (int64_t)p.M * p.h_stride) {
                    const f32x4 u0 = reinterpret_cast<const f32x4*>(src)[0], u1 = reinterpret_cast<const f32x4*>(src)[1];
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] += u0[e], h[4 + e] += u1[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = h[2 * e] * factor, w = h[2 * e + 1] * factor;
                hi[s][e] = pack_bf16x2(v, w);
                lo[s][e] = pack_bf16x2(rest(v, hi[s][e] << 16), rest(w, hi[s][e] & 0xFFFF0000u));
            }
        }
        const uint16_t* y = p.y + m * p.y_stride;
        uint16_t* out = p.out + m * p.out_stride;
#pragma unroll
        for (int t = 0; t < kTilesPerWave; ++t) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                acc = lora_mfma(b[t][s], lo[s], acc);
                acc = lora_mfma(b[t][s], hi[s], acc);
            }
            const int at = n0 + 16 * t + 4 * g;
            if (!live || at >= end) continue;
            if (WIDE && at + 4 <= end) {
                uint2 v = *reinterpret_cast<const uint2*>(y + at);
                v.x = bare ? v.x : pack_bf16x2(bf16_to_f32(v.x & 0xFFFFu) + acc[0], __uint_as_float(v.x & 0xFFFF0000u) + acc[1]);
                v.y = bare ? v.y : pack_bf16x2(bf16_to_f32(v.y & 0xFFFFu) + acc[2], __uint_as_float(v.y & 0xFFFF0000u) + acc[3]);
                *reinterpret_cast<uint2*>(out + at) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e < end)
                        out[at + e] = bare ? y[at + e] : (uint16_t)f32_to_bf16_out(bf16_to_f32(y[at + e]) + acc[e]);
            }
        }
    }
}

static int launch_lora(const LoraParams& p, hipStream_t st)
{
    const int cap = device_facts().cus * 4;
    const int64_t shrink = (int64_t)p.M * (p.h_stride / 16) * kMaxPieces, expand = (int64_t)p.M * p.unit_first[p.slices];
    hipLaunchKernelGGL(lora_shrink_kernel, dim3((uint32_t)(shrink < cap ? shrink : cap)), dim3(kLoraBlock), 0, st, p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    const dim3 grid((uint32_t)(expand < cap ? expand : cap));
    auto go = [&](auto wide, auto narrow) { hipLaunchKernelGGL(p.wide ? wide : narrow, grid, dim3(kLoraBlock), 0, st, p); };
    const int steps = (p.R + 31) / 32;
    if (steps <= 1) go(lora_expand_kernel<1, true>, lora_expand_kernel<1, false>);
    else if (steps <= 2) go(lora_expand_kernel<2, true>, lora_expand_kernel<2, false>);
    else if (steps <= 4) go(lora_expand_kernel<4, true>, lora_expand_kernel<4, false>);
    else go(lora_expand_kernel<8, true>, lora_expand_kernel<8, false>);
    return (int)hipGetLastError();
}

static int64_t lora_workspace(int M, int R, int slices)
{
    const int64_t rows = M < kLoraRows ? M : kLoraRows, stride = ((int64_t)slices * R + 15) / 16 * 16;
    return kMaxPieces * rows * stride * (int64_t)sizeof(float);
}
static bool lora_sizes(int M, int R, int slices)
{
    return M >= 0 && R > 0 && R % 8 == 0 && R <= 256 && slices > 0 && slices <= kMaxSlices;
}

}  // namespace paia

extern "C" {

long long paia_lora_add_workspace(int M, int rank, int slices)
{
    return paia::lora_sizes(M, rank, slices) ? paia::lora_workspace(M, rank, slices) : -2;
}

int paia_lora_add(const void* y, long long y_stride, const void* x, long long x_stride, const void* A, const void* B,
                  const void* ids, const void* scaling, void* out, long long out_stride, int M, int K, int rank,
                  const int* splits, int slices, int adapters, void* workspace, long long workspace_bytes, void* stream)
{
    using namespace paia;
    if (!lora_sizes(M, rank, slices) || K <= 0 || K % 8 || adapters <= 0 || splits == nullptr) return -2;
    LoraParams p;
    int64_t N = 0, units = 0;
    constexpr int kUnit = kLoraWaves * kTilesPerWave * 16;
    p.wide = true;
    for (int j = 0; j < slices; ++j) {
        if (splits[j] <= 0) return -2;
        p.first[j] = (int)N, p.unit_first[j] = (int)units;
        N += splits[j], units += ((int64_t)splits[j] + kUnit - 1) / kUnit;
        p.wide = p.wide && p.first[j] % 4 == 0;
        // outputs and units of a launch are counted in 31 bits
        if (N > INT_MAX - kUnit || units * kLoraRows > INT_MAX) return -2;
    }
    p.first[slices] = (int)N, p.unit_first[slices] = (int)units;
    if (M == 0) return 0;
    if (y == nullptr || x == nullptr || A == nullptr || B == nullptr || ids == nullptr || out == nullptr) return -2;
    if (!aligned(x, 16) || !aligned(A, 16) || !aligned(B, 16) || !aligned(y, 2) || !aligned(out, 2) || !aligned(ids, 4) ||
        !aligned(scaling, 4) || x_stride < 0 || x_stride % 8 || y_stride < 0 || out_stride < 0 || (M > 1 && out_stride < N))
        return -2;
    if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < lora_workspace(M, rank, slices)) return -2;
    p.wide = p.wide && aligned(y, 8) && aligned(out, 8) && (M == 1 || (y_stride % 4 == 0 && out_stride % 4 == 0));
    p.A = static_cast<const uint16_t*>(A);
    p.B = static_cast<const uint16_t*>(B);
    p.scaling = static_cast<const float*>(scaling);
    p.part = static_cast<float*>(workspace);
    p.x_stride = x_stride, p.y_stride = y_stride, p.out_stride = out_stride;
    p.K = K, p.N = (int)N, p.R = rank, p.adapters = adapters, p.slices = slices;
    p.h_rows = slices * rank, p.h_stride = (p.h_rows + 15) / 16 * 16;
    for (int m = 0; m < M; m += kLoraRows) {
        p.M = M - m < kLoraRows ? M - m : kLoraRows;
        p.x = static_cast<const uint16_t*>(x) + m * x_stride;
        p.y = static_cast<const uint16_t*>(y) + m * y_stride;
        p.out = static_cast<uint16_t*>(out) + m * out_stride;
        p.ids = static_cast<const int32_t*>(ids) + m;
        if (const int e = launch_lora(p, static_cast<hipStream_t>(stream)); e != 0) return e;
    }
    return 0;
}

}  // extern "C"
