// Low-rank adapters of many requests beside a shared projection.
//
//   out[m, n] = bf16( y[m, n] + s_a sum_r B_a[n, r] h[m, j(n) R + r] ),   h[m, :] = A_a x[m],   a = ids[m]
//
// j(n) is the slice of the projection that output n belongs to (q | k | v, gate | up): each slice has its own R rows of A.
// Rows without an adapter keep y. fp32 throughout, one rounding at the end. Bound by reading the adapters in use, once for
// each 16 rows that share one, and for few rows by the latency of two dependent products. Two forms (use_small):
//   * Few rows and low ranks, one launch: a block is one row and 512 outputs of a slice, and takes the slice's h for itself:
//     each wave dots its columns of x with the rank rows of A (v_dot2, whole lines), then a thread has an output. The
//     repeated reads of A come from the caches; a second launch and its dependent reads would cost more.
//   * Otherwise two launches on v_mfma_f32_16x16x32_bf16, the adapter's rows as one operand and up to 16 rows that share it as
//     the other. The first leaves partial sums of h over pieces of K in the workspace (added in order by the second: no
//     atomics), so that few adapters still fill the chip, and the list of chunks of rows: each of its blocks finds the rows
//     that share an adapter from ids itself (row_chunks), nothing has to be sorted or counted before the call. h goes to the
//     second product as two bf16 terms (value and remainder, 16 bits together), so that out has the one rounding that matters.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "gemv_kernel.h"
#include "kv_cache.h"
#include "paia_gemv.h"

namespace paia {

constexpr int kLoraBlock = 256, kLoraWaves = kLoraBlock / kWave;
constexpr int kLoraRows = 256;           // rows of a launch
constexpr int kChunk = 16;               // rows that share a pass over an adapter
constexpr int kMaxSlices = 8, kMaxPieces = 8;
constexpr int kShrinunits = 512;        // blocks aimed at by the first product's split of K
constexpr int kShrinkCols = 64;          // columns of K a wave takes at a time
constexpr int kSmallBlock = 512, kSmallWaves = kSmallBlock / kWave;
constexpr int kSmallRank = 32;           // rank up to which the small form takes a row's h in registers
constexpr int64_t kSmallA = 1 << 20, kSmallReads = 64 << 20;     // bytes of A that a block, all blocks may read there
constexpr int kShrinkAhead = 3;          // such steps whose loads a wave has in flight

// What the first product tells the second: the pieces of K, and chunks of rows that share an adapter (-1: rows without one).
struct ChunkList {
    int count, pieces, pad[2];
    struct { int adapter, held, rows[kChunk]; } chunk[kLoraRows];
};

struct LoraParams {
    const uint16_t *x, *A, *B, *y;
    uint16_t* out;
    const int32_t* ids;
    const float* scaling;                // fp32 [adapters] or null
    struct ChunkList* list;
    float* part;                         // [piece][row][h_stride]
    int64_t x_stride, y_stride, out_stride;
    int M, K, N, R, adapters, slices, h_rows, h_stride;     // h_rows: slices * R; h_stride: that rounded up to 16
    int first[kMaxSlices + 1];           // first output of each slice, N at the end
    int unit_first[kMaxSlices + 1];      // first expand unit of each slice within a chunk
    Divisor by_row;                      // by R / 8, the 16-byte pieces of a row of B
    bool wide;                           // out and y take 8-byte accesses
};

// The rows in the order of their adapters, cut into chunks of at most kChunk rows of one adapter; rows without one last.
struct RowChunks {
    int4 keys[kLoraRows / 4];            // adapter of each row, INT_MAX without and past the last row
    int order[kLoraRows];                // rows by (key, row)
    int start[kLoraRows + 1];            // first place in `order` of each chunk
    int marks[kLoraWaves];
    int count;
    __device__ __forceinline__ int& key(int row) { return reinterpret_cast<int*>(keys)[row]; }
};
__device__ __forceinline__ void row_chunks(const LoraParams& p, RowChunks* s)
{
    const int t = (int)threadIdx.x;
    int key = INT_MAX;
    if (t < p.M) {
        const int id = p.ids[t];
        if (id >= 0 && id < p.adapters) key = id;
    }
    s->key(t) = key;
    __syncthreads();
    int place = 0, same = 0;
    for (int j = 0; j < p.M; j += 16) {
        int4 k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = s->keys[j / 4 + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = j + 4 * i;
            same += (k[i].x == key && at < t) + (k[i].y == key && at + 1 < t) + (k[i].z == key && at + 2 < t) +
                    (k[i].w == key && at + 3 < t);
            place += (k[i].x < key) + (k[i].y < key) + (k[i].z < key) + (k[i].w < key);
        }
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
    return max(1, min(most, kShrinunits / units));
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

__device__ __forceinline__ void lora_lds_order()     // a wave's LDS operations stay in order; the compiler has to keep them so
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// h: a unit is (chunk, 16 rows of A, piece of K); the block's waves take its steps of 64 columns in turn. Eight lanes load
// 128 bytes of a row, of A and of x alike; a wave-private piece of LDS brings both into the matrix layout (row n at piece
// c ^ n / 2: the 16 rows of a read cover all banks).
__global__ void __launch_bounds__(kLoraBlock) lora_shrink_kernel(const LoraParams p)
{
    __shared__ RowChunks rows;
    __shared__ u32x4 stage[kLoraWaves][2][kChunk * 8];
    __shared__ f32x4 sums[kLoraWaves][kWave];
    row_chunks(p, &rows);
    const int tiles = p.h_stride / 16, pieces = k_pieces(p, rows.count), steps = (p.K + kShrinkCols - 1) / kShrinkCols;
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    const int lr = lane >> 3, lc = lane & 7;      // row (and that plus 8) and piece of a row that the lane loads
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) p.list->count = rows.count, p.list->pieces = pieces;
        for (int e = (int)threadIdx.x; e < rows.count * kChunk; e += kLoraBlock) {
            const int c = e / kChunk, i = e % kChunk, start = rows.start[c], held = rows.start[c + 1] - start;
            const int row = rows.order[start + min(i, held - 1)], id = rows.key(row);
            p.list->chunk[c].rows[i] = row;
            if (i == 0) p.list->chunk[c].adapter = id == INT_MAX ? -1 : id, p.list->chunk[c].held = held;
        }
    }
    for (int unit = (int)blockIdx.x; unit < rows.count * tiles * pieces; unit += (int)gridDim.x) {
        const int piece = unit % pieces, tile = unit / pieces % tiles, chunk = unit / pieces / tiles;
        const int start = rows.start[chunk], held = rows.start[chunk + 1] - start;
        const int id = rows.key(rows.order[start]);
        if (id == INT_MAX) break;        // the last chunks: rows without an adapter
        const int s0 = (int)((int64_t)steps * piece / pieces), s1 = (int)((int64_t)steps * (piece + 1) / pieces);
        const uint16_t *a[2], *x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[i] = p.A + ((int64_t)id * p.h_rows + min(tile * 16 + 8 * i + lr, p.h_rows - 1)) * p.K + 8 * lc;
            x[i] = p.x + rows.order[start + min(8 * i + lr, held - 1)] * p.x_stride + 8 * lc;
        }
        u32x4 u[kShrinkAhead][2], v[kShrinkAhead][2];
        auto load = [&](int s, int at) {          // a step past the piece's end loads nothing and adds nothing
            const bool in = s < s1 && kShrinkCols * s + 8 * lc < p.K;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                u[at][i] = load16_if(a[i] + kShrinkCols * (int64_t)s, in);
                v[at][i] = load16_if(x[i] + kShrinkCols * (int64_t)s, in && 8 * i < held);
            }
        };
#pragma unroll
        for (int i = 0; i < kShrinkAhead; ++i) load(s0 + wave + i * kLoraWaves, i);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = s0 + wave; s < s1; s += kShrinkAhead * kLoraWaves) {
#pragma unroll
            for (int i = 0; i < kShrinkAhead; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * e + lr, at = r * 8 + (lc ^ (r >> 1));
                    stage[wave][0][at] = u[i][e];
                    stage[wave][1][at] = v[i][e];
                }
                lora_lds_order();
                load(s + (kShrinkAhead + i) * kLoraWaves, i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = n * 8 + ((4 * j + g) ^ (n >> 1));
                    acc = lora_mfma(stage[wave][0][at], stage[wave][1][at], acc);
                }
                lora_lds_order();
            }
        }
        sums[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && n < held) {
            const int m = rows.order[start + n];
#pragma unroll
            for (int w = 1; w < kLoraWaves; ++w) acc += sums[w][lane];
            *reinterpret_cast<f32x4*>(p.part + ((int64_t)piece * p.M + m) * p.h_stride + tile * 16 + 4 * g) = acc;
        }
        __syncthreads();
    }
}

// out: a unit is (chunk, slice, kLoraWaves * ROWS outputs of the slice). STEPS: 32-value steps of R. A wave's ROWS rows of B
// are contiguous memory, ROWS R / 8 pieces of 16 bytes, loaded as such and brought into the matrix layout through its own
// piece of LDS (rows an odd number of pieces apart: no bank conflicts). The block sums the pieces of h for its chunk once.
constexpr int expand_rows(int steps) { return steps <= 1 ? 64 : steps <= 2 ? 32 : 16; }
template <int STEPS, bool WIDE>
__global__ void __launch_bounds__(kLoraBlock) lora_expand_kernel(const LoraParams p)
{
    constexpr int ROWS = expand_rows(STEPS), kTiles = ROWS / 16, kLoads = ROWS * STEPS * 4 / kWave;
    constexpr int kHPitch = STEPS * 4 + 1, kBPitch = STEPS * 4 + 1;      // 16-byte pieces
    __shared__ u32x4 h_of[2][kChunk * kHPitch];
    __shared__ u32x4 b_of[kLoraWaves][ROWS * kBPitch];
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    const int row_pieces = p.R / 8, pitch = row_pieces | 1, u = (int)blockIdx.x;
    int slice = 0;
    while (u >= p.unit_first[slice + 1]) ++slice;
    const int count = p.list->count, pieces = p.list->pieces;
    for (int chunk = (int)blockIdx.y; chunk < count; chunk += (int)gridDim.y) {
        const auto& c = p.list->chunk[chunk];
        const int id = c.adapter, held = c.held, m = c.rows[n];
        const bool live = n < held, bare = id < 0;
        if (bare && p.out == p.y && p.out_stride == p.y_stride) continue;
        const int end = p.first[slice + 1];
        const int n0 = p.first[slice] + ((u - p.unit_first[slice]) * kLoraWaves + wave) * ROWS;
        const int width = min(ROWS, end - n0);         // outputs of this wave, none where it is not positive

        u32x4 b[kLoads];
        const u32x4* B = reinterpret_cast<const u32x4*>(p.B + ((int64_t)(bare ? 0 : id) * p.N + n0) * p.R);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = i * kWave + lane;
            b[i] = !bare && at < width * row_pieces ? B[at] : u32x4{0, 0, 0, 0};
        }
        const uint16_t* y = p.y + m * p.y_stride;
        uint16_t* out = p.out + m * p.out_stride;
        uint2 was[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int at = 16 * t + 4 * g;
            was[t] = uint2{0, 0};
            if (!live || at >= width) continue;
            if (WIDE && at + 4 <= width) {
                was[t] = *reinterpret_cast<const uint2*>(y + n0 + at);
            } else {
                const uint16_t* from = y + n0 + at;
                was[t].x = from[0] | (at + 1 < width ? (uint32_t)from[1] << 16 : 0u);
                was[t].y = at + 2 < width ? from[2] | (at + 3 < width ? (uint32_t)from[3] << 16 : 0u) : 0u;
            }
        }
        if (!bare) {
            // the chunk's values of this slice of h: the pieces' sums in order, times the adapter's factor, as bf16 value
            // and remainder
            const float factor = p.scaling == nullptr ? 1.0f : p.scaling[id];
            for (int e = (int)threadIdx.x; e < held * (p.R / 4); e += kLoraBlock) {
                const int c4 = e / held, r = e - c4 * held;
                const float* src = p.part + (int64_t)c.rows[r] * p.h_stride + slice * p.R + 4 * c4;
                f32x4 term[kMaxPieces], h = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < kMaxPieces; ++i)
                    term[i] = i < pieces ? *reinterpret_cast<const f32x4*>(src + (int64_t)i * p.M * p.h_stride)
                                         : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < kMaxPieces; ++i) h += term[i];
                h *= factor;
                const uint2 hi = {pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])};
                const uint2 lo = {pack_bf16x2(rest(h[0], hi.x << 16), rest(h[1], hi.x & 0xFFFF0000u)),
                                  pack_bf16x2(rest(h[2], hi.y << 16), rest(h[3], hi.y & 0xFFFF0000u))};
                reinterpret_cast<uint2*>(h_of[0])[r * (2 * kHPitch) + c4] = hi;
                reinterpret_cast<uint2*>(h_of[1])[r * (2 * kHPitch) + c4] = lo;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t at = (uint32_t)(i * kWave + lane), r = p.by_row.of(at);
            if (r < (uint32_t)ROWS) b_of[wave][r * pitch + at - r * row_pieces] = b[i];
        }
        lora_lds_order();
        u32x4 hi[STEPS], lo[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const bool in = !bare && 4 * s + g < row_pieces;
            hi[s] = in ? h_of[0][min(n, held - 1) * kHPitch + 4 * s + g] : u32x4{0, 0, 0, 0};
            lo[s] = in ? h_of[1][min(n, held - 1) * kHPitch + 4 * s + g] : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const u32x4 w = 4 * s + g < row_pieces ? b_of[wave][(16 * t + n) * pitch + 4 * s + g] : u32x4{0, 0, 0, 0};
                acc = lora_mfma(w, lo[s], acc);
                acc = lora_mfma(w, hi[s], acc);
            }
            const int at = 16 * t + 4 * g;
            if (!live || at >= width) continue;
            uint2 v = was[t];
            if (!bare) {
                v.x = pack_bf16x2(bf16_to_f32(v.x & 0xFFFFu) + acc[0], __uint_as_float(v.x & 0xFFFF0000u) + acc[1]);
                v.y = pack_bf16x2(bf16_to_f32(v.y & 0xFFFFu) + acc[2], __uint_as_float(v.y & 0xFFFF0000u) + acc[3]);
            }
            uint16_t* to = out + n0 + at;
            if (WIDE && at + 4 <= width) {
                *reinterpret_cast<uint2*>(to) = v;
            } else {
                to[0] = (uint16_t)v.x;
                if (at + 1 < width) to[1] = (uint16_t)(v.x >> 16);
                if (at + 2 < width) to[2] = (uint16_t)v.y;
                if (at + 3 < width) to[3] = (uint16_t)(v.y >> 16);
            }
        }
        __syncthreads();
    }
}

// One row and kSmallBlock outputs of one slice a block. RANK: 8, 16 or 32 values of h at most.
template <int RANK>
__global__ void __launch_bounds__(kSmallBlock) lora_small_kernel(const LoraParams p)
{
    __shared__ float part[kSmallWaves][RANK];
    const int lane = lane_id(), wave = wave_id(), m = (int)blockIdx.y, u = (int)blockIdx.x;
    int slice = 0;
    while (u >= p.unit_first[slice + 1]) ++slice;
    const int n = p.first[slice] + (u - p.unit_first[slice]) * kSmallBlock + (int)threadIdx.x;
    const bool mine = n < p.first[slice + 1];
    const int id = p.ids[m];
    const uint16_t* y = p.y + m * p.y_stride + n;
    uint16_t* out = p.out + m * p.out_stride + n;
    const uint32_t was = mine ? *y : 0u;
    if (id < 0 || id >= p.adapters) {
        if (mine) *out = (uint16_t)was;
        return;
    }
    // the thread's row of B, whose R values lie together, on its way while h is made
    u32x4 b[RANK / 8];
    const u32x4* B = reinterpret_cast<const u32x4*>(p.B + ((int64_t)id * p.N + (mine ? n : 0)) * p.R);
#pragma unroll
    for (int i = 0; i < RANK / 8; ++i) b[i] = 8 * i < p.R ? B[i] : u32x4{0, 0, 0, 0};

    const uint16_t* A = p.A + ((int64_t)id * p.h_rows + slice * p.R) * p.K;
    const uint16_t* x = p.x + m * p.x_stride;
    float h[RANK];
#pragma unroll
    for (int r = 0; r < RANK; ++r) h[r] = 0.0f;
    constexpr int kBatch = RANK < 16 ? RANK : 16;        // rows of A whose loads are in flight together
    for (int k = (int)threadIdx.x * 8; k < p.K; k += kSmallBlock * 8) {
        const u32x4 xv = *reinterpret_cast<const u32x4*>(x + k);
#pragma unroll
        for (int r0 = 0; r0 < RANK; r0 += kBatch) {
            u32x4 a[kBatch];
#pragma unroll
            for (int r = 0; r < kBatch; ++r)
                a[r] = *reinterpret_cast<const u32x4*>(A + (int64_t)min(r0 + r, p.R - 1) * p.K + k);
#pragma unroll
            for (int r = 0; r < kBatch; ++r) h[r0 + r] = dot_bf16_16B(a[r], xv, h[r0 + r]);
        }
    }
#pragma unroll
    for (int r = 0; r < RANK; r += 2) {
        const float s = wave_sum2(h[r], h[r + 1]);       // lane 31: the first, lane 63: the second
        if ((lane & 31) == 31) part[wave][r + lane / 32] = s;
    }
    __syncthreads();
    float acc = 0.0f;
#pragma unroll
    for (int i = 0; i < RANK / 8; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = part[0][8 * i + e];
#pragma unroll
            for (int w = 1; w < kSmallWaves; ++w) v += part[w][8 * i + e];
            const uint32_t bw = b[i][e / 2];
            if (8 * i < p.R) acc = __builtin_fmaf(v, __uint_as_float(e & 1 ? bw & 0xFFFF0000u : bw << 16), acc);
        }
    if (mine) *out = (uint16_t)f32_to_bf16_out(bf16_to_f32(was) + acc * (p.scaling == nullptr ? 1.0f : p.scaling[id]));
}

static int launch_lora(const LoraParams& p, hipStream_t st)
{
    const int cap = device_facts().cus * 4;
    const int64_t shrink = (int64_t)p.M * (p.h_stride / 16) * kMaxPieces;
    hipLaunchKernelGGL(lora_shrink_kernel, dim3((uint32_t)(shrink < cap ? shrink : cap)), dim3(kLoraBlock), 0, st, p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    // a row of blocks for each chunk that there may be, up to 8192 blocks, beyond which a block takes several chunks
    const int per_chunk = p.unit_first[p.slices], rows = 8192 / per_chunk;
    const dim3 grid((uint32_t)per_chunk, (uint32_t)(rows < 1 ? 1 : rows < p.M ? rows : p.M));
    auto go = [&](auto wide, auto narrow) { hipLaunchKernelGGL(p.wide ? wide : narrow, grid, dim3(kLoraBlock), 0, st, p); };
    const int steps = (p.R + 31) / 32;
    if (steps <= 1) go(lora_expand_kernel<1, true>, lora_expand_kernel<1, false>);
    else if (steps <= 2) go(lora_expand_kernel<2, true>, lora_expand_kernel<2, false>);
    else if (steps <= 4) go(lora_expand_kernel<4, true>, lora_expand_kernel<4, false>);
    else go(lora_expand_kernel<8, true>, lora_expand_kernel<8, false>);
    return (int)hipGetLastError();
}

static int launch_small(const LoraParams& p, hipStream_t st)
{
    const dim3 grid((uint32_t)p.unit_first[p.slices], (uint32_t)p.M);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kSmallBlock), 0, st, p); };
    if (p.R <= 8) go(lora_small_kernel<8>);
    else if (p.R <= 16) go(lora_small_kernel<16>);
    else go(lora_small_kernel<32>);
    return (int)hipGetLastError();
}

// The small form reads a slice's rows of A once for every kSmallBlock outputs and row.
static bool use_small(int M, int K, int R, const int* splits, int slices)
{
    if (R > kSmallRank || (int64_t)R * K * 2 > kSmallA) return false;
    int64_t blocks = 0;
    for (int j = 0; j < slices; ++j) blocks += ((int64_t)splits[j] + kSmallBlock - 1) / kSmallBlock;
    return blocks * M <= kSmallReads / ((int64_t)R * K * 2);
}

static bool lora_sizes(int M, int K, int R, const int* splits, int slices)
{
    if (M < 0 || K <= 0 || K % 8 || R <= 0 || R % 8 || R > 256 || slices <= 0 || slices > kMaxSlices || splits == nullptr)
        return false;
    for (int j = 0; j < slices; ++j)
        if (splits[j] <= 0) return false;
    return true;
}
static int64_t lora_workspace(int M, int K, int R, const int* splits, int slices)
{
    if (use_small(M, K, R, splits, slices)) return 0;
    const int64_t rows = M < kLoraRows ? M : kLoraRows, stride = ((int64_t)slices * R + 15) / 16 * 16;
    return (int64_t)sizeof(ChunkList) + kMaxPieces * rows * stride * (int64_t)sizeof(float);
}

}  // namespace paia

extern "C" {

long long paia_lora_add_workspace(int M, int K, int rank, const int* splits, int slices)
{
    return paia::lora_sizes(M, K, rank, splits, slices) ? paia::lora_workspace(M, K, rank, splits, slices) : -2;
}

int paia_lora_add(const void* y, long long y_stride, const void* x, long long x_stride, const void* A, const void* B,
                  const void* ids, const void* scaling, void* out, long long out_stride, int M, int K, int rank,
                  const int* splits, int slices, int adapters, void* workspace, long long workspace_bytes, void* stream)
{
    using namespace paia;
    if (!lora_sizes(M, K, rank, splits, slices) || adapters <= 0) return -2;
    LoraParams p;
    int64_t N = 0, units = 0;
    const bool small = use_small(M, K, rank, splits, slices);
    const int unit = small ? kSmallBlock : kLoraWaves * expand_rows((rank + 31) / 32);
    p.wide = true;
    for (int j = 0; j < slices; ++j) {
        p.first[j] = (int)N, p.unit_first[j] = (int)units;
        N += splits[j], units += ((int64_t)splits[j] + unit - 1) / unit;
        p.wide = p.wide && p.first[j] % 4 == 0;
        // outputs and units of a launch are counted in 31 bits
        if (N > INT_MAX - unit || units * kLoraRows > INT_MAX) return -2;
    }
    p.first[slices] = (int)N, p.unit_first[slices] = (int)units;
    if (M == 0) return 0;
    if (y == nullptr || x == nullptr || A == nullptr || B == nullptr || ids == nullptr || out == nullptr) return -2;
    if (!aligned(x, 16) || !aligned(A, 16) || !aligned(B, 16) || !aligned(y, 2) || !aligned(out, 2) || !aligned(ids, 4) ||
        !aligned(scaling, 4) || x_stride < 0 || x_stride % 8 || y_stride < 0 || out_stride < 0 || (M > 1 && out_stride < N))
        return -2;
    const int64_t need = lora_workspace(M, K, rank, splits, slices);
    if (need > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need)) return -2;
    p.wide = p.wide && aligned(y, 8) && aligned(out, 8) && (M == 1 || (y_stride % 4 == 0 && out_stride % 4 == 0));
    p.A = static_cast<const uint16_t*>(A);
    p.B = static_cast<const uint16_t*>(B);
    p.scaling = static_cast<const float*>(scaling);
    p.list = static_cast<ChunkList*>(workspace);
    p.part = need > 0 ? reinterpret_cast<float*>(p.list + 1) : nullptr;
    p.x_stride = x_stride, p.y_stride = y_stride, p.out_stride = out_stride;
    p.K = K, p.N = (int)N, p.R = rank, p.adapters = adapters, p.slices = slices;
    p.by_row = Divisor((uint32_t)(rank / 8));
    p.h_rows = slices * rank, p.h_stride = (p.h_rows + 15) / 16 * 16;
    for (int m = 0; m < M; m += kLoraRows) {
        p.M = M - m < kLoraRows ? M - m : kLoraRows;
        p.x = static_cast<const uint16_t*>(x) + m * x_stride;
        p.y = static_cast<const uint16_t*>(y) + m * y_stride;
        p.out = static_cast<uint16_t*>(out) + m * out_stride;
        p.ids = static_cast<const int32_t*>(ids) + m;
        const hipStream_t st = static_cast<hipStream_t>(stream);
        if (const int e = small ? launch_small(p, st) : launch_lora(p, st); e != 0) return e;
    }
    return 0;
}

}  // extern "C"
