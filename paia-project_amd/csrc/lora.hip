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
//     second product as two bf16 terms (rest_bf16, 16 bits together), so that out has the one rounding that matters.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "divisor.h"
#include "gemv_kernel.h"
#include "paia_gemv.h"

namespace paia {

constexpr int kLoraBlock = 256, kLoraWaves = kLoraBlock / kWave;
constexpr int kLoraRows = 256;           // rows of a launch, a thread each
constexpr int kRowWaves = kLoraRows / kWave;
constexpr int kShrinkBlock = 512, kShrinkWaves = kShrinkBlock / kWave;
constexpr int kChunk = 16;               // rows that share a pass over an adapter
constexpr uint32_t kNoAdapter = 0xFFFFFFu;
constexpr int kMaxSlices = 8, kMaxPieces = 8;
constexpr int kShrinkUnits = 512;        // blocks aimed at by the first product's split of K
constexpr int kShrinkCols = 64;          // columns of K a wave takes at a time
constexpr int kSmallBlock = 512, kSmallWaves = kSmallBlock / kWave;
constexpr int kSmallRank = 32;           // rank up to which the small form holds a row's h in registers
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
    Divisor by_row, by_chunk;            // by R / 8, the 16-byte pieces of a row of B; by a chunk's expand units
    bool wide;                           // out and y take 8-byte accesses
};

// The rows in the order of their adapters, cut into chunks of at most kChunk rows of one adapter; rows without one last.
struct RowChunks {
    uint4 keys[kLoraRows / 4];           // adapter << 8 | row, kNoAdapter without one; past the last row the largest key
    uint32_t sorted[kLoraRows];          // the keys in order
    int start[kLoraRows + 1];            // first place in `sorted` of each chunk
    uint64_t begins[kRowWaves];          // places where another adapter begins
    int marks[kRowWaves];                // chunks that begin in each wave's places
    int count;
    __device__ __forceinline__ int row(int place) const { return (int)(sorted[place] & 255u); }
    __device__ __forceinline__ int adapter(int place) const      // -1: rows without one
    {
        const uint32_t id = sorted[place] >> 8;
        return id == kNoAdapter ? -1 : (int)id;
    }
};
__device__ __forceinline__ void row_chunks(const LoraParams& p, RowChunks* s)
{
    const int t = (int)threadIdx.x, lane = lane_id(), wave = wave_id();
    if (p.M == 1) {                      // nothing to sort (rank 64 beside 4096 -> 6144: 9.6 -> 8.8 us a call)
        if (t == 0) {
            const int id = p.ids[0];
            s->sorted[0] = (id >= 0 && id < p.adapters ? (uint32_t)id : kNoAdapter) << 8;
            s->start[0] = 0, s->start[1] = 1, s->count = 1;
        }
        __syncthreads();
        return;
    }
    uint32_t key = ~0u;
    if (t < p.M) {
        const int id = p.ids[t];
        key = (id >= 0 && id < p.adapters ? (uint32_t)id : kNoAdapter) << 8 | (uint32_t)t;
    }
    if (t < kLoraRows) reinterpret_cast<uint32_t*>(s->keys)[t] = key;
    __syncthreads();
    if (wave * kWave < p.M) {            // a row's place: the keys below its own
        int place = 0;
        for (int j = 0; j < p.M; j += 16) {
            uint4 k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) k[i] = s->keys[j / 4 + i];
#pragma unroll
            for (int i = 0; i < 4; ++i) place += (k[i].x < key) + (k[i].y < key) + (k[i].z < key) + (k[i].w < key);
        }
        if (t < p.M) s->sorted[place] = key;
    }
    __syncthreads();
    const bool begins = t < p.M && (t == 0 || s->sorted[t] >> 8 != s->sorted[t - 1] >> 8);
    const uint64_t mask = __ballot(begins);
    if (lane == 0 && wave < kRowWaves) s->begins[wave] = mask;
    __syncthreads();
    // the place where this place's adapter begins: the last mark at or before it
    uint64_t marks = mask & (~0ull >> (63 - lane));
    int w = min(wave, kRowWaves);
    while (marks == 0 && w > 0) marks = s->begins[--w];
    const int from = w * kWave + 63 - (marks != 0 ? __builtin_clzll(marks) : 63);
    const bool cut = t < p.M && (t - from) % kChunk == 0;
    const uint64_t cuts = __ballot(cut);
    if (lane == 0 && wave < kRowWaves) s->marks[wave] = __popcll(cuts);
    __syncthreads();
    int before = 0, count = 0;
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) {
        before += i < wave ? s->marks[i] : 0;
        count += s->marks[i];
    }
    if (cut) s->start[before + __popcll(cuts & ((1ull << lane) - 1))] = t;
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

__device__ __forceinline__ u32x4 load16_if(const uint16_t* p, bool take)
{
    return take ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
}

// A value cut to bf16 toward zero is its upper half; this is what it keeps beyond that, as bf16. Both terms have the value's sign, or
// an infinity in B would meet terms of both signs, or a 0: so what rounds to 0 is the smallest value instead, unless the value is 0,
// and the rest of what is not finite is the same again.
__device__ __forceinline__ uint32_t rest_bf16(float v)
{
    const uint32_t w = __float_as_uint(v);
    const uint32_t r = f32_to_bf16_out(fabsf(v) < __builtin_inff() ? v - __uint_as_float(w & 0xFFFF0000u) : v);
    return (r & 0x7FFFu) == 0 && v != 0.0f ? (w >> 16 & 0x8000u) | 1u : r;
}

// h: a unit is (chunk, 16 rows of A, piece of K); the block's waves take its steps of 64 columns in turn. Eight lanes load
// 128 bytes of a row, of A and of x alike; a wave-private piece of LDS brings both into the matrix layout (row n at piece
// c ^ n / 2: the 16 rows of a read cover all banks).
__global__ void __launch_bounds__(kShrinkBlock) lora_shrink_kernel(const LoraParams p)
{
    __shared__ RowChunks rows;
    __shared__ u32x4 stage[kShrinkWaves][2][kChunk * 8];
    __shared__ f32x4 sums[kShrinkWaves][kWave];
    row_chunks(p, &rows);
    const int tiles = p.h_stride / 16, pieces = k_pieces(p, rows.count), steps = (p.K + kShrinkCols - 1) / kShrinkCols;
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    const int lr = lane >> 3, lc = lane & 7;      // row (and that plus 8) and piece of a row that the lane loads
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) p.list->count = rows.count, p.list->pieces = pieces;
        for (int e = (int)threadIdx.x; e < rows.count * kChunk; e += kShrinkBlock) {
            const int c = e / kChunk, i = e % kChunk, start = rows.start[c], held = rows.start[c + 1] - start;
            p.list->chunk[c].rows[i] = rows.row(start + min(i, held - 1));
            if (i == 0) p.list->chunk[c].adapter = rows.adapter(start), p.list->chunk[c].held = held;
        }
    }
    for (int unit = (int)blockIdx.x; unit < rows.count * tiles * pieces; unit += (int)gridDim.x) {
        const int piece = unit % pieces, tile = unit / pieces % tiles, chunk = unit / pieces / tiles;
        const int start = rows.start[chunk], held = rows.start[chunk + 1] - start;
        const int id = rows.adapter(start);
        if (id < 0) break;               // the last chunks: rows without an adapter
        const int s0 = (int)((int64_t)steps * piece / pieces), s1 = (int)((int64_t)steps * (piece + 1) / pieces);
        const uint16_t *a[2], *x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[i] = p.A + ((int64_t)id * p.h_rows + min(tile * 16 + 8 * i + lr, p.h_rows - 1)) * p.K + 8 * lc;
            x[i] = p.x + rows.row(start + min(8 * i + lr, held - 1)) * p.x_stride + 8 * lc;
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
        for (int i = 0; i < kShrinkAhead; ++i) load(s0 + wave + i * kShrinkWaves, i);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = s0 + wave; s < s1; s += kShrinkAhead * kShrinkWaves) {
#pragma unroll
            for (int i = 0; i < kShrinkAhead; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * e + lr, at = r * 8 + (lc ^ (r >> 1));
                    stage[wave][0][at] = u[i][e];
                    stage[wave][1][at] = v[i][e];
                }
                wave_lds_order();
                load(s + (kShrinkAhead + i) * kShrinkWaves, i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = n * 8 + ((4 * j + g) ^ (n >> 1));
                    acc = mfma_16x16x32(stage[wave][0][at], stage[wave][1][at], acc);
                }
                wave_lds_order();
            }
        }
        sums[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && n < held) {
            const int m = rows.row(start + n);
#pragma unroll
            for (int w = 1; w < kShrinkWaves; ++w) acc += sums[w][lane];
            *reinterpret_cast<f32x4*>(p.part + ((int64_t)piece * p.M + m) * p.h_stride + tile * 16 + 4 * g) = acc;
        }
        __syncthreads();
    }
}

// out: a unit is (chunk, slice, kLoraWaves * ROWS outputs of the slice), ROWS of them a wave's. STEPS: 32-value steps of R.
// A wave's ROWS rows of B are contiguous memory, ROWS R / 8 pieces of 16 bytes, loaded as such and brought into the matrix
// layout through its own piece of LDS (rows an odd number of pieces apart: no bank conflicts). A block takes consecutive
// units, with kExpandAhead units' loads in flight, and sums the pieces of h anew only where the chunk or slice changes.
constexpr int expand_rows(int steps) { return steps <= 2 ? 32 : 16; }
// Blocks of the expand kernel that are launched for each CU, one wave of each on a SIMD: no more than its registers let be resident.
// Beyond rank 128 that is two: a third ran behind them (us at three / two: sixteen rows and adapters of rank 256 beside 4096 -> 6144
// 41.4 / 38.6 and -> 28672 72.4 / 64.7, of rank 192 beside 3584 -> 3584 21.1 / 18.1).
constexpr int expand_blocks(int steps) { return steps <= 4 ? 3 : 2; }
constexpr int kExpandAhead = 2;
template <int STEPS, bool WIDE>
__global__ void __launch_bounds__(kLoraBlock, expand_blocks(STEPS)) lora_expand_kernel(const LoraParams p)
{
    constexpr int ROWS = expand_rows(STEPS), kTiles = ROWS / 16, kLoads = ROWS * STEPS * 4 / kWave;
    constexpr int kHPitch = STEPS * 4 + 1, kBPitch = STEPS * 4 + 1;      // 16-byte pieces
    __shared__ u32x4 h_of[2][kChunk * kHPitch];
    __shared__ u32x4 b_of[kLoraWaves][ROWS * kBPitch];
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    const int row_pieces = p.R / 8, pitch = row_pieces | 1, per_chunk = p.unit_first[p.slices];
    const int count = p.list->count, pieces = p.list->pieces;
    const int64_t units = (int64_t)count * per_chunk;
    const int first = (int)(units * blockIdx.x / gridDim.x), last = (int)(units * (blockIdx.x + 1) / gridDim.x);
    if (first >= last) return;

    // where a unit lies
    struct Place {
        int chunk, slice, n0, width;     // width: outputs of this wave, none where it is not positive
    };
    const auto place_of = [&](int unit) {
        Place r;
        r.chunk = (int)p.by_chunk.of((uint32_t)unit);
        const int u = unit - r.chunk * per_chunk;
        r.slice = 0;
        while (u >= p.unit_first[r.slice + 1]) ++r.slice;
        r.n0 = p.first[r.slice] + ((u - p.unit_first[r.slice]) * kLoraWaves + wave) * ROWS;
        r.width = min(ROWS, p.first[r.slice + 1] - r.n0);
        return r;
    };
    Place at[kExpandAhead];
    u32x4 b[kExpandAhead][kLoads];
    uint2 was[kExpandAhead][kTiles];
    int ahead_chunk = -1, ahead_row = 0, ahead_id = 0, ahead_held = 0;     // of the last unit that was loaded
    const auto load = [&](int unit, int i) {
        if (unit >= last) return;
        const Place r = place_of(unit);
        at[i] = r;
        if (r.chunk != ahead_chunk) {
            ahead_chunk = r.chunk;
            ahead_id = p.list->chunk[r.chunk].adapter;
            ahead_held = p.list->chunk[r.chunk].held;
            ahead_row = p.list->chunk[r.chunk].rows[n];
        }
        const u32x4* B = reinterpret_cast<const u32x4*>(p.B + ((int64_t)max(ahead_id, 0) * p.N + r.n0) * p.R);
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
            const int c = e * kWave + lane;
            b[i][e] = ahead_id >= 0 && c < r.width * row_pieces ? B[c] : u32x4{0, 0, 0, 0};
        }
        const uint16_t* y = p.y + ahead_row * p.y_stride + r.n0;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int o = 16 * t + 4 * g;
            uint2 v = {0, 0};
            if (n < ahead_held && o < r.width) {
                if (WIDE && o + 4 <= r.width) {
                    v = *reinterpret_cast<const uint2*>(y + o);
                } else {
                    v.x = y[o] | (o + 1 < r.width ? (uint32_t)y[o + 1] << 16 : 0u);
                    v.y = o + 2 < r.width ? y[o + 2] | (o + 3 < r.width ? (uint32_t)y[o + 3] << 16 : 0u) : 0u;
                }
            }
            was[i][t] = v;
        }
    };
#pragma unroll
    for (int i = 0; i < kExpandAhead; ++i) load(first + i, i);

    int chunk = -1, slice = -1, m = 0, id = -1, held = 0;
    u32x4 hi[STEPS], lo[STEPS];
    for (int unit0 = first; unit0 < last; unit0 += kExpandAhead) {
#pragma unroll
        for (int i = 0; i < kExpandAhead; ++i) {
            const int unit = unit0 + i;
            if (unit >= last) break;
            const Place r = at[i];
            if (r.chunk != chunk || r.slice != slice) {
                chunk = r.chunk, slice = r.slice;
                const auto& c = p.list->chunk[chunk];
                id = c.adapter, held = c.held, m = c.rows[n];
                // the chunk's values of this slice of h: the pieces' sums in order, times the adapter's factor, in two
                // bf16 terms
                __syncthreads();
                const float factor = id < 0 || p.scaling == nullptr ? 1.0f : p.scaling[id];
                for (int e = (int)threadIdx.x; e < (id < 0 ? 0 : held * (p.R / 4)); e += kLoraBlock) {
                    const int c4 = e / held, row = e - c4 * held;
                    const float* src = p.part + (int64_t)c.rows[row] * p.h_stride + slice * p.R + 4 * c4;
                    f32x4 term[kMaxPieces], h = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < kMaxPieces; ++k)
                        term[k] = k < pieces ? *reinterpret_cast<const f32x4*>(src + (int64_t)k * p.M * p.h_stride)
                                             : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < kMaxPieces; ++k) h += term[k];
                    h *= factor;
                    uint32_t u[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) u[k] = __float_as_uint(h[k]);
                    const uint2 top = {u[0] >> 16 | (u[1] & 0xFFFF0000u), u[2] >> 16 | (u[3] & 0xFFFF0000u)};
                    const uint2 low = {rest_bf16(h[0]) | rest_bf16(h[1]) << 16, rest_bf16(h[2]) | rest_bf16(h[3]) << 16};
                    reinterpret_cast<uint2*>(h_of[0])[row * (2 * kHPitch) + c4] = top;
                    reinterpret_cast<uint2*>(h_of[1])[row * (2 * kHPitch) + c4] = low;
                }
                __syncthreads();
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const bool in = id >= 0 && 4 * s + g < row_pieces;
                    hi[s] = in ? h_of[0][min(n, held - 1) * kHPitch + 4 * s + g] : u32x4{0, 0, 0, 0};
                    lo[s] = in ? h_of[1][min(n, held - 1) * kHPitch + 4 * s + g] : u32x4{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int e = 0; e < kLoads; ++e) {
                const uint32_t c = (uint32_t)(e * kWave + lane), row = p.by_row.of(c);
                if (row < (uint32_t)ROWS) b_of[wave][row * pitch + c - row * row_pieces] = b[i][e];
            }
            uint2 y[kTiles];
#pragma unroll
            for (int t = 0; t < kTiles; ++t) y[t] = was[i][t];
            wave_lds_order();
            load(unit + kExpandAhead, i);
            uint16_t* out = p.out + m * p.out_stride + r.n0;
            const bool same = id < 0 && p.out == p.y && p.out_stride == p.y_stride;     // the row keeps y where it is
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const u32x4 w = 4 * s + g < row_pieces ? b_of[wave][(16 * t + n) * pitch + 4 * s + g] : u32x4{0, 0, 0, 0};
                    acc = mfma_16x16x32(w, lo[s], acc);
                    acc = mfma_16x16x32(w, hi[s], acc);
                }
                const int o = 16 * t + 4 * g;
                if (n >= held || o >= r.width || same) continue;
                uint2 v = y[t];
                if (id >= 0) {
                    v.x = pack_bf16x2(bf16_to_f32(v.x & 0xFFFFu) + acc[0], __uint_as_float(v.x & 0xFFFF0000u) + acc[1]);
                    v.y = pack_bf16x2(bf16_to_f32(v.y & 0xFFFFu) + acc[2], __uint_as_float(v.y & 0xFFFF0000u) + acc[3]);
                }
                if (WIDE && o + 4 <= r.width) {
                    *reinterpret_cast<uint2*>(out + o) = v;
                } else {
                    out[o] = (uint16_t)v.x;
                    if (o + 1 < r.width) out[o + 1] = (uint16_t)(v.x >> 16);
                    if (o + 2 < r.width) out[o + 2] = (uint16_t)v.y;
                    if (o + 3 < r.width) out[o + 3] = (uint16_t)(v.y >> 16);
                }
            }
            wave_lds_order();
        }
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
    // Blocks that are resident together, fewer where there are fewer units: the rest would only find the rows again (128 rows of 12
    // adapters 15.4 us at four a CU, 13.8 so; sixteen of rank 64 even).
    const int steps = (p.R + 31) / 32;
    const int cap = device_facts().cus * 2, cap_expand = device_facts().cus * expand_blocks(steps);
    const int64_t shrink = (int64_t)p.M * (p.h_stride / 16) * kMaxPieces;
    hipLaunchKernelGGL(lora_shrink_kernel, dim3((uint32_t)(shrink < cap ? shrink : cap)), dim3(kShrinkBlock), 0, st, p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    const int64_t expand = (int64_t)p.M * p.unit_first[p.slices];
    const dim3 grid((uint32_t)(expand < cap_expand ? expand : cap_expand));
    auto go = [&](auto wide, auto narrow) { hipLaunchKernelGGL(p.wide ? wide : narrow, grid, dim3(kLoraBlock), 0, st, p); };
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

// The small form reads a slice's rows of A once for every kSmallBlock outputs and row, and takes K at 4096 columns a step; its
// ranks above 16 take each step's loads in two parts. So it is the faster one up to some bytes of A a block, and in all (us in
// a graph, small / two launches; every row its own adapter, or in brackets all the same):
//   rank 16: one row 4096 -> 6144 5.0 / 9.2, 14336 -> 4096 7.3 / 9.6; 16 rows of 4096 -> 6144 (25 MB) 8.2 / 11.4 (5.1 / 10.2);
//            64 of 3584 -> 3584 (51 MB) 12.1 / 14.5; 16 of 4096 -> 28672 (117 MB) 13.4 / 15.5 (10.9 / 9.5); 16 of 14336 ->
//            4096 (59 MB) 12.8 / 10.8 (7.4 / 10.1)
//   rank 8:  64 rows of 4096 -> 6144 (50 MB) 11.8 / 16.3 (5.7 / 11.0); of 14336 -> 4096 (117 MB) 21.3 / 15.8 (8.9 / 10.4)
//   rank 32: one row 4096 -> 6144 8.6 / 9.2, 14336 -> 4096 13.8 / 9.6; 4 of 3584 -> 3584 (6 MB) 8.5 / 9.3; 8 of them (13 MB)
//            11.1 / 9.2 (8.5 / 8.9)
static bool use_small(int M, int K, int R, const int* splits, int slices)
{
    if (R > kSmallRank) return false;
    const int64_t block = (int64_t)R * K * 2, most = R <= 16 ? 640 << 10 : 256 << 10, reads = R <= 16 ? 64 << 20 : 8 << 20;
    if (block > most) return false;
    int64_t blocks = 0;
    for (int j = 0; j < slices; ++j) blocks += ((int64_t)splits[j] + kSmallBlock - 1) / kSmallBlock;
    return blocks * M <= reads / block;
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
    if (!lora_sizes(M, K, rank, splits, slices) || adapters <= 0 || adapters > (int)kNoAdapter) return -2;
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
    p.by_chunk = Divisor((uint32_t)units);
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
