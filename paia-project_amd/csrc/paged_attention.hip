// Attention of a sequence's newest tokens over a paged key-value cache, split over the cache's length and joined.
//
//   s_p = scale k_scale[h] <q, k_p>,  o = v_scale[h] sum_p exp(s_p - m) v_p / sum_p exp(s_p - m),  m = max_p s_p
//   token t of T sees positions p < len - (T-1-t), the last `window` of them where there is a window, on valid pages.
//
// Each cache byte is used for T G products a value (G query heads share a kv head), a few operations per byte: bound by
// reading the cache once. The pieces of the design:
//   * Work: a unit is one piece of one sequence for one kv head and 16 columns (token, query head of the group), or
//     up to 48 where the tables are large (attention_tiles.h). The lengths are on the device and the grid is fixed by the host, so
//     each block derives the split from the lengths itself (find_piece): about as many equal pieces as blocks fit the
//     chip, whatever the lengths are. A captured call stays balanced as the sequences grow. Pieces of one sequence leave
//     (m, l, o) in the workspace, joined by a second kernel; a sequence of one piece is written by its block.
//   * A block's four waves take its 32-position tiles in turn, each with its own running maximum, sum and output (no
//     barrier until the end), and one tile of K and V loads in flight ahead of the one in work.
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16. Both leave a column (token, head) on the same lane, so
//     P goes from the first product's result to the second's operand in registers, and the rescaling is per lane.
//   * K rows are loaded contiguously and brought to the matrix layout through a wave-private piece of LDS (XOR swizzle), by way
//     of registers or, where those are short (loads_direct), straight there.
//     V rows are loaded contiguously too, D/16 dims of eight positions per lane: 16 lanes are the 16 rows of the V^T
//     operand, whose eight contraction values are the eight positions; one v_perm_b32 per register pairs them up.
//   * e4m3 codes become bf16 exactly (v_cvt_scalef32_pk_bf16_fp8); the heads' factors go to the scores and the output.
// Scores, statistics and sums are fp32. P enters the second product as two bf16 terms (split_weights, 16 bits or more): one more
// MFMA a product, 0.3 to 1% of the time; with the value alone the output's error was 1.3 times that of its rounding.
// What no token sees (positions past the end, before the window, on a page outside the cache) contributes nothing, whatever
// its bytes are: scores are replaced, V rows zeroed, and where tokens differ in what they see and a value there is not finite,
// each takes its own product.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "attention_tiles.h"
#include "gemv_kernel.h"
#include "kv_cache.h"
#include "paia_gemv.h"

namespace paia {

constexpr int kTile = 32;            // positions a wave takes at a time
constexpr int kAttnWaves = 4, kAttnBlock = kAttnWaves * kWave;
// Blocks that a CU holds at the registers a wave takes (one wave of a block on each SIMD).
constexpr int blocks_per_cu(int dim, int tiles) { return dim <= 64 ? (tiles == 1 ? 3 : 2) : dim <= 128 ? 2 : 1; }
constexpr int kMinTiles = 4;         // a piece is at least this many tiles, where the sequence has them

struct AttnParams {
    const uint8_t* q;
    int64_t qb, qt, qh;              // bytes between sequences, tokens, heads
    uint16_t* out;                   // bf16 [B][T][heads][D]
    float* lse;                      // fp32 [B][T][heads] or null
    const int32_t *table, *lens;
    int64_t table_stride;
    CacheView cache;
    float *part_o, *part_ml;         // [item][kv head][column][D], [item][kv head][column][2]
    int2* part_of;                   // [sequence]: first item, number of items
    float scale;                     // scale * log2(e)
    int B, T, heads, group, cols, col_groups, tiles;     // tiles of columns a block takes
    int window, max_len;             // positions the table can hold
    int goal;                        // pieces per kv head at most, the items of the grid; above B
    int units;                       // items * kv heads
    Divisor by_kv_heads, by_group, by_col_groups;
};

// ---- the split of the sequences into pieces -------------------------------------------------------------------------
struct Span {
    int len, tile0, tiles;           // positions, first tile seen by any token, number of tiles (below 2^26)
};
__device__ __forceinline__ Span span_of(const AttnParams& p, int b)
{
    Span s{0, 0, 0};
    if (b < p.B) {
        s.len = min(max(p.lens[b], 0), p.max_len);
        const int first = p.window > 0 ? max(0, s.len - (p.T - 1) - p.window) : 0;
        s.tile0 = first / kTile;
        s.tiles = (s.len + kTile - 1) / kTile - s.tile0;
    }
    return s;
}
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t dpp_add_u32(uint32_t v)
{
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)      // inclusive; lane 63 holds the sum
{
    v = dpp_add_u32<0x111, 0xF>(v);   // row_shr:1, 2, 4, 8
    v = dpp_add_u32<0x112, 0xF>(v);
    v = dpp_add_u32<0x114, 0xF>(v);
    v = dpp_add_u32<0x118, 0xF>(v);
    v = dpp_add_u32<0x142, 0xA>(v);   // row_bcast:15 into rows 1, 3
    return dpp_add_u32<0x143, 0xC>(v);   // row_bcast:31 into rows 2, 3
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1); }
// Pieces of a sequence at `most` tiles a piece, at least one: ceil(tiles / most) by a float quotient, which below 2^26 tiles is a
// few off at most, its remainder's own quotient, which is within one, and a correction.
__device__ __forceinline__ uint32_t pieces_of(int tiles, int most, float inverse)
{
    int n = (int)((float)tiles * inverse);
    int left = tiles - n * most;
    const int more = (int)((float)left * inverse);
    n += more, left -= more * most;
    if (left < 0) --n, left += most;
    if (left >= most) ++n, left -= most;
    return (uint32_t)max(1, n + (left > 0 ? 1 : 0));
}
__device__ __forceinline__ int whole_rounds(float tiles)       // the next multiple of the block's waves above `tiles`
{
    return ((int)tiles / kAttnWaves + 1) * kAttnWaves;
}
struct Piece {
    int b, len, tile0, tile1;        // sequence, its length, the piece's tiles
    int index, count;                // number of the piece in its sequence, pieces of the sequence
};
__device__ __forceinline__ void take_piece(int b, const Span& s, int count, int index, Piece* r)
{
    const int each = s.tiles / count, more = s.tiles - each * count;     // the first `more` pieces get one more
    r->b = b, r->len = s.len, r->index = index, r->count = count;
    r->tile0 = s.tile0 + index * each + min(index, more);
    r->tile1 = r->tile0 + each + (index < more ? 1 : 0);
}
__device__ __forceinline__ Span lane_span(const Span& s, int lane)
{
    return {__builtin_amdgcn_readlane(s.len, lane), __builtin_amdgcn_readlane(s.tile0, lane),
            __builtin_amdgcn_readlane(s.tiles, lane)};
}
// The piece with number `item`. Every wave finds the same tile count per piece, `most`: from the least up, by the factor that
// the sequences' pieces are too many, until they are no more than p.goal.
__device__ __forceinline__ bool find_piece(const AttnParams& p, int item, Piece* r)
{
    const int lane = lane_id();
    if (p.B == 1) {
        const Span s = span_of(p, 0);
        const int mean = (s.tiles + p.goal - 1) / p.goal;
        const int most = max(kMinTiles, (mean + kAttnWaves - 1) / kAttnWaves * kAttnWaves);
        const int count = max(1, (s.tiles + most - 1) / most);
        take_piece(0, s, count, item, r);
        return item < count;
    }
    Span s = span_of(p, lane);
    const float per = __builtin_amdgcn_rcpf((float)p.goal);
    int most = kMinTiles;
    float inverse = 0.0f, tiles = 0.0f;
    uint32_t n = 0, end = 0;
#pragma nounroll
    for (int tries = 0; tries < 6; ++tries) {
        inverse = __builtin_amdgcn_rcpf((float)most);
        n = lane < p.B ? pieces_of(s.tiles, most, inverse) : 0u;
        end = wave_scan(n);
        uint64_t count = last_lane(end);
#pragma nounroll
        for (int b = kWave; b < p.B; b += kWave)
            count += last_lane(wave_scan(b + lane < p.B ? pieces_of(span_of(p, b + lane).tiles, most, inverse) : 0u));
        if (count <= (uint64_t)p.goal) break;
        const float held = (float)most * (float)count;       // no less than the tiles there are
        if (tries == 0) tiles = held;
        // the fourth step holds for any lengths: tiles / most + B pieces at most (with room for the roundings)
        most = tries < 3 ? whole_rounds(held * per) : whole_rounds(tiles * 1.001f * __builtin_amdgcn_rcpf((float)(p.goal - p.B)));
    }
    uint32_t before = 0;
#pragma nounroll
    for (int b0 = 0;;) {
        const uint64_t here = __ballot((uint32_t)item < end && (uint32_t)item >= end - n);
        if (here != 0) {
            const int src = __builtin_ctzll(here), count = __builtin_amdgcn_readlane((int)n, src);
            take_piece(b0 + src, lane_span(s, src), count, item - (__builtin_amdgcn_readlane((int)end, src) - count), r);
            return true;
        }
        before = last_lane(end);
        b0 += kWave;
        if (b0 >= p.B) return false;
        s = span_of(p, b0 + lane);
        n = b0 + lane < p.B ? pieces_of(s.tiles, most, inverse) : 0u;
        end = before + wave_scan(n);
    }
}

// ---- lanes l, l^16, l^32, l^48 ---------------------------------------------------------------------------------------
__device__ __forceinline__ float col_max(float v)
{
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_sum(float v)
{
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int N> struct Words { uint32_t w[N]; };
// 16 bytes from each lane's address to LDS, at the wave's base + 16 * lane.
template <bool STREAM>
__device__ __forceinline__ void lds_load16(uint8_t* base, const uint8_t* p)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                     (__attribute__((address_space(3))) void*)base, 16, 0, STREAM ? 2 : 0);
}
template <bool STREAM, typename T>
__device__ __forceinline__ T load_as(const uint8_t* p)
{
    const T* at = reinterpret_cast<const T*>(p);
    if constexpr (STREAM) return __builtin_nontemporal_load(at);
    return *at;
}
template <int N, bool STREAM>
__device__ __forceinline__ Words<N> load_words(const uint8_t* p)
{
    Words<N> r;
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 v = load_as<STREAM, u32x4>(p + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[4 * i + e] = v[e];
        }
    } else if constexpr (N == 2) {
        const u32x2 v = load_as<STREAM, u32x2>(p);
        r.w[0] = v.x, r.w[1] = v.y;
    } else {
        r.w[0] = load_as<STREAM, uint32_t>(p);
    }
    return r;
}

// Two weights as bf16 values and what they keep beyond them, as bf16 too. FINITE: V holds no infinities (e4m3 has none), and the
// values are the nearest (17 bits together). Else they are cut toward zero (16 bits) and no remainder of a weight above 0 is 0: both
// terms then have the weight's sign, and an infinity in V meets neither a 0 nor a negative term, which would make NaN of it.
template <bool FINITE>
__device__ __forceinline__ u32x2 split_weights(float a, float b)
{
    if constexpr (FINITE) {
        const uint32_t top = pack_bf16x2(a, b);
        return {top, pack_bf16x2(a - __uint_as_float(top << 16), b - __uint_as_float(top & 0xFFFF0000u))};
    } else {
        const auto over = [](float v) {       // v is 0, at least the smallest normal value, or NaN, which its own value keeps
            return __builtin_amdgcn_fmed3f(v - __uint_as_float(__float_as_uint(v) & 0xFFFF0000u), 0x1p-126f, v);
        };
        return {__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u), pack_bf16x2(over(a), over(b))};
    }
}

// K goes straight to LDS where its registers would spill or halve the waves of a CU: bf16 heads of 256 (12000 positions of 8
// sequences 161 -> 146 us) and of 128 with two tiles of columns. Elsewhere a tile in registers is the better prefetch: its
// LDS place is free as soon as it is written, not when the scores are done (e4m3 139 us against 143 so, bf16 248 and 245).
constexpr bool loads_direct(int dim, bool fp8, int tiles) { return !fp8 && (dim == 256 || (dim == 128 && tiles > 1)); }

// P8: pages are multiples of eight positions, so eight aligned positions lie on one page
template <int D, bool FP8, bool P8>
struct Layout {
    static constexpr int kRow = D * (FP8 ? 1 : 2);           // bytes of a cache row
    static constexpr int kRowLanes = kRow / 16;              // lanes that load a K row, 16 bytes each
    static constexpr int kKLoads = kRowLanes / 2;            // K loads (and consecutive positions) per lane and tile
    static constexpr int kVWords = D / 32 / (FP8 ? 2 : 1);   // registers of a V row per lane (D/16 dims)
    static constexpr int kKStep = P8 ? (kKLoads < 8 ? kKLoads : 8) : 1;    // positions per page lookup
    static constexpr int kVStep = P8 ? 8 : 1;
    static constexpr int kKPages = kKLoads / kKStep, kVPages = 8 / kVStep;
    static constexpr int kQueryPitch = D / 8 + 1;            // 16-byte pieces between the queries in LDS
    static constexpr int kOutStride = D + 4;                 // floats between the columns of a wave's output in LDS
    static constexpr int kWaveLds = kCols * kOutStride * 4 > kTile * kRow ? kCols * kOutStride * 4 : kTile * kRow;
    // Where row r of a tile lies in the wave's LDS; loaded directly, by load (r % kKLoads) and lane group (r / kKLoads).
    template <bool DIRECT>
    static __device__ __forceinline__ int place(int r)
    {
        return DIRECT ? r % kKLoads * 1024 + r / kKLoads * kRow : r * kRow;
    }
    // Row r of a tile, 16-byte piece c, lies at piece c ^ swizzle(r): the 16 rows that one read takes (four of every
    // eight) then cover all banks.
    static __device__ __forceinline__ int swizzle(int r)
    {
        const int m = (r >> 3) * 4 + (r & 3);
        return kRow >= 256 ? m : kRow == 128 ? (m >> 1) & 7 : (m >> 2) & 3;
    }
};

// STREAM: a cache row is read by one block alone, and need not stay in the caches
// NT: tiles of columns. One tile's queries stay in registers; those of more, which would not fit beside NT outputs, in LDS.
template <int D, bool FP8, bool P8, bool STREAM, int NT>
__global__ void __launch_bounds__(kAttnBlock, blocks_per_cu(D, NT)) paged_attention_kernel(const AttnParams p)
{
    using L = Layout<D, FP8, P8>;
    __shared__ __attribute__((aligned(16))) uint8_t smem[kAttnWaves * L::kWaveLds];
    __shared__ float stats[kAttnWaves][2][kCols];
    __shared__ u32x4 queries[NT == 1 ? 1 : NT * kCols * L::kQueryPitch];
    // the column groups of a unit on one XCD, next to each other: they read the same cache rows
    int cg = 0, unit = (int)blockIdx.x;
    if (p.col_groups > 1) {
        const uint32_t eight = blockIdx.x / 8, of = p.by_col_groups.of(eight);
        cg = (int)(eight - of * (uint32_t)p.col_groups);
        unit = (int)(of * 8 + blockIdx.x % 8);
    }
    if (unit >= p.units) return;
    const int item = (int)p.by_kv_heads.of((uint32_t)unit), h = unit - item * p.cache.kv_heads;
    Piece pc;
    if (!find_piece(p, item, &pc)) return;
    if (p.part_of != nullptr && pc.index == 0 && h == 0 && cg == 0 && threadIdx.x == 0) p.part_of[pc.b] = int2{item, pc.count};

    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    // columns past the last (of a head group that is no multiple of 16) repeat it, and are not written
    const int c0 = cg * kCols * NT;
    const auto query_of = [&](int col, int* tok) {       // a column's query, and its token
        col = min(col, p.cols - 1);
        *tok = (int)p.by_group.of((uint32_t)col);
        return p.q + pc.b * p.qb + *tok * p.qt + (h * p.group + col - *tok * p.group) * p.qh;
    };
    int tok[NT], hi[NT], lo[NT];         // the token of the lane's columns, and the positions that it sees
    u32x4 q[NT == 1 ? D / 32 : 1];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const uint8_t* src = query_of(c0 + c * kCols + n, &tok[c]) + 16 * g;
        hi[c] = pc.len - (p.T - 1 - tok[c]), lo[c] = p.window > 0 ? hi[c] - p.window : 0;
        if constexpr (NT == 1) {
#pragma unroll
            for (int j = 0; j < D / 32; ++j) q[j] = *reinterpret_cast<const u32x4*>(src + 64 * j);
        }
    }
    if constexpr (NT > 1) {
        // column n's 16-byte piece i at n * kQueryPitch + i: an odd number of pieces apart, so a read covers all banks
        for (int e = (int)threadIdx.x; e < NT * kCols * (D / 8); e += kAttnBlock) {
            int t;
            const uint8_t* src = query_of(c0 + e / (D / 8), &t);
            queries[e / (D / 8) * L::kQueryPitch + e % (D / 8)] = *reinterpret_cast<const u32x4*>(src + e % (D / 8) * 16);
        }
        __syncthreads();
    }
    const auto query = [&](int c, int j) {
        if constexpr (NT == 1) return q[j];
        else return queries[(c * kCols + n) * L::kQueryPitch + 4 * j + g];
    };
    const int t_first = __builtin_amdgcn_readlane(tok[0], 0), t_last = __builtin_amdgcn_readlane(tok[NT - 1], kCols - 1);
    // positions that every token of the block sees
    const int all_hi = pc.len - (p.T - 1 - t_first), all_lo = p.window > 0 ? pc.len - (p.T - 1 - t_last) - p.window : 0;

    const float score_scale = p.scale * (p.cache.k_scale != nullptr ? p.cache.k_scale[h] : 1.0f);
    const int32_t* table = p.table + pc.b * p.table_stride;
    const int kpiece = lane % L::kRowLanes, krow = lane / L::kRowLanes * L::kKLoads;
    const uint8_t* kbase = p.cache.k + h * p.cache.kh;
    const uint8_t* vbase = p.cache.v + h * p.cache.vh + 4 * L::kVWords * n;
    const uint32_t last = (uint32_t)pc.len - 1;
    uint8_t* mine = smem + wave * L::kWaveLds;

    int kpage[L::kKPages], vpage[L::kVPages];
    // Page numbers of a tile's rows. Rows past the end take the last row's page (its bytes are there), and are masked.
    auto position = [&](uint32_t pos, uint32_t step) { return min(pos, last & ~(step - 1)); };
    auto lookup = [&](int tile) {
        const uint32_t p0 = (uint32_t)tile * kTile;
#pragma unroll
        for (int i = 0; i < L::kKPages; ++i)
            kpage[i] = table[p.cache.by_page.of(position(p0 + krow + i * L::kKStep, L::kKStep))];
#pragma unroll
        for (int i = 0; i < L::kVPages; ++i)
            vpage[i] = table[p.cache.by_page.of(position(p0 + 8 * g + i * L::kVStep, L::kVStep))];
    };
    auto in_cache = [&](int page) { return (uint32_t)page < (uint32_t)p.cache.pages; };
    constexpr bool kDirect = loads_direct(D, FP8, NT);
    Words<4> k[kDirect ? 1 : L::kKLoads];
    Words<L::kVWords> v[8];
    auto load_k = [&](int tile) {
#pragma unroll
        for (int i = 0; i < L::kKPages; ++i) {
            const uint32_t pos = position((uint32_t)tile * kTile + krow + i * L::kKStep, L::kKStep);
            const uint32_t at = pos - p.cache.by_page.of(pos) * (uint32_t)p.cache.page_size;
            const uint8_t* row = kbase + (in_cache(kpage[i]) ? kpage[i] : 0) * p.cache.kp + at * p.cache.kr;
#pragma unroll
            for (int e = 0; e < L::kKStep; ++e) {
                const int j = i * L::kKStep + e;       // row krow + j; directly, the lane asks for the piece its place holds
                if constexpr (kDirect)
                    lds_load16<STREAM>(mine + 1024 * j, row + e * p.cache.kr + 16 * (kpiece ^ L::swizzle(krow + j)));
                else
                    k[j] = load_words<4, STREAM>(row + e * p.cache.kr + 16 * kpiece);
            }
        }
    };
    const uint8_t* vrow[L::kVPages];
    uint32_t vok = 0;                  // bit i: the page of row 8 g + i is in the cache
    auto address_v = [&](int tile) {
        uint32_t ok = 0;
#pragma unroll
        for (int i = 0; i < L::kVPages; ++i) {
            const uint32_t pos = position((uint32_t)tile * kTile + 8 * g + i * L::kVStep, L::kVStep);
            const uint32_t at = pos - p.cache.by_page.of(pos) * (uint32_t)p.cache.page_size;
            const bool in = in_cache(vpage[i]);
            vrow[i] = vbase + (in ? vpage[i] : 0) * p.cache.vp + at * p.cache.vr;
            if (in) ok |= (P8 ? 0xFFu : 1u) << i;
        }
        return ok;
    };
    auto load_v = [&]() {
#pragma unroll
        for (int i = 0; i < L::kVPages; ++i)
#pragma unroll
            for (int e = 0; e < L::kVStep; ++e)
                v[i * L::kVStep + e] = load_words<L::kVWords, STREAM>(vrow[i] + e * p.cache.vr);
    };

    float m[NT], l[NT];
    f32x4 o[NT][D / 16];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        m[c] = -INFINITY, l[c] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[c][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    int tile = pc.tile0 + wave;
    if (tile < pc.tile1) {
        lookup(tile);
        vok = address_v(tile);
        load_k(tile);
        load_v();
        if (tile + kAttnWaves < pc.tile1) lookup(tile + kAttnWaves);
    }
    for (; tile < pc.tile1; tile += kAttnWaves) {
        const int next = tile + kAttnWaves;
        const bool more = next < pc.tile1;
        uint32_t vok_next = 0;
        const auto load_next = [&]() {
            if (!more) return;
            load_k(next);
            vok_next = address_v(next);
            if (next + kAttnWaves < pc.tile1) lookup(next + kAttnWaves);
        };
        if constexpr (kDirect) {
            __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt(0): the tile's rows are there
            wave_lds_order();
        } else {
#pragma unroll
            for (int i = 0; i < L::kKLoads; ++i) {
                const int r = krow + i;
                *reinterpret_cast<u32x4*>(mine + L::template place<false>(r) + 16 * (kpiece ^ L::swizzle(r))) =
                    u32x4{k[i].w[0], k[i].w[1], k[i].w[2], k[i].w[3]};
            }
            wave_lds_order();
            load_next();
        }
        const int p0 = tile * kTile;
        const bool masked = p0 + kTile > all_hi || p0 < all_lo || __ballot(vok != 0xFFu) != 0;
        u32x4 top8[NT], rest8[NT];       // the lane's eight weights of each column as bf16 values and remainders
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            // S^T: row m of half `half` is position 8 (m / 4) + 4 half + m % 4 of the tile, so a lane ends with positions
            // 8 g + 4 half + i, i = 0..3, of its column
            f32x4 s[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = (n >> 2) * 8 + half * 4 + (n & 3);
                const uint8_t* row = mine + L::template place<kDirect>(r);
                s[half] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    u32x4 a;
                    if constexpr (FP8) {
                        const uint2 w = *reinterpret_cast<const uint2*>(row + 16 * ((2 * j + (g >> 1)) ^ L::swizzle(r)) + 8 * (g & 1));
                        a = u32x4{fp8x2_to_bf16x2<false>(w.x), fp8x2_to_bf16x2<true>(w.x), fp8x2_to_bf16x2<false>(w.y),
                                  fp8x2_to_bf16x2<true>(w.y)};
                    } else {
                        a = *reinterpret_cast<const u32x4*>(row + 16 * ((4 * j + g) ^ L::swizzle(r)));
                    }
                    s[half] = mfma_16x16x32(a, query(c, j), s[half]);
                }
            }
            float top = -INFINITY, x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = s[i / 4][i % 4] * score_scale;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int pos = p0 + 8 * g + i;
                    const bool seen = (pos < hi[c]) & (pos >= lo[c]) & ((vok >> i & 1u) != 0u);
                    x[i] = seen ? x[i] : -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
            top = fmaxf(m[c], col_max(top));
            const float base = top == -INFINITY ? 0.0f : top;
            if (__ballot(top > m[c]) != 0) {
                const float fade = __builtin_amdgcn_exp2f(m[c] - base);
                l[c] *= fade;
#pragma unroll
                for (int j = 0; j < D / 16; ++j) o[c][j] *= fade;
                m[c] = top;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - base);
                l[c] += x[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x2 w = split_weights<FP8>(x[2 * i], x[2 * i + 1]);
                top8[c][i] = w.x, rest8[c][i] = w.y;
            }
        }
        wave_lds_order();
        if constexpr (kDirect) {
            __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0): the tile's rows are read, the next one's may take their place
            wave_lds_order();
            load_next();
        }
        // What no token sees of the tile goes out of V here. Where the tokens differ in what they see, weights of 0 keep the rest
        // of it out, unless a value there is not finite: then each token takes a product of its own.
        bool together = true;
        if (__builtin_expect(masked, 0)) {
            const int last_hi = pc.len - (p.T - 1 - t_last), first_lo = p.window > 0 ? pc.len - (p.T - 1 - t_first) - p.window : 0;
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pos = p0 + 8 * g + i;
                const bool some = (pos < last_hi) & (pos >= first_lo) & ((vok >> i & 1u) != 0u);
#pragma unroll
                for (int e = 0; e < L::kVWords; ++e) {
                    const uint32_t w = some ? v[i].w[e] : 0u;
                    v[i].w[e] = w;
                    // the top bit of each value whose exponent (e4m3: everything but the sign) is all ones
                    odd |= FP8 ? ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u : ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
                }
            }
            together = t_first == t_last || __ballot(odd != 0) == 0;
        }
        // O^T += V^T P^T: rows 8 g + i, i = 0..7, of the tile against the lane's own eight weights. `see`: bit i keeps row
        // i; with `all` every row and column takes the product, else those of token t.
        auto add_pv = [&](uint32_t see, bool all, int t) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                uint32_t x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (FP8)
                        x[i] = d % 2 ? fp8x2_to_bf16x2<true>(v[i].w[d / 2]) : fp8x2_to_bf16x2<false>(v[i].w[d / 2]);
                    else
                        x[i] = v[i].w[d];
                    if (!all) x[i] = see >> i & 1u ? x[i] : 0u;
                }
                const u32x4 even = {__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                                    __builtin_amdgcn_perm(x[5], x[4], 0x05040100u), __builtin_amdgcn_perm(x[7], x[6], 0x05040100u)};
                const u32x4 odd = {__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                                   __builtin_amdgcn_perm(x[5], x[4], 0x07060302u), __builtin_amdgcn_perm(x[7], x[6], 0x07060302u)};
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    const f32x4 a = mfma_16x16x32(even, top8[c], mfma_16x16x32(even, rest8[c], o[c][2 * d]));
                    const f32x4 b = mfma_16x16x32(odd, top8[c], mfma_16x16x32(odd, rest8[c], o[c][2 * d + 1]));
                    if (all) {
                        o[c][2 * d] = a, o[c][2 * d + 1] = b;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[c][2 * d][e] = tok[c] == t ? a[e] : o[c][2 * d][e];
                            o[c][2 * d + 1][e] = tok[c] == t ? b[e] : o[c][2 * d + 1][e];
                        }
                    }
                }
            }
        };
        if (__builtin_expect(together, 1)) {
            add_pv(0xFFu, true, 0);
        } else {
            for (int t = t_first; t <= t_last; ++t) {
                const int thi = pc.len - (p.T - 1 - t), tlo = p.window > 0 ? thi - p.window : 0;
                uint32_t see = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int pos = p0 + 8 * g + i;
                    if (pos < thi && pos >= tlo) see |= 1u << i;
                }
                add_pv(see, false, t);
            }
        }
        vok = vok_next;
        if (more) load_v();
    }

    // join the block's waves, a tile of columns at a time: column n of a wave's O^T lies at [n][dim], dims (4 g + i) D/16 + j
    const float v_scale = p.cache.v_scale != nullptr ? p.cache.v_scale[h] : 1.0f;
    float* part = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
        if (ct > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 16; j += 4)
                *reinterpret_cast<f32x4*>(part + n * L::kOutStride + (4 * g + i) * (D / 16) + j) =
                    f32x4{o[ct][j][i], o[ct][j + 1][i], o[ct][j + 2][i], o[ct][j + 3][i]};
        const float weight = col_sum(l[ct]);
        if (g == 0) stats[wave][0][n] = m[ct], stats[wave][1][n] = weight;
        __syncthreads();
        for (int e = (int)threadIdx.x; e < kCols * (D / 4); e += kAttnBlock) {
            const int cn = e / (D / 4), d = e % (D / 4) * 4, c = c0 + ct * kCols + cn;
            if (c >= p.cols) break;
            float all = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) all = fmaxf(all, stats[w][0][cn]);
            const float base = all == -INFINITY ? 0.0f : all;
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(stats[w][0][cn] - base);
                sum += f * stats[w][1][cn];
                acc += f * *reinterpret_cast<const f32x4*>(smem + w * L::kWaveLds + 4 * (cn * L::kOutStride + d));
            }
            if (pc.count > 1) {
                const int64_t at = (int64_t)unit * p.cols + c;
                *reinterpret_cast<f32x4*>(p.part_o + at * D + d) = acc;
                if (d == 0) p.part_ml[2 * at] = all, p.part_ml[2 * at + 1] = sum;
                continue;
            }
            const int t = (int)p.by_group.of((uint32_t)c);
            const int64_t row = ((int64_t)pc.b * p.T + t) * p.heads + h * p.group + c - t * p.group;
            const float f = sum == 0.0f ? 0.0f : v_scale / sum;
            const uint2 y = {pack_bf16x2(acc[0] * f, acc[1] * f), pack_bf16x2(acc[2] * f, acc[3] * f)};
            *reinterpret_cast<uint2*>(p.out + row * D + d) = y;
            if (d == 0 && p.lse != nullptr) p.lse[row] = (all + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
        }
    }
}

// Joins the pieces of the sequences that have several: a block per sequence, kv head and column; D/4 lanes hold the output,
// the block's groups of them take the pieces in turn, kJoinAhead loads of each in flight.
constexpr int kJoinAhead = 4;
template <int D>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p)
{
    constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
    __shared__ f32x4 acc_of[kGroups][kLanes];
    __shared__ float m_of[kGroups], l_of[kGroups];
    const int b = (int)blockIdx.x, h = (int)blockIdx.y, c = (int)blockIdx.z, hkv = p.cache.kv_heads;
    const int2 items = p.part_of[b];
    if (items.y == 1) return;
    const int grp = (int)threadIdx.x / kLanes, i4 = (int)threadIdx.x % kLanes;
    float m = -INFINITY, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = grp; j < items.y; j += kGroups * kJoinAhead) {
        f32x4 x[kJoinAhead];
        float pm[kJoinAhead], pl[kJoinAhead];
#pragma unroll
        for (int i = 0; i < kJoinAhead; ++i) {
            const bool in = j + i * kGroups < items.y;
            const int64_t at = ((int64_t)(items.x + (in ? j + i * kGroups : j)) * hkv + h) * p.cols + c;
            x[i] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + 4 * i4);
            pm[i] = p.part_ml[2 * at], pl[i] = p.part_ml[2 * at + 1];
            if (!in) pm[i] = -INFINITY, pl[i] = 0.0f, x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < kJoinAhead; ++i) top = fmaxf(top, pm[i]);
        const float base = top == -INFINITY ? 0.0f : top, fade = __builtin_amdgcn_exp2f(m - base);
        acc *= fade;
        l *= fade;
#pragma unroll
        for (int i = 0; i < kJoinAhead; ++i) {
            const float f = __builtin_amdgcn_exp2f(pm[i] - base);
            acc += x[i] * f;
            l += pl[i] * f;
        }
        m = top;
    }
    acc_of[grp][i4] = acc;
    if (i4 == 0) m_of[grp] = m, l_of[grp] = l;
    __syncthreads();
    if (grp != 0) return;
    float all = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kGroups; ++w) all = fmaxf(all, m_of[w]);
    const float base = all == -INFINITY ? 0.0f : all;
    acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
        const float f = __builtin_amdgcn_exp2f(m_of[w] - base);
        sum += f * l_of[w];
        acc += f * acc_of[w][i4];
    }
    const int t = (int)p.by_group.of((uint32_t)c);
    const int64_t row = ((int64_t)b * p.T + t) * p.heads + h * p.group + c - t * p.group;
    const float f = sum == 0.0f ? 0.0f : (p.cache.v_scale != nullptr ? p.cache.v_scale[h] : 1.0f) / sum;
    const uint2 y = {pack_bf16x2(acc[0] * f, acc[1] * f), pack_bf16x2(acc[2] * f, acc[3] * f)};
    *reinterpret_cast<uint2*>(p.out + row * D + 4 * i4) = y;
    if (i4 == 0 && p.lse != nullptr) p.lse[row] = (all + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// ---- host ------------------------------------------------------------------------------------------------------------
// A launch has less than 2^32 threads; a block of the first grid for every sequence at least, so the joining one is bounded too.
constexpr int64_t kMostBlocks = ((1ll << 32) - 1) / 256;
static_assert(kAttnBlock == 256);
// The launch's plan with up to `most` tiles of columns a block, and its workspace; false where it is more than a launch takes.
static bool plan_blocks(const paia_kv_cache* c, int most, AttnParams* p, int64_t* bytes)
{
    const int B = p->B;
    // The columns' tiles over the fewest blocks, evenly.
    const int tiles = (p->cols + kCols - 1) / kCols;
    p->tiles = (tiles + (tiles + most - 1) / most - 1) / ((tiles + most - 1) / most);
    p->col_groups = (tiles + p->tiles - 1) / p->tiles;
    const int64_t wide = (int64_t)c->kv_heads * p->col_groups, slots = (int64_t)device_facts().cus * blocks_per_cu(c->head_dim, p->tiles);
    int64_t target = slots / wide;
    target = target < 2 ? 2 : target;
    // One round of blocks where the sequences are few; many sequences have a piece of their own each, and as many more as a
    // round (200 sequences of 30 to 3000: 114 us; half a round more 125, two rounds 111, but 64 of 1000 48, 51 and 53).
    const int64_t goal = B <= target / 2 ? target : target + B;
    // pieces per sequence that the table's width allows
    const int64_t per_seq = ((int64_t)p->max_len / kTile + 1 + kMinTiles - 1) / kMinTiles;
    const int64_t items = goal < per_seq * B ? goal : per_seq * B;
    const int64_t units = items * c->kv_heads, blocks = (units + 7) / 8 * 8 * p->col_groups;
    if (blocks > kMostBlocks) return false;
    p->goal = (int)goal;
    p->units = (int)units;
    p->by_kv_heads = Divisor((uint32_t)c->kv_heads);
    p->by_group = Divisor((uint32_t)p->group);
    p->by_col_groups = Divisor((uint32_t)p->col_groups);
    // one piece a sequence at most: nothing is joined
    *bytes = per_seq <= 1 ? 0 : units * p->cols * (c->head_dim + 2) * (int64_t)sizeof(float) + B * (int64_t)sizeof(int2);
    return true;
}
// The same for a call; false where its sizes leave the contract. The workspace serves any window: where the tiles that a block takes go
// by the window, it is the larger one of both forms.
static bool attention_plan(const paia_kv_cache* c, int table_width, int B, int T, int heads, int window, AttnParams* p, int64_t* bytes)
{
    if (!cache_view(c, &p->cache) || table_width < 0 || B < 0 || T <= 0 || heads <= 0 || heads % c->kv_heads || window < 0) return false;
    p->B = B, p->T = T, p->heads = heads;
    p->group = heads / c->kv_heads;
    const int64_t cols = (int64_t)T * p->group, max_len = (int64_t)table_width * c->page_size;
    if (cols > 65535 || c->kv_heads > 65535) return false;      // dimensions of the joining grid
    // tile numbers times 32, with a tile to spare, and a length less T and a window (below max_len) stay within 32 bits
    constexpr int kLongest = INT_MAX - (1 << 17);
    p->max_len = (int)(max_len < kLongest ? max_len : kLongest);
    p->cols = (int)cols;
    p->window = window >= p->max_len ? 0 : window;     // it hides nothing
    const double row = 2.0 * c->kv_heads * c->head_dim * (c->fp8 ? 1 : 2);
    const int most = most_tiles(c->head_dim, c->page_size % 8 == 0);
    if (!table_is_large(row, B, p->max_len)) return plan_blocks(c, 1, p, bytes);
    const bool together = window_is_large(row, B, T, p->window);
    int64_t other = 0;
    if (!plan_blocks(c, together ? 1 : most, p, &other)) other = 0;
    if (!plan_blocks(c, together ? most : 1, p, bytes)) return false;
    *bytes = *bytes > other ? *bytes : other;
    return true;
}

// Several column groups read the same rows, next to each other on one XCD: with streaming loads its L2 served them worse (heads
// of 256, five tokens of 8 heads a group, 12000 positions: 532 us against 281).
template <int D, bool FP8, bool P8>
static auto attention_kernel(int tiles, bool stream)
{
    if constexpr (most_tiles(D, P8) >= 2)
        if (tiles == 2) return paged_attention_kernel<D, FP8, P8, false, 2>;
    if constexpr (most_tiles(D, P8) >= 3)
        if (tiles == 3) return paged_attention_kernel<D, FP8, P8, false, 3>;
    return stream ? paged_attention_kernel<D, FP8, P8, true, 1> : paged_attention_kernel<D, FP8, P8, false, 1>;
}
template <int D>
static int launch_attention(const AttnParams& p, bool fp8, bool join, hipStream_t st)
{
    const dim3 grid((uint32_t)((p.units + 7) / 8 * 8 * p.col_groups));
    const bool p8 = p.cache.page_size % 8 == 0;
    const bool alone = p.col_groups == 1;
    const auto kernel = fp8 ? (p8 ? attention_kernel<D, true, true>(p.tiles, alone) : attention_kernel<D, true, false>(p.tiles, alone))
                            : (p8 ? attention_kernel<D, false, true>(p.tiles, alone) : attention_kernel<D, false, false>(p.tiles, alone));
    hipLaunchKernelGGL(kernel, grid, dim3(kAttnBlock), 0, st, p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    if (join) {
        hipLaunchKernelGGL((attention_join_kernel<D>), dim3((uint32_t)p.B, (uint32_t)p.cache.kv_heads, (uint32_t)p.cols), dim3(256), 0, st, p);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
    }
    return 0;
}

}  // namespace paia

extern "C" {

long long paia_paged_attention_workspace(const paia_kv_cache* cache, int table_width, int B, int T, int heads)
{
    paia::AttnParams p;
    int64_t bytes = 0;
    return paia::attention_plan(cache, table_width, B, T, heads, 0, &p, &bytes) ? bytes : -2;
}

int paia_paged_attention(const void* q, const long long* q_strides, const paia_kv_cache* cache, const void* block_table,
                         long long table_stride, int table_width, const void* lens, float scale, int window, void* out,
                         void* lse, int B, int T, int heads, void* workspace, long long workspace_bytes, void* stream)
{
    using namespace paia;
    AttnParams p;
    int64_t bytes = 0;
    if (!attention_plan(cache, table_width, B, T, heads, window, &p, &bytes) || table_stride < 0) return -2;
    if (B == 0) return 0;
    if (q == nullptr || q_strides == nullptr || lens == nullptr || out == nullptr || (block_table == nullptr && table_width > 0))
        return -2;
    if (out == q || !aligned(q, 16) || !aligned(block_table, 4) || !aligned(lens, 4) || !aligned(out, 16) || !aligned(lse, 4)) return -2;
    for (int i = 0; i < 3; ++i)
        if (q_strides[i] < 0 || q_strides[i] % 8) return -2;
    if (bytes > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < bytes)) return -2;
    p.q = static_cast<const uint8_t*>(q);
    p.qb = q_strides[0] * 2, p.qt = q_strides[1] * 2, p.qh = q_strides[2] * 2;
    p.out = static_cast<uint16_t*>(out);
    p.lse = static_cast<float*>(lse);
    p.table = static_cast<const int32_t*>(block_table);
    p.lens = static_cast<const int32_t*>(lens);
    p.table_stride = table_stride;
    p.scale = scale * 1.4426950408889634f;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + (int64_t)p.units * p.cols * cache->head_dim;
    p.part_of = bytes > 0 ? reinterpret_cast<int2*>(p.part_ml + (int64_t)p.units * p.cols * 2) : nullptr;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (cache->head_dim) {
    case 64: return launch_attention<64>(p, cache->fp8, bytes > 0, st);
    case 128: return launch_attention<128>(p, cache->fp8, bytes > 0, st);
    default: return launch_attention<256>(p, cache->fp8, bytes > 0, st);
    }
}

}  // extern "C"
