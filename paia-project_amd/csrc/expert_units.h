// Which pairs, columns and part of K each block and wave of the experts' products has: arithmetic on sizes and offsets alone, the
// same for the kernels (constexpr: on either side) and for a host compiler, which tests it without a GPU.
#pragma once
#include <stdint.h>

namespace paia {

constexpr int64_t kMostBlocks = 1 << 22;         // of a launch
constexpr int64_t kMostItems = 1 << 20;          // of the form for few rows: item * block stays below 2^32

#define PAIA_UNITS __attribute__((always_inline)) constexpr

PAIA_UNITS int lesser(int a, int b) { return a < b ? a : b; }
PAIA_UNITS int greater(int a, int b) { return a > b ? a : b; }

// Chunks of at most BM pairs that R pairs of E experts, those without an expert apart, can make.
PAIA_UNITS int64_t most_chunks(int64_t R, int64_t E, int BM) { return (R + (R < E + 1 ? R : E + 1) * (BM - 1)) / BM; }
PAIA_UNITS int chunks_of(int pairs, int BM) { return (int)(((uint32_t)pairs + (uint32_t)BM - 1u) / (uint32_t)BM); }     // pairs >= 0

// Where expert e's pairs begin. Offsets are taken as they are but for their range: whatever they hold, the pairs of a chunk
// lie within the call's.
PAIA_UNITS int pairs_begin(const int32_t* offsets, int e, int E, int R)
{
    return lesser(greater(offsets[lesser(e, E)], 0), R);
}

// A lane's share of the experts, n from expert e0 on: their chunks, no more than the launch has blocks for (unless the offsets are not
// in order there are no more in all), where the pairs of the first begin, and of the last end.
struct LaneChunks {
    int own, from, to;
};
PAIA_UNITS LaneChunks lane_chunks(const int32_t* offsets, int E, int R, int BM, int e0, int n, int most)
{
    LaneChunks c = {0, pairs_begin(offsets, e0, E, R), 0};
    for (int i = 1, begin = c.from; i <= n; ++i) {
        c.to = pairs_begin(offsets, e0 + i, E, R);
        c.own += chunks_of(greater(c.to - begin, 0), BM);
        begin = c.to;
    }
    c.own = lesser(c.own, most);
    return c;
}

// The expert of a chunk, its pairs order[lo .. hi), and its chunks begin .. begin + n - 1.
struct ChunkExpert {
    int expert, lo, hi, begin, n;
};
// That of chunk c, which is one of the lane's own: begin .. begin + own - 1.
PAIA_UNITS ChunkExpert expert_of(const int32_t* offsets, int E, int R, int BM, int e0, int n, const LaneChunks lane, int begin, int c)
{
    ChunkExpert x = {e0, lane.from, lane.to, begin, lane.own};
    if (n > 1) {
        int at = begin, a = lane.from;
        for (int i = 1; i <= n; ++i) {
            const int b = pairs_begin(offsets, e0 + i, E, R), k = chunks_of(greater(b - a, 0), BM);
            if (c >= at && c < at + k) x = {e0 + i - 1, a, b, at, k};
            at += k;
            a = b;
        }
    }
    return x;
}

// Block b's place when each of the 8 XCDs, to which blocks are dealt in turn, takes a contiguous range of n.
PAIA_UNITS int xcd_contiguous(int b, int n) { return b % 8 * (n / 8) + lesser(b % 8, n % 8) + b / 8; }

struct ExpertUnit {
    int expert;              // E: pairs without an expert; -1: no unit
    int first, held, tile;   // its pairs are order[first .. first + held)
    int chunks;              // of its expert
};
// Unit u, of a chunk of expert x: units of one expert and tile (or group of tiles) follow each other.
template <int BM>
PAIA_UNITS ExpertUnit unit_in(const ChunkExpert x, int u, int tiles)
{
    // eight tiles at a time through all of many chunks: of 8 tiles by 8 chunks, as an XCD holds at a time, rows and weights alike come
    // once to its L2 (us, two of 8 experts 28672x4096 e4m3, 8001 tokens 3836 -> 3265, 4001 1738 -> 1681; fewer chunks +-1%)
    const int local = u - x.begin * tiles;
    int tile = 0, chunk = 0;
    if (BM < 256 && x.n >= 6) {
        const int g = local / (8 * x.n), in = local - g * 8 * x.n, wide = lesser(8, tiles - g * 8);
        chunk = in / wide, tile = g * 8 + in - chunk * wide;
    } else {
        tile = local / x.n, chunk = local - tile * x.n;
    }
    const int first = x.lo + chunk * BM;
    return {x.expert, first, lesser(BM, x.hi - first), tile, x.n};
}
// Unit u of chunk c of the pairs without an expert, which are order[at .. R).
template <int BM>
PAIA_UNITS ExpertUnit unit_without(int E, int R, int at, int c, int u_in_chunk)
{
    const int first = at + c * BM;
    return {E, first, lesser(BM, R - first), u_in_chunk, 0};
}

// Where the share of block b of `blocks` begins among n (T holds n * blocks); where the part of wave w of `waves` does among a row's
// stages.
template <typename T>
PAIA_UNITS T share_begin(T n, T b, T blocks) { return n * b / blocks; }
PAIA_UNITS int wave_begin(int stages, int w, int waves) { return stages * w / waves; }

#undef PAIA_UNITS

}  // namespace paia
