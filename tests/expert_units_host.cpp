// The experts' kernels' arithmetic (csrc/expert_units.h) compiled for the host: 64 lanes as a loop where a wave has them side by side.
#include "expert_units.h"

using namespace paia;

namespace {

struct Wave {
    const int32_t* offsets;
    int E, R, BM, per, count, rest_at, rest;
    LaneChunks lane[64];
    int upto[64];
    Wave(const int32_t* o, int E_, int R_, int BM_) : offsets(o), E(E_), R(R_), BM(BM_), per((E_ + 63) / 64)
    {
        const int most = (int)most_chunks(R, E, BM);
        int sum = 0;
        for (int l = 0; l < 64; ++l) {
            lane[l] = lane_chunks(offsets, E, R, BM, l * per, per, most);
            upto[l] = sum += lane[l].own;
        }
        count = lesser(sum, most);
        rest_at = pairs_begin(offsets, E, E, R);
        rest = lesser(chunks_of(R - rest_at, BM), most - count);
    }
    ChunkExpert of(int c) const
    {
        int l = 0;
        while (upto[l] <= c) ++l;
        return expert_of(offsets, E, R, BM, l * per, per, lane[l], upto[l] - lane[l].own, c);
    }
};

template <int BM>
void units(const Wave& w, int tiles, int blocks, ExpertUnit* out)
{
    const int n = w.count * tiles;
    for (int b = 0; b < blocks; ++b) {
        if (b >= n + w.rest * tiles) {
            out[b] = {-1, 0, 0, 0, 0};
            continue;
        }
        const int u = b < n ? xcd_contiguous(b, n) : b, c = u / tiles;
        out[b] = c >= w.count ? unit_without<BM>(w.E, w.R, w.rest_at, c - w.count, u - c * tiles) : unit_in<BM>(w.of(c), u, tiles);
    }
}

}  // namespace

extern "C" {

int64_t host_most_chunks(int64_t R, int64_t E, int BM) { return most_chunks(R, E, BM); }
int64_t host_most_blocks() { return kMostBlocks; }
int64_t host_most_items() { return kMostItems; }
int host_wave_begin(int stages, int w, int waves) { return wave_begin(stages, w, waves); }
uint64_t host_share(uint64_t n, uint64_t b, uint64_t blocks) { return share_begin<uint64_t>(n, b, blocks); }
uint32_t host_share32(uint32_t n, uint32_t b, uint32_t blocks) { return share_begin<uint32_t>(n, b, blocks); }
int host_xcd(int b, int n) { return xcd_contiguous(b, n); }

// The units of all blocks of a launch of the form for many rows.
int host_units(const int32_t* offsets, int E, int R, int BM, int tiles, int blocks, ExpertUnit* out)
{
    const Wave w(offsets, E, R, BM);
    switch (BM) {
    case 16: units<16>(w, tiles, blocks, out); return 0;
    case 32: units<32>(w, tiles, blocks, out); return 0;
    case 64: units<64>(w, tiles, blocks, out); return 0;
    case 128: units<128>(w, tiles, blocks, out); return 0;
    case 256: units<256>(w, tiles, blocks, out); return 0;
    }
    return -1;
}

// The runs of items of all blocks of a launch of the form for few rows, five numbers each: expert, first pair, pairs, first tile, tiles;
// how many runs, or -1 where they are more than `room`.
int host_runs(const int32_t* offsets, int E, int R, int MT, int tiles, int blocks, int room, int32_t* out)
{
    const Wave w(offsets, E, R, MT);
    const uint32_t items = (uint32_t)(w.count * tiles);
    int n = 0;
    for (int b = 0; b < blocks; ++b) {
        const uint32_t block = (uint32_t)xcd_contiguous(b, blocks), end = share_begin<uint32_t>(items, block + 1, (uint32_t)blocks);
        for (uint32_t item = share_begin<uint32_t>(items, block, (uint32_t)blocks); item < end;) {
            const int chunk = (int)item / tiles, tile = (int)item - chunk * tiles, wide = lesser(tiles - tile, (int)(end - item));
            const ChunkExpert x = w.of(chunk);
            const int first = x.lo + (chunk - x.begin) * MT;
            if (n == room) return -1;
            const int32_t run[5] = {x.expert, first, lesser(MT, x.hi - first), tile, wide};
            for (int i = 0; i < 5; ++i) out[5 * n + i] = run[i];
            ++n;
            item += (uint32_t)wide;
        }
    }
    return n;
}

}  // extern "C"
