// How many tiles of columns (token, head) a block of paged attention takes together: the rule alone, plain C++.
#pragma once
#include <stdint.h>

namespace paia {

constexpr int kCols = 16;            // columns of a matrix tile
// Tiles of columns that a block takes together, so that each row is read once for all: as many as a lane's registers hold the
// outputs of, or nearly. Heads of 128 with two tiles spill (132 bytes a lane in e4m3, 36 in bf16), and so do heads of 64 with three on
// pages that are no multiple of eight (36 and 100); all gain on large caches all the same.
constexpr int most_tiles(int dim, bool p8) { return dim <= 64 ? 3 : dim <= 128 && p8 ? 2 : 1; }
// A block of several tiles stages its queries and does more after its last row, so it takes caches that fill the chip for longer. The
// host knows what the sequences may hold, not what they do: the bytes of B tables, and with a window those of B windows, which need
// only be half as many. Five tokens of 4 and of 8 heads a group, 8 sequences, us with one tile a block / together:
//   bf16 heads of 128, 2500 positions 20.7 / 22.2 and 23.9 / 25.9; 6000 (164 MB) 43.7 / 41.0 and 53.1 / 49.0; 16000 87.1 / 81.5
//   and 116.8 / 97.7; heads of 64, 6000 (82 MB) 22.0 / 24.5 and 28.9 / 29.3; 16000 (200 MB) 51.9 / 47.3 and 65.3 / 52.1; e4m3
//   heads of 128, 16000 (200 MB) 67.0 / 55.6 and 98.8 / 86.9; of 64 (100 MB) 43.4 / 40.8 and 57.4 / 47.3.
// Tables of 32768 positions: a window of 1024, bf16 heads of 128 (34 MB) 16.4 / 18.3 and 19.9 / 20.8, of 64 13.0 / 14.5 and 15.7 /
//   19.1; e4m3 15.2 / 17.9 and 19.5 / 21.2, 11.5 / 13.0 and 14.6 / 17.9; of 4096, e4m3 heads of 128 (67 MB) 26.3 / 27.5 and 40.6 / 35.7,
//   bf16 heads of 64 on pages of 7 (67 MB) 24.6 / 23.4 and 32.8 / 29.1, e4m3 heads of 64 (34 MB) 19.1 / 20.2 and 24.3 / 25.8.
// Sequences that are short beside their tables, without a window, pay for it: 1000 positions 16.4 / 16.9 and 18.7 / 20.7 (bf16 heads of
//   128), 15.2 / 16.2 and 17.8 / 21.3 (e4m3).
constexpr int64_t kTogether = 120 << 20, kTogetherWindow = 60 << 20;
// `row`: bytes of a position's k and v over all kv heads
constexpr bool table_is_large(double row, int B, int max_len) { return row * B * max_len >= (double)kTogether; }
constexpr bool window_is_large(double row, int B, int T, int window)      // window 0: none
{
    return window == 0 || row * B * ((double)window + T - 1) >= (double)kTogetherWindow;
}

}  // namespace paia
