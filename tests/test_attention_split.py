"""How paged attention splits sequences into pieces, replayed on the CPU: the kernels derive the split from lengths that only
the device knows, within a grid and a workspace that the host fixed before (csrc/paged_attention.hip: find_piece, pieces_of,
attention_plan). Every tile must lie in exactly one piece and the pieces must fit the grid, whatever the lengths are."""
import random
import struct

import pytest

TILE, MIN_TILES, WAVES = 32, 4, 4


def span(n, T, window, max_len):
    n = min(max(n, 0), max_len)
    tile0 = max(0, n - (T - 1) - window) // TILE if window else 0
    return tile0, -(-n // TILE) - tile0


def f32(v):
    return struct.unpack("f", struct.pack("f", v))[0]


def pieces_of(tiles, most, inverse):
    n = int(f32(f32(tiles) * inverse))
    left = tiles - n * most
    more = int(f32(f32(left) * inverse))
    n, left = n + more, left - more * most
    if left < 0:
        n, left = n - 1, left + most
    if left >= most:
        n, left = n + 1, left - most
    assert 0 <= left < most and n >= 0
    return max(1, n + (left > 0))


def whole_rounds(tiles):
    return (int(tiles) // WAVES + 1) * WAVES


def piece_tiles(tiles, goal, jitter):
    """`jitter`: relative error of the hardware's reciprocal, at most 1 ulp."""
    rcp = lambda v: f32(f32(1.0 / v) * (1.0 + jitter))  # noqa: E731
    if len(tiles) == 1:
        mean = -(-tiles[0] // goal)
        most = max(MIN_TILES, -(-mean // WAVES) * WAVES)
        return most, rcp(most), 0
    per, most = rcp(goal), MIN_TILES
    for tries in range(6):
        inverse = rcp(most)
        count = sum(pieces_of(t, most, inverse) for t in tiles)
        if count <= goal:
            break
        held = f32(most * f32(count))
        if tries == 0:
            total = held
        most = whole_rounds(f32(held * per) if tries < 3 else f32(f32(total * f32(1.001)) * rcp(goal - len(tiles))))
    return most, inverse, tries


def plan(B, target, max_len):
    goal = target if B <= target // 2 else target + B
    per_seq = (max_len // TILE + 1 + MIN_TILES - 1) // MIN_TILES
    return goal, min(goal, per_seq * B), per_seq


@pytest.mark.parametrize("seed", range(40))
def test_pieces_cover_every_tile_once_and_fit(seed):
    r = random.Random(seed)
    for _ in range(60):
        B, target, T = r.choice([1, 2, 3, 16, 63, 64, 65, 200]), r.choice([2, 3, 7, 64, 96, 128, 768]), r.choice([1, 2, 5])
        max_len = r.choice([0, 1, 31, 32, 256, 257, 5000, 131072, 2 ** 31 - 5000])
        window = r.choice([0, 0, 1, 33, 4096])
        lens = [r.choice([0, 1, max_len, r.randint(0, max(1, max_len)), r.randint(0, 2 ** 31 - 1)]) for _ in range(B)]
        spans = [span(n, T, window, max_len) for n in lens]
        goal, items, per_seq = plan(B, target, max_len)
        most, inverse, tries = piece_tiles([t for _, t in spans], goal, r.choice([-1, 0, 1]) * 2.0 ** -23)
        assert tries <= 4
        used = 0
        for tile0, tiles in spans:
            n = max(1, -(-tiles // most))
            assert B == 1 or n == pieces_of(tiles, most, inverse)
            used += n
            each, more = divmod(tiles, n)
            ends = [(j * each + min(j, more), (j + 1) * each + min(j + 1, more)) for j in range(n)]
            assert ends[0][0] == 0 and ends[-1][1] == tiles
            assert all(a[1] == b[0] for a, b in zip(ends, ends[1:]))
            assert all(a < b for a, b in ends) or tiles == 0
            assert all(b - a <= most for a, b in ends) and tile0 >= 0 and tiles >= 0
        assert used <= items, (used, B, target, max_len)
        if per_seq <= 1:
            assert used == B


def test_uniform_lengths_use_what_is_aimed_at():
    """Equal sequences: between half and all of the pieces aimed at, and never more."""
    for B in (1, 4, 16, 32):
        for n in (4096, 32768, 131072):
            goal, _, _ = plan(B, 64, n)
            most, inverse, _ = piece_tiles([n // TILE] * B, goal, 0.0)
            used = B * pieces_of(n // TILE, most, inverse)
            assert 32 <= used <= 64 or most == MIN_TILES


def test_division_by_multiplication():
    """csrc/divisor.h: exact for every dividend below 2^31."""
    r = random.Random(1)
    for d in list(range(1, 300)) + [2 ** k + e for k in range(8, 31) for e in (-1, 0, 1)] + [2 ** 31 - 1]:
        s = 0
        while 2 ** s < d:
            s += 1
        m = (2 ** (31 + s) + d - 1) // d
        assert m < 2 ** 32
        for n in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1, (2 ** 31 - 1) // d * d, (2 ** 31 - 1) // d * d - 1] + \
                [r.randrange(2 ** 31) for _ in range(50)]:
            if 0 <= n < 2 ** 31:
                assert ((2 * n) % 2 ** 32 * m >> 32) >> s == n // d, (n, d)
