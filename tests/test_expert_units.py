"""How blocks find their work among the experts (unit_of in csrc/experts_kernel.h), replayed on the CPU: for offsets in order every
pair and tile is some block's exactly once and the launch has blocks enough; whatever the offsets hold, what a block takes lies
within the pairs."""
import random

import pytest


def blocks_of(R, E, BM, tiles):
    most = (R + min(R, E + 1) * (BM - 1)) // BM
    return most, most * tiles


def units(offsets, R, E, BM, tiles):
    """[(expert, first, held, tile)] of all blocks, None for one without work."""
    per = -(-E // 64)
    most, blocks = blocks_of(R, E, BM, tiles)
    place = lambda e: min(max(offsets[min(e, E)], 0), R)  # noqa: E731
    own = []
    for lane in range(64):
        n, at = 0, place(lane * per)
        for i in range(1, per + 1):
            to = place(lane * per + i)
            n += (max(to - at, 0) + BM - 1) // BM
            at = to
        own.append(min(n, most))
    upto = [sum(own[:i + 1]) for i in range(64)]
    chunks = min(upto[63], most)
    rest = place(E)
    total = min(chunks + (R - rest + BM - 1) // BM, most) * tiles
    out = []
    for b in range(blocks):
        if b >= total:
            out.append(None)
            continue
        xcd, real = b % 8, chunks * tiles
        u = xcd * (real // 8) + min(xcd, real % 8) + b // 8 if b < real else b
        c = u // tiles
        if c >= chunks:
            first = rest + (c - chunks) * BM
            out.append((E, first, min(BM, R - first), u - c * tiles))
            continue
        lane = next(i for i in range(64) if upto[i] > c)
        found, at, start = (0, 0, 0, 0, 1), upto[lane] - own[lane], place(lane * per)
        for i in range(1, per + 1):
            to = place(lane * per + i)
            k = (max(to - start, 0) + BM - 1) // BM
            if at <= c < at + k:
                found = (lane * per + i - 1, at, start, to, k)
            at, start = at + k, to
        e, begin, lo, hi, n = found
        local, group = u - begin * tiles, 8 if BM < 256 and n >= 6 else 1
        g = local // (group * n)
        wide = min(group, tiles - g * group)
        chunk, at = divmod(local - g * group * n, wide)
        tile, first = g * group + at, lo + chunk * BM
        out.append((e, first, min(BM, hi - first), tile))
    return out


def counts_of(rng, E, R):
    cuts = sorted(rng.randint(0, R) for _ in range(E))
    if rng.random() < 0.5:
        cuts = sorted(rng.choice(cuts) for _ in range(E))
    return [0] + cuts


@pytest.mark.parametrize("seed", range(60))
def test_every_pair_and_tile_once(seed):
    rng = random.Random(seed)
    E, R = rng.choice([1, 2, 8, 63, 64, 65, 200]), rng.choice([1, 2, 7, 64, 300, 1000])
    BM, tiles = rng.choice([4, 8, 16, 32, 256]), rng.choice([1, 3, 8, 20])
    offsets = counts_of(rng, E, R)
    seen = {}
    for u in units(offsets, R, E, BM, tiles):
        if u is None:
            continue
        e, first, held, tile = u
        assert 0 < held <= BM and 0 <= tile < tiles
        assert e == E and first >= offsets[E] or e < E and offsets[e] <= first and first + held <= offsets[e + 1]
        for i in range(first, first + held):
            seen[i, tile] = seen.get((i, tile), 0) + 1
    assert len(seen) == R * tiles and set(seen.values()) == {1}


@pytest.mark.parametrize("seed", range(60))
def test_any_offsets_stay_within_the_pairs(seed):
    rng = random.Random(seed)
    E, R = rng.choice([1, 3, 64, 65, 130]), rng.choice([1, 5, 64, 333])
    BM, tiles = rng.choice([4, 16, 64]), rng.choice([1, 5])
    offsets = [rng.choice([rng.randint(-2 ** 31, 2 ** 31 - 1), rng.randint(-5, R + 5), 0, R]) for _ in range(E + 1)]
    for u in units(offsets, R, E, BM, tiles):
        if u is not None:
            e, first, held, tile = u
            assert 0 <= e <= E and 0 <= tile < tiles, (offsets, u)
            assert 0 < held <= BM and 0 <= first and first + held <= R, (offsets, u)


def shares(chunks, tiles, cus):
    """What the blocks of the form for few rows take: runs of items (chunk, first tile, tiles), as the kernel cuts them."""
    items = chunks * tiles
    blocks = min(items, 3 * cus)
    assert items * (blocks + 1) < 2 ** 32
    for b in range(blocks):
        block = b % 8 * (blocks // 8) + min(b % 8, blocks % 8) + b // 8
        item, end = items * block // blocks, items * (block + 1) // blocks
        while item < end:
            chunk = item // tiles
            at = item - chunk * tiles
            n = min(tiles - at, end - item)
            yield chunk, at, n
            item += n


@pytest.mark.parametrize("seed", range(60))
def test_shares_cover_every_item_once(seed):
    rng = random.Random(seed)
    chunks, tiles, cus = rng.choice([1, 2, 7, 40, 300]), rng.choice([1, 3, 88, 896]), rng.choice([4, 80, 256])
    seen = set()
    for chunk, at, n in shares(chunks, tiles, cus):
        assert chunk < chunks and n > 0 and at + n <= tiles
        for i in range(at, at + n):
            assert (chunk, i) not in seen
            seen.add((chunk, i))
    assert len(seen) == chunks * tiles


def test_the_largest_share_bounds_fit():
    assert 2 ** 20 * (3 * 256 + 1) < 2 ** 32


@pytest.mark.parametrize("seed", range(40))
def test_waves_share_stages(seed):
    """The four waves' stages of a row: in order, all of them, and the scales of four stages at a time are there when first used."""
    rng = random.Random(seed)
    stages = rng.randint(1, 200)
    at = 0
    for wave in range(4):
        k0, k1 = stages * wave // 4, stages * (wave + 1) // 4
        assert k0 == at
        at = k1
        have = None
        for kb in range(k0, k1):
            if kb == k0 or kb % 4 == 0:
                have = kb & ~3
            assert have <= kb < have + 4
    assert at == stages


@pytest.mark.parametrize("seed", range(40))
def test_rows_without_an_expert_are_all_cleared(seed):
    rng = random.Random(seed)
    rest, cols, blocks = rng.choice([0, 1, 4, 300]), rng.choice([1, 255, 256, 257, 5000]), rng.choice([1, 7, 88, 768])
    pieces, seen = -(-cols // 256), set()
    for block in range(blocks):
        for i in range(rest * pieces * block // blocks, rest * pieces * (block + 1) // blocks):
            r, at = divmod(i, pieces)
            for thread in range(256):
                if at * 256 + thread < cols:
                    assert (r, at * 256 + thread) not in seen
                    seen.add((r, at * 256 + thread))
    assert len(seen) == rest * cols
