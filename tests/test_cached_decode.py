"""CPU check of how the cached attention divides a call (csrc/kv4_attention.cuh `span_of`, `request_of`,
`share_of`; the parts that kv4_attention_merge puts together): restated here line by line and swept over
lengths, windows, global tokens, groups and tile shapes.

* the tiles of an item hold every key that some row of it sees, each once (the band's whole tiles, then
  the globals in front of them);
* no item has more tiles than its request reckons for each of its items;
* the CTAs' shares cover the line of tiles once: whole items each by one CTA, cut items by consecutive
  CTAs whose parts the merge looks for in the places where they were put.
"""
import bisect
import random

import pytest


def span_of(rows, tile, group, window, glob, length, count, q_tile):
    """(first band tile, band tiles, gathered keys, gathered tiles) of one item."""
    n = count // group
    lo_pos = length - n + q_tile * rows // group
    hi_pos = length - n + (min(q_tile * rows + rows, count) - 1) // group
    if hi_pos < 0:
        return 0, 0, 0, 0
    lo = max(0, lo_pos - window)
    gathered = 0
    if glob:
        if lo > 0:
            at = bisect.bisect_left(glob, lo_pos)
            if at < len(glob) and glob[at] <= hi_pos:
                lo = 0
        lo &= ~(tile - 1)
        gathered = bisect.bisect_left(glob, lo)
    first = lo // tile
    return first, hi_pos // tile - first + 1, gathered, -(-gathered // tile)


def tiles_of(rows, tile, group, window, glob, length, count):
    """(query tiles, tiles reckoned for each item) of a request with `count` rows."""
    if count == 0:
        return 0, 0
    q_tiles = -(-count // rows)
    _, band, _, gathered = span_of(rows, tile, group, window, glob, length, count, q_tiles - 1)
    tiles = band + gathered
    if q_tiles > 1:
        tokens = (rows - 2) // group + 2
        band = min((window + tokens - 1) // tile + 2, length // tile + 1)
        at = bisect.bisect_left(glob, length - count // group)
        if at < len(glob) and glob[at] < length:
            band = length // tile + 1
        tiles = band + -(-bisect.bisect_left(glob, max(0, length - window)) // tile)
    return q_tiles, max(tiles, 1)


SHAPES = [(8, 32), (8, 64), (16, 32), (32, 32), (256, 64)]  # rows and keys of the kernels' tiles


@pytest.mark.parametrize("rows,tile", SHAPES)
def test_items_hold_the_keys_that_their_rows_see(rows, tile):
    rng = random.Random(rows + tile)
    for _ in range(60):
        group = rng.choice([1, 1, 2, 3, 4, 8, 20])
        length = rng.choice([0, 1, 31, 32, 33, 63, 64, 65, rng.randint(1, 900)])
        new = rng.choice([1, 1, 2, 5, rng.randint(1, 300), length or 1])  # at times more than the length
        window = rng.choice([0, 1, 31, 32, 64, 100, 10 ** 6])
        glob = sorted(rng.sample(range(1000), rng.choice([0, 0, 1, 3, 40])))
        count = new * group
        q_tiles, tiles = tiles_of(rows, tile, group, window, glob, length, count)
        for q_tile in range(q_tiles):
            first, band, gathered, extra = span_of(rows, tile, group, window, glob, length, count, q_tile)
            assert band + extra <= tiles
            held = list(range(first * tile, (first + band) * tile)) + glob[:gathered]
            assert len(held) == len(set(held)) and all(k < first * tile for k in glob[:gathered])
            held = set(held)
            for row in {q_tile * rows, min(q_tile * rows + rows, count) - 1, rng.randrange(q_tile * rows, min(q_tile * rows + rows, count))}:
                pos = length - new + row // group
                for key in range(max(0, pos + 1)):
                    if pos - key <= window or key in glob or pos in glob:
                        assert key in held, (length, new, window, glob, q_tile, pos, key)


@pytest.mark.parametrize("split", [False, True])
def test_shares_cover_the_line_once(split):
    rng = random.Random(split)
    for _ in range(120):
        rows, tile = rng.choice(SHAPES)
        group, heads, window = rng.choice([1, 2, 8]), rng.choice([1, 2, 5]), rng.choice([0, 100, 10 ** 6])
        requests = []
        for _ in range(rng.choice([1, 2, 7, 40])):
            length = rng.choice([0, 1, rng.randint(1, 3000)])
            q_tiles, tiles = tiles_of(rows, tile, group, window, [], length, rng.choice([0, 1, 1, 3, 200]) * group)
            requests.append((q_tiles * heads, tiles))
        line = sum(i * t for i, t in requests)
        ctas, least = rng.choice([1, 3, 148, 444]), 256 // tile
        per = -(-line // ctas)
        if split:
            per = max(per, least)
        item_of, start = [], 0  # every item's [begin, end) on the line
        for items, tiles in requests:
            for i in range(items):
                item_of.append((start + i * tiles, start + (i + 1) * tiles))
            start += items * tiles
        done, parts = {}, {}
        for c in range(ctas):
            at, end = c * per, min(c * per + per, line)
            begun = at
            while at < end:
                s, e = next(x for x in item_of if x[0] <= at < x[1])
                if not split and at > s:  # belongs to the CTA before
                    at = e
                    continue
                stop = min(e, end) if split else e
                if (at, stop) == (s, e):
                    assert s not in done
                    done[s] = c
                else:
                    slot = (c, int(at != begun))
                    assert slot not in parts
                    parts[slot] = (at, stop)
                at = stop
        for s, e in item_of:
            if s in done:
                continue
            c0, c1 = s // per, (e - 1) // per
            assert split and c1 > c0  # what the merge takes for granted
            found = [parts.pop((c, int(s > c * per) if c == c0 else 0)) for c in range(c0, c1 + 1)]
            assert found[0][0] == s and found[-1][1] == e and all(a[1] == b[0] for a, b in zip(found, found[1:]))
        assert not parts
