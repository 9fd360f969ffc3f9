"""How the work of a ragged batch is dealt to CTAs (csrc/paged.cuh), restated: every (sequence, head group, row tile, key tile) belongs to one
CTA's stretch of the line, a cut row tile's parts lie in the slots where the merge looks for them, and no slot is written twice."""
import random

import pytest


def row_span(n_q, kv, G, window, r):
    end = kv - n_q + r // G + 1
    if end <= 0:
        return 0, 0
    return (end - window if window and end > window else 0), end


def tile_range(n_q, kv, G, window, keys, r0, r1):
    lo, hi = row_span(n_q, kv, G, window, r0)[0], row_span(n_q, kv, G, window, r1)[1]
    return lo // keys, ((hi + keys - 1) // keys - lo // keys if hi > lo else 1)


def line(seqs, Hkv, G, window, rows, keys):
    """[(seq, head group, first row, first key tile, key tiles)] in the line's order."""
    out = []
    for s, (n_q, kv) in enumerate(seqs):
        R = n_q * G
        for h in range(Hkv):
            for r in range(0, R, rows):
                out.append((s, h, r, *tile_range(n_q, kv, G, window, keys, r, min(r + rows, R) - 1)))
    return out


def last_cta(e, ctas, total):
    return (e * ctas + total - 1) // total - 1


@pytest.mark.parametrize("seed", range(40))
def test_stretches_cover_the_line_and_parts_meet(seed):
    rng = random.Random(seed)
    rows, keys = rng.choice([(16, 128), (16, 64), (256, 128)])
    G, Hkv, window = rng.randint(1, 9), rng.randint(1, 4), rng.choice([0, 0, rng.randint(1, 400)])
    top = rng.choice([1, 6, 400])
    seqs = [(rng.randint(0, top), rng.choice([0, rng.randint(1, 3000)])) for _ in range(rng.randint(1, 12))]
    over = rng.randint(0, 3)      # places behind a row tile's key tiles that stand for its other work
    items = line(seqs, Hkv, G, window, rows, keys)
    total = sum(x[4] + over for x in items)
    grid = rng.choice([1, 5, 148])
    ctas = min(grid, total)
    starts = [c * total // ctas for c in range(ctas + 1)] if ctas else [0]
    slots, finished, noted = {}, [], {}
    begin_of, at = [], 0
    for x in items:
        begin_of.append(at)
        at += x[4] + over
    for c in range(ctas):
        t, cut = starts[c], 0
        i = max(j for j, b in enumerate(begin_of) if b <= t)
        while t < starts[c + 1]:
            n, rem = items[i][4], t - begin_of[i]
            step = min(n + over - rem, starts[c + 1] - t)
            a, b = min(rem, n), min(n, rem + step)
            t += step
            if b > a and a == 0 and b == n:
                finished.append(i)
            elif b > a:
                slot = 2 * c + (1 if a == 0 else 0)
                assert slot not in slots and slot < 2 * grid
                slots[slot] = (i, a, b)
                if a == 0:
                    cut += 1
                    noted[c] = (i, last_cta(begin_of[i] + n, ctas, total) - c + 1)
            i += 1
        assert cut <= 1
    for c, (i, parts) in noted.items():
        got = [slots.pop(2 * c + 1 if j == 0 else 2 * (c + j)) for j in range(parts)]
        assert all(x[0] == i for x in got)
        assert [x[1] for x in got] == [0] + [x[2] for x in got[:-1]] and got[-1][2] == items[i][4]
        finished.append(i)
    assert not slots and sorted(finished) == list(range(len(items)))


@pytest.mark.parametrize("seed", range(20))
def test_key_tiles_hold_what_the_rows_see(seed):
    rng = random.Random(100 + seed)
    n_q, kv, G, window, keys, rows = rng.randint(1, 300), rng.randint(0, 900), rng.randint(1, 8), rng.choice([0, rng.randint(1, 200)]), 128, 256
    R = n_q * G
    for r0 in range(0, R, rows):
        r1 = min(r0 + rows, R) - 1
        first, n = tile_range(n_q, kv, G, window, keys, r0, r1)
        assert n >= 1
        for r in range(r0, r1 + 1):
            lo, hi = row_span(n_q, kv, G, window, r)
            assert hi - lo <= (window or kv)
            if hi > lo:
                assert first * keys <= lo and hi <= (first + n) * keys
