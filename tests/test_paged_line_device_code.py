"""The arithmetic with which csrc/paged.cuh deals a batch to the CTAs, compiled for the host, against its restatement (test_paged_line.py), with the
tiles and allowances that the kernels have."""
import importlib
import os
import random
import subprocess

import pytest

from conftest import ROOT
from test_paged_line import last_cta, row_span, tile_range

build = importlib.import_module("ameva-compute_b200.build")
SOURCE = r"""
#include <cstdio>
#include "paged.cuh"
using namespace amv::paged;
// a request per line of stdin, an answer per line of stdout
int main() {
    char what;
    uint64_t v[10];
    while (scanf(" %c", &what) == 1) {
        for (uint64_t& x : v)
            if (scanf("%lu", &x) != 1) return 1;
        Args pc = {};
        if (what == 'q') {          // row, G
            set_group(pc, v[1]);
            printf("%u\n", query_of(pc, v[0]));
        } else if (what == 's') {   // total, CTA, grid
            const Stretch x = stretch_of(v[0], v[1], v[2]);
            printf("%u %u %u\n", x.begin, x.end, x.ctas);
        } else if (what == 'l') {   // end of a piece, total, CTAs
            Stretch x = {};
            x.total = v[1];
            x.ctas = v[2];
            printf("%u\n", last_cta(x, v[0]));
        } else {                    // 't': queries, keys, G, window, log2 of a tile's keys, rows r0 .. r1, whether a shared prefix
            set_group(pc, v[2]);
            pc.window = v[3];
            pc.keys_log2 = v[4];
            const int32_t one = 0;
            pc.prefix = v[7] ? &one : nullptr;
            const Seq q = {0u, (uint32_t)v[0], (uint32_t)v[1], nullptr};
            uint32_t first, count;
            tile_range(pc, q, v[5], v[6], first, count);
            const Span a = row_span(pc, q, v[5]), b = row_span(pc, q, v[6]);
            printf("%u %u %u %u %u %u\n", first, count, a.lo, a.hi, b.lo, b.hi);
        }
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    at = tmp_path_factory.mktemp("line")
    (at / "line.cu").write_text(SOURCE)
    flags = [f for f in build.NVCC_FLAGS if f != "-O3"]
    subprocess.run([build._nvcc(), *flags, "-I", os.path.join(ROOT, "ameva-compute_b200", "csrc"), "-o", str(at / "line"), str(at / "line.cu")],
                   check=True, capture_output=True)

    def run(requests):
        text = "".join(" ".join(map(str, r + (0,) * (11 - len(r)))) + "\n" for r in requests)
        out = subprocess.run([str(at / "line")], input=text, check=True, capture_output=True, text=True).stdout.splitlines()
        return [tuple(int(x) for x in line.split()) for line in out]

    return run


def test_queries_of_rows(ask):
    rng = random.Random(1)
    cases = [(r, G) for G in (1, 2, 3, 5, 7, 8, 11, 64, 127, 4097, 65535) for r in (0, 1, G - 1, G, G + 1, 2**31 - 1, 2**31 - G, rng.randrange(2**31))]
    assert ask([("q", *c) for c in cases]) == [(r // G,) for r, G in cases]


@pytest.mark.parametrize("seed", range(20))
def test_stretches(ask, seed):
    """Equal stretches without gaps, also of lines near 2^32; the last CTA of a piece is the one whose stretch holds its last tile."""
    rng = random.Random(seed)
    total, grid = rng.choice([rng.randint(1, 300), rng.randint(1, 10**6), rng.randint(2**31, 2**32 - 1), 2**32 - 1]), rng.choice([1, 2, 147, 148, 160])
    ctas = min(total, grid)
    got = ask([("s", total, c, grid) for c in range(grid)])
    assert got[:ctas] == [(c * total // ctas, (c + 1) * total // ctas, ctas) for c in range(ctas)] and all(x[:2] == (0, 0) for x in got[ctas:])
    ends = [rng.randint(1, total) for _ in range(50)] + [1, total] + [x[1] for x in got[:ctas]]
    for e, (c,) in zip(ends, ask([("l", e, total, ctas) for e in ends])):
        assert c == last_cta(e, ctas, total) and got[c][0] < e <= got[c][1], (e, total)


@pytest.mark.parametrize("rows,keys,over", [(16, 32, 2), (16, 64, 2), (16, 128, 2), (16, 256, 2), (128, 64, 6), (256, 64, 6)])
@pytest.mark.parametrize("seed", range(5))
def test_tiles(ask, rows, keys, over, seed):
    """Every row tile's key tiles as restated; what a whole line adds up to, and the parts of its cut tiles, come out of the real stretches."""
    rng = random.Random(seed)
    G, window, top = rng.choice([1, 2, 3, 4, 7, 16]), rng.choice([0, 0, rng.randint(1, 3000)]), rng.choice([1, 6, 900])
    seqs = [(rng.randint(0, top), rng.choice([0, 1, rng.randint(1, 9000)])) for _ in range(12)]
    log2 = keys.bit_length() - 1
    asked, want = [], []
    for n, kv in seqs:
        R = n * G
        for r in range(0, R, rows):
            r1 = min(r + rows, R) - 1
            asked.append(("t", n, kv, G, window, log2, r, r1, 0))
            want.append((*tile_range(n, kv, G, window, keys, r, r1), *row_span(n, kv, G, window, r), *row_span(n, kv, G, window, r1)))
            asked.append(("t", n, kv, G, 0, log2, r, r1, 1))      # of a shared prefix every row sees all
            want.append((0, max(1, (kv + keys - 1) // keys), 0, kv, 0, kv))
    got = ask(asked)
    assert got == want
    items = [x[1] for x in got[::2]]
    total = sum(x + over for x in items)
    if not total:
        return
    ctas = min(148, total)
    cuts = [x[0] for x in ask([("s", total, c, 148) for c in range(ctas)])] + [total]
    at, covered = 0, 0
    for n in items:
        begin, end = at, at + n
        inside = [c for c in range(ctas) if cuts[c] < end and cuts[c + 1] > begin]
        (last,), = ask([("l", end, total, ctas)])
        assert inside[-1] == last and inside == list(range(inside[0], last + 1))
        covered += sum(min(end, cuts[c + 1]) - max(begin, cuts[c]) for c in inside)
        at = end + over
    assert covered == sum(items)
