"""How exact f16 results of the attention over a paged KV cache are: as near to the 64-bit result as its rounding leaves, whichever kernel forms them,
however long the context is, and however few CTAs share it."""
import numpy as np
import pytest

from conftest import load_pkg
from test_gpu_paged import Setup, ctx  # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu
rt, paged = load_pkg().runtime, load_pkg().paged


@pytest.mark.parametrize("D,H,Hkv,q,prefix", [(128, 8, 2, 40, 0), (64, 8, 2, 40, 0), (128, 8, 2, 1, 0), (256, 8, 2, 40, 0), (128, 8, 2, 1, 900), (64, 4, 1, 30, 900)])
@pytest.mark.parametrize("scratch", [None, 1])
def test_results_of_16_bits_are_rounded_once(ctx, D, H, Hkv, q, prefix, scratch):  # noqa: F811
    """Before its rounding, a result of 1000 keys is off by a relative 126 * 2^-24 = 7.5e-6 at most on the average (63 instructions of 16 keys
    and as many of the remainders add to its sum, each cut by less than 2^-23 of what it has grown to, half of its end). A step of f16 is 2^-10
    of a value at most, and 2^-11 at least: 7.5e-6 / 2^-11 = 1.5 % of the results are rounded to the neighbour, one step away: 2-norm sqrt(0.015) *
    2^-10 = 1.2e-4 of the result. Weights of 11 bits without their remainders leave 2.6e-4."""
    n = 1 if q > 1 else 70
    kv = 1000 if not prefix else 60
    s = Setup(ctx, [q] * n, [kv] * n, H, Hkv, D, seed=D + q, prefix=prefix)
    want = s.want()
    y = np.stack([want[r] for r in range(s.rows)])
    own = s.held * H * (D + 4) * 4 + 256 if prefix else 0
    got = s.attend(f16=True, scratch=scratch and own + 256)[:s.rows].astype(np.float64)
    assert np.linalg.norm(got - y.astype(np.float16).astype(np.float64)) <= 1.2e-4 * np.linalg.norm(y)
    s.close()


@pytest.mark.parametrize("D,page", [(128, 64), (64, 256)])
@pytest.mark.parametrize("q,kv,window", [(64, 131072, 0), (33, 70001, 0), (40, 131072, 90001)])
@pytest.mark.parametrize("scratch", [None, 600000, 4096])
def test_long_sums_of_16_bits(ctx, D, page, q, kv, window, scratch):  # noqa: F811
    """A rounding to f16 is off by 2^-11 / sqrt(3) = 2.82e-4 on the average at most. The sum in front of it is added up at least every 128 key
    tiles, 1024 instructions, each cut by less than 2^-23 of what it has grown to, half of its end on the average: 1024 * 2^-24 = 6.1e-5 for
    values of one sign. Left in its accumulator, 131072 keys would be off by another 6e-4 (16384 instructions)."""
    s = Setup(ctx, [q], [kv], 4, 1, D, page, "head", seed=D)
    s.v[:] = np.abs(s.v)
    s.cache.v.write(s.in_memory(s.v))
    want = s.want(window=window)
    y = np.stack([want[r] for r in range(q)])
    for f16 in (True, False):
        got = s.attend(f16=f16, window=window, scratch=scratch)[:q].astype(np.float64)
        assert np.linalg.norm(got - y) <= (2.82e-4 + 6.1e-5 if f16 else 2.6e-6) * np.linalg.norm(y)
    s.close()


@pytest.mark.parametrize("scratch", [None, 600000, 4096])
def test_long_sums_that_grow_or_are_not_there(ctx, scratch):  # noqa: F811
    """The accumulator begins anew where the maximum has grown since, where nothing has been seen yet, and where no page of the tiles behind is
    there; a NaN in what it has handed over is found."""
    D, kv, q = 128, 40000, 40
    s = Setup(ctx, [q], [kv], 4, 1, D, 64, seed=9)
    s.q[:] = np.abs(s.q)
    flat = np.abs(s.k[s.table[0]]).reshape(-1, 1, D)
    flat *= np.linspace(0.0, 2.0, flat.shape[0])[:, None, None].astype(np.float16)      # scores up to 20
    s.k[s.table[0]] = flat.reshape(-1, 64, 1, D)
    s.cache.k.write(s.in_memory(s.k))
    s.qb.write(s.q)
    want = s.want()
    got = s.attend(f16=True, scratch=scratch)
    # (a score of 20 is off by 16 * 2^-23 * 20 at most, a result by twice that of the largest value, and by its rounding)
    tol = 2 * 16 * 2.0 ** -23 * 20 * 5.5 + 2.0 ** -11 * 5.5
    assert max(np.max(np.abs(want[j] - got[j])) for j in want) <= tol
    s.v[s.table[0, 3], 5, 0, 7] = np.nan
    s.cache.v.write(s.in_memory(s.v))
    got = s.attend(f16=True, scratch=scratch)
    assert np.isnan(got[:q, :, 7]).all() and np.isfinite(np.delete(got[:q], 7, axis=2)).all()
    assert max(np.max(np.abs(np.delete(want[j] - got[j], 7, axis=1))) for j in want) <= tol
    s.v[s.table[0, 3], 5, 0, 7] = 1.0
    s.cache.v.write(s.in_memory(s.v))
    from oracle import paged as ref
    for gone in (range(0, 300), range(256, 600), range(100, 625)):      # pages of 64: in front, behind the second time, to the end
        bad = s.table.copy()
        bad[0, list(gone)] = -1
        s.seqs.table.write(bad)
        got = s.attend(f16=True, scratch=scratch)
        keep = [p for i, p in enumerate(s.table[0]) if i not in gone]
        for j in (0, q - 1):
            seen = sum(max(0, min(64, kv - q + j + 1 - 64 * i)) for i in range(len(s.table[0])) if i not in gone)
            w = ref.attention(s.q[j:j + 1], s.k, s.v, [keep], [0, 1], [seen], D ** -0.5)[0]
            assert np.max(np.abs(w - got[j])) <= tol, (gone, j)
    s.close()
