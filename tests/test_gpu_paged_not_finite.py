"""NaN and infinities in the pages of a paged KV cache, against the definition in 64 bits: a column is NaN or infinite where the row sees such
a value in it, and what it would be without them where it does not. Tolerances of finite columns: tests/test_gpu_paged.py."""
import numpy as np
import pytest

from conftest import load_pkg
from test_gpu_paged import TOL16, TOL32, Setup, ctx  # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu
rt, paged = load_pkg().runtime, load_pkg().paged


def upload(s):
    s.cache.k.write(s.in_memory(s.k))
    s.cache.v.write(s.in_memory(s.v))
    s.qb.write(s.q)


def place(s, seq, key):
    return s.table[seq, key // s.page], key % s.page


def check(s, **kw):
    with np.errstate(all="ignore"):
        want = s.want(**kw)
    rows = sorted(want)
    y = np.stack([want[r] for r in rows])
    for f16 in (False, True):
        got = s.attend(f16=f16, **kw)[rows].astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(y)), f16
        inf = np.isinf(y)
        assert np.array_equal(got[inf], y[inf]) and np.array_equal(np.isinf(got), inf), f16
        fine = np.isfinite(y)
        assert np.max(np.abs(got[fine] - y[fine]), initial=0.0) <= (TOL16 if f16 else TOL32), f16
    return y


SHAPES = [(128, 8, 2, 16, "token"), (64, 14, 2, 32, "head"), (256, 4, 2, 64, "token"), (128, 5, 5, 16, "head")]
BATCHES = [([40, 300, 1, 90], [900, 333, 700, 91]), ([1, 4, 2, 6], [900, 33, 17, 300]), ([200], [2600])]


@pytest.mark.parametrize("D,H,Hkv,page,layout", SHAPES)
@pytest.mark.parametrize("q,kv", BATCHES)
@pytest.mark.parametrize("window", [0, 75])
@pytest.mark.parametrize("what", ["first", "last", "both", "row", "some", "many"])
def test_values(ctx, D, H, Hkv, page, layout, q, kv, window, what):  # noqa: F811
    s = Setup(ctx, q, kv, H, Hkv, D, page, layout, seed=D + sum(q) + window, pad=2, garbage=True)
    rng = np.random.default_rng(window + len(what))
    odd = np.array([np.nan, np.inf, -np.inf], np.float16)
    for i, n in enumerate(kv):
        if what == "first":       # every row sees it
            s.v[place(s, i, 0)][:, 3] = np.inf
        elif what == "last":      # the last row alone
            s.v[place(s, i, n - 1)][0, 5] = -np.inf
            s.v[place(s, i, max(0, n - 2))][-1, 5] = np.nan
        elif what == "both":      # infinities of both signs meet in a NaN
            s.v[place(s, i, n // 3)][:, 7], s.v[place(s, i, n // 2)][:, 7] = np.inf, -np.inf
        elif what == "row":       # a key's whole row
            s.v[place(s, i, n // 2)] = np.nan
        elif what == "some":
            for key in rng.integers(0, n, 3):
                s.v[place(s, i, key)][rng.integers(Hkv), rng.integers(D)] = rng.choice(odd)
        else:
            for key in rng.integers(0, n, n // 10 + 1):
                s.v[place(s, i, key)][:, rng.integers(D // 4)] = rng.choice(odd)
    upload(s)
    y = check(s, window=window)
    assert window or what == "some" or not np.isfinite(y).all()      # (under a window no row may see the keys)
    s.close()


@pytest.mark.parametrize("D,H,Hkv,page,layout", SHAPES)
@pytest.mark.parametrize("q,kv", BATCHES)
def test_values_beside_keys_and_queries(ctx, D, H, Hkv, page, layout, q, kv):  # noqa: F811
    """Scores that are not finite make a row NaN, whatever the values are that it sees."""
    s = Setup(ctx, q, kv, H, Hkv, D, page, layout, seed=1, pad=2, garbage=True)
    for i, n in enumerate(kv):
        s.v[place(s, i, n // 4)] = np.inf
        s.k[place(s, i, n // 2)][0, 9] = np.nan
        s.k[place(s, i, n - 1)][-1, 11] = np.inf
    s.q[0, 0, 1], s.q[s.rows - 1, H - 1, 2] = np.nan, np.inf
    upload(s)
    check(s)
    s.close()


@pytest.mark.parametrize("D,H,Hkv,page,layout", SHAPES)
@pytest.mark.parametrize("q,prefix", [([1, 2, 1], 300), ([1] * 60, 900), ([30, 2, 40], 77)])
@pytest.mark.parametrize("softcap", [0.0, 4.0])
def test_prefix(ctx, D, H, Hkv, page, layout, q, prefix, softcap):  # noqa: F811
    kv = [n + 20 for n in q]
    s = Setup(ctx, q, kv, H, Hkv, D, page, layout, seed=prefix, pad=2, garbage=True, prefix=prefix)
    s.v[s.prefix[1], 5, 0, 3] = np.inf
    s.v[s.prefix[1 + (prefix - 1) // page], (prefix - 1) % page, -1, 4] = np.nan
    s.v[place(s, 0, 2)][0, 3] = -np.inf       # meets the prefix's: NaN
    s.v[place(s, 1, 1)][:, 6] = np.inf
    s.v[place(s, len(q) - 1, kv[-1] - 1)][:, 8] = -np.inf
    upload(s)
    check(s, softcap=softcap)
    s.close()


@pytest.mark.parametrize("q,kv,D", [([300, 40], [700, 900], 128), ([200, 70], [2000, 300], 64), ([1] * 6, [900] * 6, 128), ([2] * 3, [600] * 3, 256)])
def test_one_cta_takes_all(ctx, q, kv, D):  # noqa: F811
    """Many pieces for the second pass of one CTA, none of them cut."""
    s = Setup(ctx, q, kv, 8, 2, D, seed=D, pad=1, garbage=True)
    for i, n in enumerate(kv):
        s.v[place(s, i, 0)][0, 3], s.v[place(s, i, n - 2)][1, 70 % D] = np.nan, np.inf
    upload(s)
    want = s.want()
    for f16 in (False, True):
        got = s.attend(f16=f16, scratch=256)
        for r, y in want.items():
            assert np.array_equal(np.isnan(got[r]), np.isnan(y)) and np.array_equal(np.isinf(got[r]), np.isinf(y))
            fine = np.isfinite(y)
            assert np.max(np.abs(got[r][fine] - y[fine])) <= (TOL16 if f16 else TOL32)
    s.close()


def test_a_weight_below_32_bits_is_one(ctx):  # noqa: F811
    """exp(-200) of an infinity is infinite, in whatever kernel."""
    for q, D in ((1, 128), (100, 128), (100, 64), (2, 256)):
        kv = q + 30
        s = Setup(ctx, [q], [kv], 2, 1, D, seed=2)
        s.q[:], s.k[:] = 1.0, 0.0
        s.k[place(s, 0, 3)][:] = 200.0 / D ** 0.5      # a score of 200 beside others of 0
        s.v[place(s, 0, 7)][0, 3] = np.inf
        upload(s)
        assert np.isposinf(check(s)[:, :, 3]).all()
        s.close()


@pytest.mark.parametrize("q,D,H,Hkv,prefix", [(1, 128, 2, 1, 0), (1, 64, 8, 8, 0), (100, 128, 2, 1, 0), (100, 64, 4, 2, 0), (2, 256, 2, 1, 0), (1, 128, 4, 2, 500),
                                              (40, 64, 4, 1, 500)])
@pytest.mark.parametrize("scratch", [None, 1])
def test_parts_whose_weight_is_below_32_bits(ctx, q, D, H, Hkv, prefix, scratch):  # noqa: F811
    """The same where the infinity and the score of 200 are seen by different warps, CTAs or launches, whose results are joined: it does not
    depend on where the keys are cut."""
    kv = 3000
    s = Setup(ctx, [q], [kv], H, Hkv, D, seed=3, prefix=prefix)
    s.q[:], s.k[:] = 1.0, 0.0
    s.k[place(s, 0, 2500)][:] = 200.0 / D ** 0.5
    s.v[place(s, 0, 7)][:, 3], s.v[place(s, 0, 1200)][:, 4], s.v[place(s, 0, 1900)][:, 5] = np.inf, -np.inf, np.nan
    if prefix:
        s.v[s.prefix[1], 9, :, 6] = np.inf
    upload(s)
    want, own = s.want(), s.held * H * (D + 4) * 4 + 256 if prefix else 0
    y = np.stack([want[r] for r in range(q)])
    assert np.isposinf(y[:, :, 3]).all() and np.isneginf(y[:, :, 4]).all() and np.isnan(y[:, :, 5]).all()
    for f16 in (False, True):
        got = s.attend(f16=f16, scratch=scratch and own + 256)[:q]
        assert np.array_equal(np.isnan(got), np.isnan(y)) and np.array_equal(np.isposinf(got), np.isposinf(y)) and np.array_equal(np.isneginf(got), np.isneginf(y))
        fine = np.isfinite(y)
        assert np.max(np.abs(got[fine] - y[fine])) <= (TOL16 if f16 else TOL32)
    s.close()


@pytest.mark.parametrize("q,kv,H,Hkv,D", [(2048, 2048, 8, 2, 128), (2048, 2048, 8, 2, 64), (1, 60000, 8, 2, 128), (1, 30000, 4, 1, 256)])
def test_a_sequence_that_is_not_finite_does_not_stall_its_batch(ctx, q, kv, H, Hkv, D):  # noqa: F811
    """One infinity that all rows see: the call takes some times as long as without, not hundreds of times (a row at a time, every key's
    score again: 380 times for the first of these)."""
    import torch
    s = Setup(ctx, [q], [kv], H, Hkv, D, 64)
    dst = s.own(size=q * H * D * 2)
    batch = ctx.batch(4)
    paged.record_attention(batch, s.cache, s.seqs, s.qb, dst, s.own(size=paged.scratch_bytes(ctx, s.seqs, heads=H, head_dim=D)), s.status, heads=H,
                           scale=D ** -0.5, f16_out=True)
    batch.instantiate()
    stream, times = torch.cuda.ExternalStream(ctx.stream), []
    for odd in (False, True):
        if odd:
            s.v[place(s, 0, 0)][:, 3] = np.inf
            s.cache.v.write(s.in_memory(s.v))
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record(stream)
            ev = batch.replay()
            b.record(stream)
            ev.wait()
            ev.destroy()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[1] <= 40 * times[0], times
    batch.destroy()
    s.close()


def test_a_prefix_that_is_not_finite_behind_sequences_that_are_not(ctx):  # noqa: F811
    """Columns whose only such values are among a row's own keys, others of the prefix, others of both: in every row of the batch."""
    for D, f in ((128, 300), (64, 900), (256, 100)):
        q = [1, 3, 40]
        s = Setup(ctx, q, [n + 30 for n in q], 8, 2, D, 16, "token", seed=D, pad=1, garbage=True, prefix=f)
        s.v[s.prefix[1], 2, :, 3], s.v[s.prefix[1], 3, :, 4], s.v[s.prefix[2], 5, :, 9] = np.inf, np.nan, np.inf
        for i in range(3):
            s.v[place(s, i, 0)][:, 5], s.v[place(s, i, 1)][:, 6] = np.inf, np.nan
            s.v[place(s, i, 4)][:, 9], s.v[place(s, i, 2)][:, 3] = -np.inf, np.inf
        upload(s)
        y = check(s)
        assert np.isposinf(y[:, :, 3]).all() and np.isposinf(y[:, :, 5]).all() and all(np.isnan(y[:, :, c]).all() for c in (4, 6, 9))
        s.close()
