"""ameva_paged_append, ameva_paged_attn and ameva_paged_prefix_attn against the definition in 64 bits (oracle/paged.py).

Tolerances. Rows, keys and values are standard normal and D <= 256, so scores scale * q . k with scale = D^-0.5 are of order one.
An f32 result: a score is a sum of D products in f32 on the matrix instructions, whose absolute error is below 16 * 2^-23 * scale * sum
|q k| < 16 * 2^-23 * D^-0.5 * 0.8 D < 2.5e-5 for D = 256; the exponential adds 2^-22 relative, P as two halves 2^-22. A result is a weighted
mean of values, so it moves by at most twice the relative error of a weight times the largest |v| (5.5): 3e-4 at most (TOL32), and by far
less on the average: the errors of the keys are independent, 2-norm below 1e-5 (NORM32). An f16 result adds the rounding of P (2^-11 of the
mean's terms at most) and of the result (2^-11 of it): 2 * 2^-11 * 5.5 = 5.4e-3 (TOL16), both of random sign: 2-norm below 2^-11 (NORM16).
The rotation: two products and a sum in f32 of elements below 6, cosines to 2^-22: below 6 * 3 * 2^-22, then half a step of f16."""
import numpy as np
import pytest

from conftest import load_pkg
from oracle import paged as ref

pytestmark = pytest.mark.gpu
pkg = load_pkg()
rt, paged = pkg.runtime, pkg.paged
TOL32, NORM32, TOL16, NORM16 = 3e-4, 1e-5, 5.4e-3, 2.0 ** -11


@pytest.fixture(scope="module")
def ctx():
    c = rt.init()
    yield c
    c.destroy()


class Setup:
    """A pool of pages in random order, the sequences' tables, everything on the device."""

    def __init__(self, ctx, q_lens, kv_lens, H, Hkv, D, page=16, layout="token", seed=0, spare=2, pad=0, garbage=False, prefix=0, stride=None, max_q=None, max_kv=None):
        rng = np.random.default_rng(seed)
        self.ctx, self.H, self.Hkv, self.D, self.layout, self.page = ctx, H, Hkv, D, layout, page
        self.kv_len = np.array(kv_lens, np.int32)
        self.q_start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.rows = int(self.q_start[-1])
        self.held = max(1, self.rows + pad)
        need = [(n + page - 1) // page for n in kv_lens]
        n_prefix = (prefix + page - 1) // page
        self.n_pages = sum(need) + n_prefix + spare
        pages = rng.permutation(self.n_pages)
        self.stride = stride or max(1, max(need))
        self.table = np.full((len(kv_lens), self.stride), -7, np.int32)      # behind the last page: nothing
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = pages[at:at + n]
            at += n
        self.prefix = np.concatenate([[prefix], pages[at:at + n_prefix]]).astype(np.int32) if prefix else None
        self.k, self.v = (rng.standard_normal((self.n_pages, page, Hkv, D)).astype(np.float16) for _ in range(2))
        if garbage:      # whatever no sequence has written
            used = np.zeros((self.n_pages, page), bool)
            for s, n in enumerate(kv_lens):
                for i in range(n):
                    used[self.table[s, i // page], i % page] = True
            for i in range(prefix):
                used[self.prefix[1 + i // page], i % page] = True
            self.k[~used], self.v[~used] = np.nan, np.inf
            self.v[~used, :, ::2] = np.nan
        self.q = rng.standard_normal((self.held, H, D)).astype(np.float16)
        self.max_q, self.max_kv = max_q or max(1, max(q_lens)), max_kv or max(1, max(kv_lens))
        self.buffers = []
        self.upload()

    def own(self, data=None, size=0):
        self.buffers.append(self.ctx.buffer(size, data=data))
        return self.buffers[-1]

    def in_memory(self, cache):
        return np.ascontiguousarray(cache if self.layout == "token" else cache.transpose(0, 2, 1, 3))

    def from_memory(self, raw):
        if self.layout == "token":
            return raw.reshape(self.n_pages, self.page, self.Hkv, self.D)
        return raw.reshape(self.n_pages, self.Hkv, self.page, self.D).transpose(0, 2, 1, 3)

    def upload(self):
        self.cache = paged.Cache(self.own(self.in_memory(self.k)), self.own(self.in_memory(self.v)), self.n_pages, self.page, self.Hkv, self.D, self.layout)
        self.seqs = paged.Sequences(self.own(self.table), self.own(self.q_start), self.own(self.kv_len), n_seqs=len(self.kv_len),
                                    table_stride=self.stride, rows=self.held, max_q=self.max_q, max_kv=self.max_kv)
        self.status = self.own(np.array([0, 0xFFFFFFFF], np.uint32))
        self.qb = self.own(self.q)

    def attend(self, f16=False, scratch=None, softcap=0.0, window=0, scale=None, node=3, wider=0):
        """wider: elements between the rows of q and of the result beside their own."""
        dt = np.float16 if f16 else np.float32
        width = self.H * self.D + wider
        dst, qb = self.own(np.full((self.held, width), 77.0, dt)), self.qb
        if wider:
            qb = self.own(np.concatenate([self.q.reshape(self.held, -1), np.full((self.held, wider), np.nan, np.float16)], axis=1))
        prefix = self.prefix is not None
        need = paged.scratch_bytes(self.ctx, self.seqs, heads=self.H, head_dim=self.D, prefix=prefix)
        sb = self.own(np.full((scratch or need) // 4, np.nan, np.float32))      # (its contents do not matter)
        batch = self.ctx.batch(4)
        kw = dict(heads=self.H, scale=self.D ** -0.5 if scale is None else scale, softcap=softcap, f16_out=f16, node=node, q_stride=width, dst_stride=width)
        try:
            if prefix:
                paged.record_prefix_attention(batch, self.cache, self.seqs, qb, dst, sb, self.status, prefix=self.own(self.prefix),
                                              max_prefix=int(self.prefix[0]), **kw)
            else:
                paged.record_attention(batch, self.cache, self.seqs, qb, dst, sb, self.status, window=window, **kw)
            ev = batch.submit()
            ev.wait()
            ev.destroy()
        finally:
            batch.destroy()
        got = dst.read(dt).reshape(self.held, width)
        assert np.all(got[:, self.H * self.D:] == 77.0)
        return got[:, :self.H * self.D].reshape(self.held, self.H, self.D)

    def want(self, **kw):
        kw.setdefault("scale", self.D ** -0.5)
        prefix = None if self.prefix is None else (self.prefix[1:], int(self.prefix[0]))
        return ref.attention(self.q, self.k, self.v, self.table, self.q_start, self.kv_len, prefix=prefix, **kw)

    def check(self, got, want, f16):
        rows = sorted(want)
        y = np.stack([want[r] for r in rows]) if rows else np.zeros((0, self.H, self.D))
        x = got[rows].astype(np.float64)
        assert np.all(np.isfinite(x))
        assert np.max(np.abs(x - y), initial=0.0) <= (TOL16 if f16 else TOL32)
        norm = np.linalg.norm(y)
        assert np.linalg.norm(x - y) <= (NORM16 if f16 else NORM32) * norm
        others = np.ones(self.held, bool)
        others[rows] = False
        assert np.all(got[others] == 77.0)      # rows behind the last sequence

    def refused(self):
        return [int(x) for x in self.status.read(np.uint32)]

    def close(self):
        for b in self.buffers:
            b.destroy()


def both(s, **kw):
    want = s.want(**{name: x for name, x in kw.items() if name != "wider"})
    for f16 in (False, True):
        s.check(s.attend(f16=f16, **kw), want, f16)
    assert s.refused() == [0, 0xFFFFFFFF]
    s.close()


@pytest.mark.parametrize("D,H,Hkv,page,layout", [(128, 8, 2, 16, "token"), (64, 7, 1, 32, "head"), (128, 5, 5, 64, "head"), (256, 4, 2, 16, "token"),
                                                 (64, 32, 2, 128, "token"), (128, 33, 3, 256, "head")])
def test_single_tokens(ctx, D, H, Hkv, page, layout):
    """Lengths around every border of pages, 16-key blocks and key tiles; groups of 1, 2, 4, 7, 11, 16 heads."""
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000, 0, 257]
    both(Setup(ctx, [1] * len(kv), kv, H, Hkv, D, page, layout, seed=D + H, pad=3, garbage=True))


@pytest.mark.parametrize("D,H,Hkv,page,layout", [(128, 8, 2, 16, "token"), (64, 14, 2, 32, "head"), (256, 4, 2, 64, "token")])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (40, 0.0), (1, 0.0), (0, 5.0)])
def test_drafted_tokens(ctx, D, H, Hkv, page, layout, window, softcap):
    """A few rows per sequence, sequences without rows and with more rows than keys."""
    q, kv = [3, 0, 5, 2, 1, 4, 6, 0, 2], [3, 10, 50, 129, 17, 2, 300, 0, 0]
    both(Setup(ctx, q, kv, H, Hkv, D, page, layout, seed=window + 1, pad=1, garbage=True), window=window, softcap=softcap)


@pytest.mark.parametrize("D,H,Hkv,page,layout", [(128, 8, 2, 16, "token"), (64, 14, 2, 64, "head"), (128, 3, 3, 256, "token"), (64, 8, 8, 16, "head"),
                                                 (256, 2, 1, 32, "token")])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (100, 0.0), (0, 8.0)])
def test_prompts(ctx, D, H, Hkv, page, layout, window, softcap):
    """Row tiles of the tensor-core kernel (more than 64 rows per KV head) beside sequences of few rows; ragged everything."""
    q, kv = [70, 1, 130, 33, 300, 0, 90], [70, 200, 140, 500, 333, 5, 50]
    both(Setup(ctx, q, kv, H, Hkv, D, page, layout, seed=7 + window, pad=2, garbage=True), window=window, softcap=softcap)


@pytest.mark.parametrize("D,H,Hkv,page,layout,q,prefix", [
    (128, 8, 2, 16, "token", [1, 1, 1], 100), (128, 8, 2, 16, "token", [1] * 40, 1000), (64, 14, 2, 32, "head", [2, 0, 3, 1, 5], 257),
    (128, 4, 4, 64, "head", [1] * 70 + [9], 130), (256, 4, 1, 16, "token", [1, 2, 3, 4], 333), (64, 8, 1, 128, "token", [50, 1, 40], 1)])
def test_shared_prefix(ctx, D, H, Hkv, page, layout, q, prefix):
    rng = np.random.default_rng(prefix)
    kv = [n + int(rng.integers(0, 70)) for n in q]
    kv[0] = q[0]
    both(Setup(ctx, q, kv, H, Hkv, D, page, layout, seed=prefix, pad=2, garbage=True, prefix=prefix))


@pytest.mark.parametrize("D,H,Hkv", [(128, 40, 2), (64, 128, 1), (128, 65, 1), (64, 200, 1), (128, 18, 9), (64, 17, 17), (256, 12, 6), (256, 96, 1)])
def test_groups_of_all_sizes(ctx, D, H, Hkv):
    """Many query heads per KV head (more than 64: single tokens in the tensor-core kernel), KV heads that are no multiple of the warps."""
    both(Setup(ctx, [1, 3, 1, 0, 40], [70, 300, 1, 9, 41], H, Hkv, D, 16, "token", seed=H, pad=1, garbage=True))


@pytest.mark.parametrize("q,kv,page", [([1] * 500, [17] * 500, 16), ([1, 0, 2] * 1365, [5, 3, 2] * 1365, 16), ([70, 1, 90, 3] * 20, [75, 30, 90, 3] * 20, 32),
                                       ([1, 2000, 5], [4000, 2500, 1025], 1024), ([1] * 3, [1023, 1024, 1025], 1024)])
@pytest.mark.parametrize("prefix", [0, 77])
def test_many_sequences_and_large_pages(ctx, q, kv, page, prefix):
    """Up to the most sequences of a batch; prompts of many; pages of 1024 tokens."""
    H = 2 if max(q) < 1000 else 1
    both(Setup(ctx, q, kv, H, 1, 64, page, "head", seed=len(q), pad=1, prefix=prefix))


@pytest.mark.parametrize("q,kv", [([1, 3, 5], [100, 40, 300]), ([90, 1, 200], [100, 40, 300])])
@pytest.mark.parametrize("kw", [dict(scale=0.0), dict(scale=-0.1), dict(scale=-0.1, softcap=3.0), dict(wider=8), dict(wider=520, window=33)])
def test_scales_and_strides(ctx, q, kv, kw):
    both(Setup(ctx, q, kv, 8, 2, 128, 16, "token", seed=11, pad=2, garbage=True), **kw)
    if "window" not in kw:
        both(Setup(ctx, q, kv, 6, 2, 64, 16, "token", seed=12, pad=2, garbage=True, prefix=150), **kw)


def test_announced_maxima_may_be_larger(ctx):
    """Launches are sized by the announcement: the same results where it is wide of the mark, and none where nothing is to be done."""
    both(Setup(ctx, [1, 1], [100, 40], 8, 2, 128, pad=200, max_q=150, max_kv=5000, stride=320))
    # 33 .. 64 rows: the tensor-core kernel where much work is announced, beside 32 and fewer in the other one
    both(Setup(ctx, [10, 3, 16, 0, 8, 9], [100, 40, 300, 5, 8, 700], 8, 2, 128, pad=2, max_kv=200000, garbage=True))
    both(Setup(ctx, [10, 3, 16, 0, 8, 9], [100, 40, 300, 5, 8, 700], 8, 2, 64, pad=2, max_kv=200000, garbage=True), window=90000)
    both(Setup(ctx, [0, 0, 0], [100, 0, 40], 8, 2, 128, pad=200, max_q=150, max_kv=5000, stride=320))
    both(Setup(ctx, [0, 0], [100, 40], 8, 2, 64, pad=3, prefix=33))


@pytest.mark.parametrize("q,D", [(3, 128), (100, 128), (100, 64), (3, 256)])
def test_keys_that_are_not_finite(ctx, q, D):
    """A NaN in K at one key: rows that do not see it are what they were, rows that see it are NaN."""
    kv = q + 60
    s = Setup(ctx, [q], [kv], 4, 2, D)
    at = kv - (q + 1) // 2
    s.k[s.table[0, at // 16], at % 16, 1, 7] = np.nan
    s.close()
    s.buffers = []
    s.upload()
    with np.errstate(invalid="ignore"):
        want = s.want()
    for f16 in (False, True):
        got = s.attend(f16=f16)
        for j in range(q):
            assert np.array_equal(np.isnan(want[j]), np.isnan(got[j])) and np.isnan(got[j, 2:]).all() == (kv - q + j >= at), (f16, j)
            assert np.nanmax(np.abs(want[j] - got[j])) <= (TOL16 if f16 else TOL32)
    s.close()


@pytest.mark.parametrize("q,kv,H,D", [(1, 200000, 4, 128), (128, 40000, 1, 128), (70, 40000, 1, 64), (2, 60000, 2, 256)])
def test_long_sums(ctx, q, kv, H, D):
    """The error of a 32-bit result does not grow with the keys: sums leave the matrix instructions, which cut them instead of rounding, every
    256 keys or earlier. In there at most 32 instructions add to one sum, each off by less than 2^-23 of what the sum has grown to, half its
    end on the average: 32 * 2^-24 = 1.9e-6 at most for values of one sign. The n ordinary additions behind them are rounded, sqrt(n) 2^-24 of
    random sign: 7e-7 for 40000 keys at the most. Left in one accumulator, 40000 keys would be off by 5000 * 2^-24 = 3e-4."""
    s = Setup(ctx, [q], [kv], H, 1, D, 64)
    s.v[:] = np.abs(s.v)      # (sums of one sign: the cuts add up)
    s.close()
    s.buffers = []
    s.upload()
    want, got = s.want(), s.attend()
    y = np.stack([want[j] for j in range(q)])
    assert np.linalg.norm(got - y) <= 2.6e-6 * np.linalg.norm(y)
    s.close()


@pytest.mark.parametrize("q,D,H,Hkv", [(1, 128, 8, 2), (100, 128, 4, 1), (90, 64, 2, 1), (2, 256, 4, 2)])
@pytest.mark.parametrize("softcap", [30.0, 3.0])
def test_capped_scores_of_32_bits(ctx, q, D, H, Hkv, softcap):
    """A score's error is a weight's relative one, and independent from key to key: a result is off by as much of itself as a score is on the
    average. Scores of one: the sum's error (16 additions, 2^-24 each of partial sums below one) 2^-20 at most and 2^-22 on the average, the cap
    2^-23 of the score for small ones and, above a quarter of the cap, 2^-22 of the cap at most: 7e-7 for a cap of 3, where all of it is rare
    for a cap of 30. Twice their sum on the average: 1e-6."""
    s = Setup(ctx, [q], [700], H, Hkv, D, seed=3)
    want, got = s.want(softcap=softcap), s.attend(softcap=softcap)
    y = np.stack([want[j] for j in range(q)])
    assert np.linalg.norm(got - y) <= 1e-6 * np.linalg.norm(y)
    s.close()


def test_recorded_batches_share_a_scratch(ctx):
    """Two graphs whose launches use the same scratch and status words, replayed in turn, and one batch with the same call twice."""
    a = Setup(ctx, [1] * 7, [3000, 5, 17, 900, 2000, 64, 1], 8, 2, 128, seed=1, pad=1)
    b = Setup(ctx, [200, 3], [900, 2000], 8, 2, 128, seed=2, pad=1)
    size = max(paged.scratch_bytes(ctx, s.seqs, heads=8, head_dim=128) for s in (a, b))
    scratch, made = ctx.buffer(size), []
    for s, twice in ((a, False), (b, True)):
        dst = [s.own(np.full((s.held, 8, 128), 77.0, np.float32)) for _ in range(1 + twice)]
        batch = ctx.batch(4)
        for d in dst:
            paged.record_attention(batch, s.cache, s.seqs, s.qb, d, scratch, a.status, heads=8, scale=128 ** -0.5)
        batch.instantiate()
        made.append((s, dst, batch))
    for _ in range(3):
        events = [batch.replay() for _, _, batch in made]
        for ev in events:
            ev.wait()
            ev.destroy()
        for s, dst, _ in made:
            got = [d.read(np.float32) for d in dst]
            assert all(x.tobytes() == got[0].tobytes() for x in got)
            s.check(got[0].reshape(s.held, 8, 128), s.want(), False)
            for d in dst:
                d.write(np.full((s.held, 8, 128), 77.0, np.float32))
    assert a.refused() == [0, 0xFFFFFFFF]
    for _, _, batch in made:
        batch.destroy()
    for s, _, _ in made:
        s.close()
    scratch.destroy()


def test_a_sequence_that_does_not_fit_is_counted_once(ctx):
    s = Setup(ctx, [1, 90, 2], [50, 90, 60], 4, 2, 128)      # both kernels run
    s.seqs.kv_len.write(np.array([50, 90, 10 ** 6], np.int32))
    got = s.attend()
    assert s.refused() == [1, 3] and np.all(got[91:] == 77.0) and np.all(np.isfinite(got[:91]))
    s.close()


@pytest.mark.parametrize("q,kv,prefix", [([1] * 5, [3000, 1, 500, 2000, 77], 0), ([400, 1, 20], [900, 3000, 20], 0), ([1] * 30, [40] * 30, 3000)])
def test_less_scratch_means_fewer_ctas(ctx, q, kv, prefix):
    s = Setup(ctx, q, kv, 8, 2, 128, prefix=prefix)
    want = s.want()
    own = s.held * 8 * 132 * 4 + 256 if prefix else 0
    for scratch in (own + 64, own + 300000, own + 3000000):
        s.check(s.attend(scratch=scratch), want, False)
    a, b = s.attend(), s.attend()
    assert a.tobytes() == b.tobytes()      # nothing depends on the order in which CTAs run
    s.close()


def test_values_that_are_not_finite_reach_the_rows_that_see_them(ctx):
    """A NaN and an infinity in V at key 20: rows before it are what they were, rows from it on are not finite in that column."""
    for q_len, D in ((40, 128), (6, 128), (40, 64), (6, 256)):
        kv = q_len + 10
        s = Setup(ctx, [q_len], [kv], 4, 2, D)
        at = min(20, kv - 3)
        page, token = s.table[0, at // 16], at % 16
        s.v[page, token, 0, 5], s.v[page, token, 1, 9] = np.nan, np.inf
        s.close()
        s.buffers = []
        s.upload()
        got, place = s.attend(), np.arange(kv - q_len, kv)
        with np.errstate(invalid="ignore"):
            want = s.want()
        for j in range(q_len):
            w = want[j]
            assert np.array_equal(np.isnan(w), np.isnan(got[j])) and np.array_equal(np.isposinf(w), np.isposinf(got[j])), (q_len, D, j)
            fine = np.isfinite(w)
            assert np.max(np.abs(w[fine] - got[j][fine])) <= TOL32
            assert np.isnan(got[j, :2, 5]).all() == (place[j] >= at) and np.isposinf(got[j, 2:, 9]).all() == (place[j] >= at)
        s.close()


def test_growing_scores(ctx):
    """Keys sorted so that the maximum grows from tile to tile, by more than the accumulator's rescale step and by less."""
    for q_len, kv in ((100, 1500), (1, 1500)):
        s = Setup(ctx, [q_len], [kv], 4, 1, 128, seed=5)
        s.q[:] = np.abs(s.q)
        flat = np.abs(s.k[s.table[0]]).reshape(-1, 1, 128)
        flat *= np.linspace(0.0, 3.0, flat.shape[0])[:, None, None].astype(np.float16)
        s.k[s.table[0]] = flat.reshape(-1, 16, 1, 128)
        s.close()
        s.buffers = []
        s.upload()
        # scores up to 25: their f32 spacing and the sums' error grow with them, 16 * 2^-23 * 25 of a weight
        want, got = s.want(), s.attend()
        assert max(np.max(np.abs(want[j] - got[j])) for j in want) <= 2 * 16 * 2.0 ** -23 * 25 * 2 * 5.5
        s.close()


def test_numbers_that_do_not_fit_are_left_out_and_counted(ctx):
    """Pages outside the cache are not seen, sequences whose numbers do not fit their buffers are not served."""
    s = Setup(ctx, [1, 1, 90], [200, 60, 90], 4, 2, 128)
    bad = s.table.copy()
    bad[0, 3], bad[2, 1] = s.n_pages, -1
    s.seqs.table.write(bad)
    got = s.attend()
    assert s.refused()[0] > 0 and s.refused()[1] == 3
    # the definition, with those keys taken out: keys and values of the pages packed together
    for row, seq, gone in ((0, 0, 3), (2 + 89, 2, 1)):
        keep = [p for i, p in enumerate(s.table[seq]) if i != gone][:(s.kv_len[seq] + 15) // 16 - 1]
        n = int(s.kv_len[seq]) - 16
        w = ref.attention(s.q[row:row + 1], s.k, s.v, [keep], [0, 1], [n], s.D ** -0.5)[0]
        assert np.max(np.abs(w - got[row])) <= TOL32
    s.seqs.table.write(s.table)
    s.status.write(np.array([0, 0xFFFFFFFF], np.uint32))
    for field, value in (("kv", np.array([10 ** 6, 60, 90], np.int32)), ("kv", np.array([-1, 60, 90], np.int32)),
                         ("q", np.array([0, 1, 2, 2000], np.int32)), ("q", np.array([0, -5, 2, 92], np.int32))):
        (s.seqs.kv_len if field == "kv" else s.seqs.q_start).write(value)
        got = s.attend()
        assert s.refused()[0] >= 1
        if field == "kv":
            assert np.all(got[0] == 77.0)
            s.check(np.concatenate([np.full_like(got[:1], 77.0), got[1:]]), {r: w for r, w in s.want().items() if r}, False)
        s.seqs.kv_len.write(s.kv_len)
        s.seqs.q_start.write(s.q_start)
        s.status.write(np.array([0, 0xFFFFFFFF], np.uint32))
    s.close()


@pytest.mark.parametrize("D", [64, 128])
def test_runs_of_pages_that_are_not_there(ctx, D):
    """Whole key tiles, and more of them than lie between two additions of an accumulator, without a page: in front, inside, at the end."""
    kv, q = 2500, 90
    for gone in (range(0, 60), range(40, 100), range(70, 156)):
        s = Setup(ctx, [q], [kv], 4, 2, D, garbage=True)
        bad = s.table.copy()
        bad[0, list(gone)] = -1
        s.seqs.table.write(bad)
        got = s.attend(), s.attend(f16=True)
        keep = [p for i, p in enumerate(s.table[0]) if i not in gone]
        for j in range(q):
            seen = sum(1 for key in range(kv - q + j + 1) if key // 16 not in gone)
            w = ref.attention(s.q[j:j + 1], s.k, s.v, [keep], [0, 1], [seen], s.D ** -0.5)[0]
            assert np.max(np.abs(w - got[0][j])) <= TOL32 and np.max(np.abs(w - got[1][j])) <= TOL16, (gone, j)
        s.close()


def test_prefix_batches_that_do_not_fit_are_left_out(ctx):
    s = Setup(ctx, [1, 2, 1], [20, 30, 5], 4, 2, 128, prefix=200)
    for buf, value in ((s.seqs.kv_len, np.array([20, 999, 5], np.int32)), (s.seqs.q_start, np.array([1, 1, 3, 4], np.int32))):
        keep = s.kv_len if buf is s.seqs.kv_len else s.q_start
        buf.write(value)
        assert np.all(s.attend() == 77.0) and s.refused()[0] >= 1
        buf.write(keep)
        s.status.write(np.array([0, 0xFFFFFFFF], np.uint32))
    s.check(s.attend(), s.want(), False)
    s.close()


def test_pages_far_into_a_large_cache(ctx):
    """Elements past 2^32: the offsets of pages are 64 bits wide."""
    page, Hkv, D = 64, 8, 128
    per = page * Hkv * D
    n_pages = (1 << 32) // per + 40
    k, v = (ctx.buffer(n_pages * per * 2) for _ in range(2))
    rng = np.random.default_rng(1)
    kv, H = 150, 16
    pages = np.array([[n_pages - 1, n_pages - 30, 3]], np.int32)
    data = [rng.standard_normal((3, page, Hkv, D)).astype(np.float16) for _ in range(2)]
    for buf, x in ((k, data[0]), (v, data[1])):
        for i in range(3):
            buf.write(x[i], offset=int(pages[0, i]) * per * 2)
    for n in (1, 100):
        q = rng.standard_normal((n, H, D)).astype(np.float16)
        bufs = [ctx.buffer(data=x) for x in (pages, np.array([0, n], np.int32), np.array([kv], np.int32), q, np.array([0, 0xFFFFFFFF], np.uint32))]
        dst, scratch = ctx.buffer(n * H * D * 4), ctx.buffer(1 << 26)
        seqs = paged.Sequences(bufs[0], bufs[1], bufs[2], n_seqs=1, table_stride=3, rows=n, max_q=n, max_kv=kv)
        batch = ctx.batch(4)
        paged.record_attention(batch, paged.Cache(k, v, n_pages, page, Hkv, D), seqs, bufs[3], dst, scratch, bufs[4], heads=H, scale=D ** -0.5)
        ev = batch.submit()
        ev.wait()
        ev.destroy()
        batch.destroy()
        got = dst.read(np.float32).reshape(n, H, D)
        want = ref.attention(q, data[0], data[1], [[0, 1, 2]], [0, n], [kv], D ** -0.5)
        assert max(np.max(np.abs(want[r] - got[r])) for r in want) <= TOL32
        for b in bufs + [dst, scratch]:
            b.destroy()
    k.destroy()
    v.destroy()


# ---- append ------------------------------------------------------------------------------------------------------------
def append_and_check(ctx, q_lens, kv_lens, H, Hkv, D, n_dims, neox, page=16, layout="token", far=0, factors=False, yarn=False, pad=0, seed=0, base=10000.0):
    s = Setup(ctx, q_lens, kv_lens, H, Hkv, D, page, layout, seed=seed, pad=pad)
    rng = np.random.default_rng(seed + 1)
    width = (H + 2 * Hkv) * D      # one product's rows: q, k and v beside one another
    rows = rng.standard_normal((s.held, width)).astype(np.float32)
    src = s.own(rows)
    theta = float(np.float32(base ** (-2.0 / max(1, n_dims))))
    kw = dict(freq_scale=0.25, ext_factor=1.0, corr=(0.2 * n_dims, 0.4 * n_dims)) if yarn else {}
    kw = {k: (float(np.float32(v)) if not isinstance(v, tuple) else tuple(float(np.float32(x)) for x in v)) for k, v in kw.items()}
    where = ref.places(s.q_start, s.kv_len)
    pos = np.zeros(s.held, np.int32)
    pos[:s.rows] = [p + far for _, p in where]
    ff = rng.uniform(1.0, 8.0, max(1, n_dims // 2)).astype(np.float32) if factors else None
    out = s.own(np.full((s.held, H, D), 77.0, np.float16))
    batch = ctx.batch(4)
    q_bytes, k_bytes = H * D * 4, Hkv * D * 4
    views = [(src, 0), (src, q_bytes), (src, q_bytes + k_bytes)]
    paged.record_append(batch, s.cache, s.seqs, *views, out, s.status, heads=H, rope=paged.Rope(n_dims, theta, neox=neox, **kw),
                        positions=s.own(pos) if far else None, factors=s.own(ff) if factors else None, q_stride=width, k_stride=width, v_stride=width)
    ev = batch.submit()
    ev.wait()
    ev.destroy()
    batch.destroy()
    cos, sin = ref.rope_angles(pos[:s.rows], n_dims, theta, factors=ff, **kw)
    x = rows[:s.rows]
    wq = ref.rotate(x[:, :H * D].reshape(-1, H, D), cos, sin, n_dims, neox)
    wk = ref.rotate(x[:, H * D:(H + Hkv) * D].reshape(-1, Hkv, D), cos, sin, n_dims, neox)
    wv = x[:, (H + Hkv) * D:].reshape(-1, Hkv, D).astype(np.float64)
    k, v = s.k.astype(np.float64), s.v.astype(np.float64)
    for i, (seq, p) in enumerate(where):
        k[s.table[seq, p // page], p % page], v[s.table[seq, p // page], p % page] = wk[i], wv[i]
    got = out.read(np.float16).reshape(s.held, H, D)
    assert np.all(got[s.rows:] == 77.0)

    def close(a, b):
        b64 = np.abs(b)
        assert np.all(np.abs(a.astype(np.float64) - b) <= b64 * 2.0 ** -11 + 2.0 ** -24 + 8 * 3 * 2.0 ** -22 * (1.2 if yarn else 1.0))

    close(got[:s.rows], wq)
    close(s.from_memory(s.cache.k.read(np.float16)), k)
    close(s.from_memory(s.cache.v.read(np.float16)), v)
    assert s.refused() == [0, 0xFFFFFFFF]
    s.close()


@pytest.mark.parametrize("D,n_dims,neox", [(128, 128, False), (128, 128, True), (64, 32, True), (128, 50, True), (64, 6, False), (256, 256, True),
                                           (128, 0, False), (40, 24, False), (96, 96, True)])
def test_append(ctx, D, n_dims, neox):
    """Rotated widths that are whole units of eight and not, none at all; one product's rows as the source of all three."""
    append_and_check(ctx, [1, 0, 5, 17, 2], [1, 4, 5, 40, 100], 8, 2, D, n_dims, neox, layout="head" if neox else "token", pad=5, seed=D + n_dims)


@pytest.mark.parametrize("far,factors,yarn", [(0, True, False), (1000000, False, False), (123456, True, True), (0, False, True)])
def test_append_angles(ctx, far, factors, yarn):
    append_and_check(ctx, [3, 30], [60, 30], 4, 1, 128, 96, True, page=32, far=far, factors=factors, yarn=yarn, base=500000.0, seed=far)


def test_append_of_many_tokens(ctx):
    """Several tokens per CTA."""
    append_and_check(ctx, [1500, 1, 3600], [1500, 900, 4000], 3, 1, 64, 64, False, page=64, pad=7)


def test_append_refuses_places_without_a_page(ctx):
    s = Setup(ctx, [1, 2, 1, 1], [5, 40, 70, 3], 4, 2, 64)
    bad = s.table.copy()
    bad[1, 2], bad[3, 0] = s.n_pages + 5, -1        # tokens 38, 39 of sequence 1; token 2 of sequence 3
    s.seqs.table.write(bad)
    kv = s.kv_len.copy()
    kv[0], kv[2] = 0, 10 ** 7                       # the token stands at place -1; behind the table
    s.seqs.kv_len.write(kv)
    rng = np.random.default_rng(0)
    q, k = rng.standard_normal((s.held, 4, 64)).astype(np.float32), rng.standard_normal((s.held, 2, 64)).astype(np.float32)
    out = s.own(np.full((s.held, 4, 64), 77.0, np.float16))
    batch = ctx.batch(2)
    paged.record_append(batch, s.cache, s.seqs, s.own(q), s.own(k), s.own(k), out, s.status, heads=4, rope=paged.Rope(64, 0.75), node=9)
    ev = batch.submit()
    ev.wait()
    ev.destroy()
    batch.destroy()
    assert s.refused() == [5, 9]
    assert np.all(out.read(np.float16) == 77.0)
    assert s.cache.k.read(np.float16).tobytes() == s.in_memory(s.k).tobytes() and s.cache.v.read(np.float16).tobytes() == s.in_memory(s.v).tobytes()
    s.close()


# ---- a run of them together --------------------------------------------------------------------------------------------
def test_serving_steps_replayed(ctx):
    """Two prompts appended and attended to, then token steps of both: one recorded batch (append and attention), replayed with lengths
    and tables written between the steps; the same sequences behind a shared prefix in another recorded batch."""
    H, Hkv, D, page, prompts, steps = 8, 2, 128, 16, [70, 23], 5
    rng = np.random.default_rng(4)
    stride, theta = 8, float(np.float32(10000.0 ** (-2.0 / D)))
    pages = rng.permutation(24).astype(np.int32)
    table, prefix_pages, n_prefix = pages[:16].reshape(2, 8), pages[16:19], 41
    k, v = (np.full((24, page, Hkv, D), np.nan, np.float16) for _ in range(2))
    for i in range(n_prefix):      # the prefix has been appended before
        k[prefix_pages[i // page], i % page], v[prefix_pages[i // page], i % page] = rng.standard_normal((2, Hkv, D))
    cb = [ctx.buffer(data=x) for x in (k, v)]
    cache = paged.Cache(cb[0], cb[1], 24, page, Hkv, D)
    rows = 96      # room for the prompts; the step's batch is padded to its rows

    def build(held, max_q):
        b = {name: ctx.buffer(data=x) for name, x in (("table", table), ("q_start", np.zeros(3, np.int32)), ("kv_len", np.zeros(2, np.int32)),
                                                      ("status", np.array([0, 0xFFFFFFFF], np.uint32)),
                                                      ("prefix", np.concatenate([[n_prefix], prefix_pages]).astype(np.int32)))}
        for name, width, size in (("q", H, 4), ("k", Hkv, 4), ("v", Hkv, 4), ("qr", H, 2), ("out", H, 4), ("out_p", H, 2)):
            b[name] = ctx.buffer(held * width * D * size)
        seqs = paged.Sequences(b["table"], b["q_start"], b["kv_len"], n_seqs=2, table_stride=stride, rows=held, max_q=max_q, max_kv=128)
        b["scratch"] = ctx.buffer(paged.scratch_bytes(ctx, seqs, heads=H, head_dim=D, prefix=True))
        batch = ctx.batch(8)
        paged.record_append(batch, cache, seqs, b["q"], b["k"], b["v"], b["qr"], b["status"], heads=H, rope=paged.Rope(D, theta))
        paged.record_attention(batch, cache, seqs, b["qr"], b["out"], b["scratch"], b["status"], heads=H, scale=D ** -0.5)
        paged.record_prefix_attention(batch, cache, seqs, b["qr"], b["out_p"], b["scratch"], b["status"], prefix=b["prefix"], max_prefix=48,
                                      heads=H, scale=D ** -0.5, f16_out=True)
        batch.instantiate()
        return b, batch

    first, token = build(rows, 70), build(4, 1)
    lens = [0, 0]
    for step in range(1 + steps):
        b, batch = first if step == 0 else token
        new = prompts if step == 0 else [1, 1]
        held = rows if step == 0 else 4
        lens = [a + n for a, n in zip(lens, new)]
        q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        x = {n: rng.standard_normal((held, w, D)).astype(np.float32) for n, w in (("q", H), ("k", Hkv), ("v", Hkv))}
        for name in x:
            b[name].write(x[name])
        b["q_start"].write(q_start)
        b["kv_len"].write(np.array(lens, np.int32))
        ev = batch.replay()
        ev.wait()
        ev.destroy()
        # the definition, on what the operators before have stored
        where = ref.places(q_start, lens)
        cos, sin = ref.rope_angles([p for _, p in where], D, theta)
        n = len(where)
        qr = ref.rotate(x["q"][:n], cos, sin, D, False)
        kr = ref.rotate(x["k"][:n], cos, sin, D, False)
        for i, (s, p) in enumerate(where):
            k[table[s, p // page], p % page], v[table[s, p // page], p % page] = kr[i], x["v"][i]
        got_q = b["qr"].read(np.float16).reshape(held, H, D)[:n]
        assert np.max(np.abs(got_q - qr)) <= 8 * 2.0 ** -11
        got_k, got_v = (c.read(np.float16).reshape(k.shape) for c in cb)
        assert np.array_equal(np.isnan(got_k), np.isnan(k)) and np.array_equal(got_v, v, equal_nan=True)
        assert np.nanmax(np.abs(got_k.astype(np.float64) - k)) <= 8 * 2.0 ** -10      # (k here is rounded from 64 bits, there from 32)
        for name, f16, prefix in (("out", False, None), ("out_p", True, (prefix_pages, n_prefix))):
            want = ref.attention(got_q, got_k, got_v, table, q_start, lens, D ** -0.5, prefix=prefix)
            got = b[name].read(np.float16 if f16 else np.float32).reshape(held, H, D)
            y = np.stack([want[r] for r in range(n)])
            assert np.linalg.norm(got[:n] - y) <= (NORM16 if f16 else NORM32) * np.linalg.norm(y), (step, name)
        assert list(b["status"].read(np.uint32)) == [0, 0xFFFFFFFF]
    for b, batch in (first, token):
        batch.destroy()
        for x in b.values():
            x.destroy()
    for x in cb:
        x.destroy()
