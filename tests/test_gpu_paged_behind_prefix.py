"""Appending behind a shared prefix: with the positions that count the prefix, sequences that share its pages get what sequences with copies of it get."""
import numpy as np
import pytest

from conftest import load_pkg
from test_gpu_paged import NORM32, ctx  # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu
rt, paged = load_pkg().runtime, load_pkg().paged


@pytest.mark.parametrize("D,neox,prefix,new", [(128, False, 41, [3, 1, 30]), (64, True, 64, [1, 1]), (128, True, 200, [70, 2])])
def test_positions_count_the_prefix(ctx, D, neox, prefix, new):  # noqa: F811
    H, Hkv, page = 8, 2, 16
    rng = np.random.default_rng(prefix)
    theta = float(np.float32(10000.0 ** (-2.0 / D)))
    rows, S, made = sum(new), len(new), []
    x = {n: rng.standard_normal((prefix + rows, w, D)).astype(np.float32) for n, w in (("q", H), ("k", Hkv), ("v", Hkv))}
    per = (prefix + max(new) + page - 1) // page

    def buf(data=None, size=0):
        made.append(ctx.buffer(size, data=data))
        return made[-1]

    def run(lens, before, rows_of, shared):
        """Appends and attends: sequence s has lens[s] new rows, the `rows_of`[s] of x, and before[s] keys in front of them on pages of its own."""
        n = sum(lens)
        table = rng.permutation(S * per + per)[:S * per].reshape(S, per).astype(np.int32)
        pages = np.setdiff1d(np.arange(S * per + per), table).astype(np.int32)[:(prefix + page - 1) // page]
        cache = paged.Cache(*(buf(np.full((S * per + per, page, Hkv, D), np.nan, np.float16)) for _ in range(2)), S * per + per, page, Hkv, D)
        status = buf(np.array([0, 0xFFFFFFFF], np.uint32))
        take = np.concatenate(rows_of)
        out = {}

        def append(batch, table, lens, kv, take, positions):
            seqs = paged.Sequences(buf(table.astype(np.int32)), buf(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)), buf(np.array(kv, np.int32)),
                                   n_seqs=len(lens), table_stride=table.shape[1], rows=len(take), max_q=max(lens), max_kv=max(kv))
            q = buf(size=len(take) * H * D * 2)
            paged.record_append(batch, cache, seqs, *(buf(x[name][take]) for name in ("q", "k", "v")), q, status, heads=H, rope=paged.Rope(D, theta, neox=neox),
                                positions=None if positions is None else buf(np.array(positions, np.int32)))
            return seqs, q

        for offset in ((0, prefix) if shared else (None,)):
            batch = ctx.batch(8)
            if shared:      # the prefix once, as a sequence of its own; then the sequences behind it
                append(batch, pages.reshape(1, -1), [prefix], [prefix], np.arange(prefix), None)
                place = np.concatenate([np.arange(m) for m in lens])
                seqs, q = append(batch, table, lens, lens, take, place + offset)
            else:
                seqs, q = append(batch, table, lens, [a + b for a, b in zip(lens, before)], take, None)
            dst = buf(size=n * H * D * 4)
            kw = dict(heads=H, scale=D ** -0.5)
            scratch = buf(size=paged.scratch_bytes(ctx, seqs, heads=H, head_dim=D, prefix=shared))
            if shared:
                paged.record_prefix_attention(batch, cache, seqs, q, dst, scratch, status, prefix=buf(np.concatenate([[prefix], pages]).astype(np.int32)),
                                              max_prefix=prefix, **kw)
            else:
                paged.record_attention(batch, cache, seqs, q, dst, scratch, status, **kw)
            ev = batch.submit()
            ev.wait()
            ev.destroy()
            batch.destroy()
            out[offset] = dst.read(np.float32).reshape(n, H, D)
            assert list(status.read(np.uint32)) == [0, 0xFFFFFFFF]
        return out

    own = np.split(np.arange(rows) + prefix, np.cumsum(new)[:-1])
    whole = run([prefix + n for n in new], [0] * S, [np.concatenate([np.arange(prefix), r]) for r in own], False)[None]
    at = np.cumsum([0] + [prefix + n for n in new])
    want = np.concatenate([whole[at[s] + prefix:at[s + 1]] for s in range(S)])
    got = run(new, None, own, True)
    assert np.linalg.norm(got[prefix] - want) <= 2 * NORM32 * np.linalg.norm(want)
    assert np.linalg.norm(got[0] - want) > 0.01 * np.linalg.norm(want)      # (positions without the prefix are others)
    for b in made:
        b.destroy()
