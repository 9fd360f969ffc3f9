"""What the attention over a paged KV cache reads beside the keys it is asked about (the rest of a page, shared memory that an earlier kernel
has left, rows of q behind the batch) takes no part in its results: the bytes are the same, whatever is there."""
import numpy as np
import pytest

from conftest import load_pkg
from test_gpu_paged import Setup, ctx  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
rt, paged = load_pkg().runtime, load_pkg().paged


def used_tokens(s):
    used = np.zeros((s.n_pages, s.page), bool)
    for seq, n in enumerate(s.kv_len):
        for i in range(n):
            used[s.table[seq, i // s.page], i % s.page] = True
    for i in range(0 if s.prefix is None else int(s.prefix[0])):
        used[s.prefix[1 + i // s.page], i % s.page] = True
    return used


def bytes_of(s, used, fill, f16, **kw):
    """The results with every token that no sequence has, and every row of q behind the last, set to `fill`."""
    for x in (s.k, s.v):
        x[~used] = fill
    s.q[s.rows:] = fill
    s.cache.k.write(s.in_memory(s.k))
    s.cache.v.write(s.in_memory(s.v))
    s.qb.write(s.q)
    return s.attend(f16=f16, **kw)[:s.rows].tobytes()


@pytest.mark.parametrize("D,H,Hkv,page,layout", [(128, 8, 2, 16, "token"), (64, 14, 2, 32, "head"), (256, 4, 2, 64, "token")])
@pytest.mark.parametrize("q,window,prefix", [(1, 0, 0), (1, 21, 0), (5, 37, 0), (80, 0, 0), (80, 45, 0), (2, 0, 70)])
@pytest.mark.parametrize("softcap", [30.0, 3.0])
def test_a_cap_does_not_depend_on_what_nobody_sees(ctx, D, H, Hkv, page, layout, q, window, prefix, softcap):  # noqa: F811
    """Lengths that end inside a block of 16 keys, inside a pair of them and at their borders; windows that begin inside one. Between the runs
    a call over other pages leaves its own keys in shared memory."""
    kv = [q, q + 1, q + 7, q + 14, q + 15, q + 16, q + 20, q + 47]
    s = Setup(ctx, [q] * len(kv), kv, H, Hkv, D, page, layout, seed=D + q + window, pad=3, prefix=prefix)
    other = Setup(ctx, [q], [300], H, Hkv, D, page, layout, seed=1)
    used, kw = used_tokens(s), dict(softcap=softcap, **({"window": window} if window else {}))
    for f16 in (False, True):
        got = set()
        for fill in (0.0, 200.0, -60000.0, np.inf, np.nan):
            other.cache.k.write(np.full(other.k.shape, fill, np.float16))
            other.attend(f16=f16)
            got.add(bytes_of(s, used, fill, f16, **kw))
        assert len(got) == 1, f16
    other.close()
    s.close()
