"""A prefix's length is read on the device: none at all, or a part of what is announced, in a recorded call."""
import numpy as np
import pytest

from conftest import load_pkg
from oracle import paged as ref
from test_gpu_paged import NORM16, NORM32, Setup, ctx  # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu
rt, paged = load_pkg().runtime, load_pkg().paged


@pytest.mark.parametrize("D,H,Hkv,q", [(128, 8, 2, [1, 3, 0, 2]), (64, 14, 2, [1] * 20), (128, 4, 2, [90, 1]), (256, 4, 2, [2, 1])])
@pytest.mark.parametrize("f16", [False, True])
def test_replayed(ctx, D, H, Hkv, q, f16):  # noqa: F811
    kv = [n + 30 for n in q]
    s = Setup(ctx, q, kv, H, Hkv, D, seed=D, pad=1, garbage=True, prefix=500)
    dt = np.float16 if f16 else np.float32
    dst, pb = s.own(np.full((s.held, H, D), 77.0, dt)), s.own(s.prefix)
    scratch = s.own(size=paged.scratch_bytes(ctx, s.seqs, heads=H, head_dim=D, prefix=True))
    batch = ctx.batch(4)
    paged.record_prefix_attention(batch, s.cache, s.seqs, s.qb, dst, scratch, s.status, prefix=pb, max_prefix=500, heads=H, scale=D ** -0.5, f16_out=f16)
    batch.instantiate()
    for n in (500, 0, 1, 17, 499, 0, 64):
        pb.write(np.concatenate([[n], s.prefix[1:]]).astype(np.int32))
        ev = batch.replay()
        ev.wait()
        ev.destroy()
        want = ref.attention(s.q, s.k, s.v, s.table, s.q_start, s.kv_len, D ** -0.5, prefix=(s.prefix[1:], n) if n else None)
        got = dst.read(dt).reshape(s.held, H, D)
        y = np.stack([want[r] for r in range(s.rows)])
        assert np.linalg.norm(got[:s.rows] - y) <= (NORM16 if f16 else NORM32) * np.linalg.norm(y), n
        assert np.all(got[s.rows:] == 77.0)
    assert s.refused() == [0, 0xFFFFFFFF]
    batch.destroy()
    s.close()
