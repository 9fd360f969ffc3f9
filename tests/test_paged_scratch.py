"""The scratch of the attention over a paged KV cache is sized by the SMs of the context's device."""
import types

import pytest

from conftest import load_pkg

rt, paged = load_pkg().runtime, load_pkg().paged
SEQS = paged.Sequences(None, None, None, n_seqs=3, table_stride=4, rows=100, max_q=10, max_kv=1000)


@pytest.mark.parametrize("prefix", [False, True])
def test_by_the_context(prefix):
    kw = dict(heads=8, head_dim=128, prefix=prefix)
    sizes = [paged.scratch_bytes(types.SimpleNamespace(sm_count=n), SEQS, **kw) for n in (37, 148, 160)]
    per_sm = 2 * (8 * 16 + 256) * 132 * 4 + 128
    assert sizes[1] - sizes[0] == 111 * per_sm and sizes[2] - sizes[1] == 12 * per_sm
    assert paged.scratch_bytes(types.SimpleNamespace(sm_count=148), SEQS, sms=37, **kw) == sizes[0]


@pytest.mark.gpu
def test_the_device_is_asked():
    import torch
    ctx = rt.init()
    assert ctx.sm_count == torch.cuda.get_device_properties(0).multi_processor_count
    assert paged.scratch_bytes(ctx, SEQS, heads=8, head_dim=64) == paged.scratch_bytes(ctx, SEQS, heads=8, head_dim=64, sms=ctx.sm_count)
    ctx.destroy()
