"""How exact f16 results of the attention over a paged KV cache are: as near to the 64-bit result as its rounding leaves, whichever kernel forms
them, and however few CTAs share it."""
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
