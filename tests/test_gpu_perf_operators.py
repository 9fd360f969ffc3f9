"""The timed cases of the paged KV cache as a torch program uses them: nothing between a pass and what torch does before and after it waits on the
host, so that the order of the streams has to do."""
import importlib.util
import os

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu
SLEEP = 200_000_000      # clocks, about a tenth of a second


@pytest.mark.parametrize("name", ["attend_draft_32", "append_padded_200", "prefix_6x1000"])
def test_a_pass_is_ordered_with_torchs_stream(name):
    import torch
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
    operators = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(operators)
    case = next(c for c in operators.listed() if c["name"] == name)
    operators.own = True
    s = operators.prepare(case, 1)
    other = operators.prepare(case, 2).q
    first = s.q.clone()

    def passes(wait):
        """The output of a pass over `other`, copied behind it, with torch's stream busy before the input is written."""
        for x in (first, other):
            if not wait:
                torch.cuda._sleep(SLEEP)
            s.q.copy_(x)
            if wait:
                torch.cuda.synchronize()
            out = operators.run(s)
            if wait:
                torch.cuda.synchronize()
            got = [t.clone() for t in (out if isinstance(out, list) else [out])]
            s.q.zero_()      # behind the pass, which has read it
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return got

    before = torch.cuda.current_stream()
    try:
        want = passes(True)
        assert want[0].float().abs().max() > 0
        got = passes(False)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        del s
    finally:
        torch.cuda.synchronize()
        torch.cuda.set_stream(before)      # (the program has made the context's stream torch's)
