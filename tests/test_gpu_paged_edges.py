"""Calls of the paged operators at the edges of what their interface allows."""
import pytest

import vb200
from test_gpu_paged import PAIRS, Setup, attn_reference

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------- descriptors

@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("starts", [[0, 1000, 2000], [0, 1000, 1000, 2000, 2000], [0, 1000, 1999]])
def test_a_sequence_behind_the_rows_takes_no_other_ones_place(io, cache, starts):
    # the last rows claimed lie behind `tokens`; sequence 0 has all of its own
    n = len(starts) - 1
    s = Setup([1000] + [0] * (n - 1), [1000] * n, io, cache, seed=3)
    want, _, tol, _ = attn_reference(s)
    s.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
    out = s.out()
    vb200.paged_attn(s.pc, s.pb, s.q, out)
    assert int(s.status) == vb200.PAGED_BAD_ROWS
    assert ((out.double() - want).abs() <= tol).all()
