"""CPU: workspaces of the serving steps.  A program sizes one for the largest
call that it makes and passes it to every smaller one, so a size never falls
as a call grows."""
from __future__ import annotations

import pytest

# either side of every bound on the rows that the choice of segments has
ROWS = sorted({r + d for r in (1, 2, 8, 9, 16, 32, 63, 64, 128, 255, 256, 342, 512, 1000, 1024, 4096)
               for d in (-1, 0, 1)} - {0})


@pytest.mark.parametrize("n_top", [0, 1, 20, 32])
def test_logprob_workspaces_grow_with_the_call(lib, n_top):
    before = [0] * len(ROWS)
    for V in (1, 4096, 4097, 8192, 8193, 9000, 12289, 32000, 50257, 128256, 262145, 600000, 1 << 30):
        need = [lib.cgx_token_logprobs_ws(r, V, n_top) for r in ROWS]
        assert need == sorted(need), V                                 # rows
        assert all(a <= b for a, b in zip(before, need)), V            # vocabulary
        if n_top:
            assert all(lib.cgx_token_logprobs_ws(r, V, n_top - 1) <= n for r, n in zip(ROWS, need))
        before = need
    assert lib.cgx_token_logprobs_ws(0, 32000, n_top) == 0
