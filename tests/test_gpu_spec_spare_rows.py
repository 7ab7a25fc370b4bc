"""Verification in a captured step's manner: n_tok is room for more rows than there are."""
import numpy as np
import pytest
import torch

from test_gpu_spec_verify import Verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("kids", [1, 3])
@pytest.mark.parametrize("n", [[5, 1, 9, 0, 4], [0, 0], [30]])
def test_spare_rows(flh, gpu, n, kids, draft):
    """Rows behind the last request change nothing, whatever stands in their place; parents there that point at rows."""
    rng = np.random.default_rng(60)
    v = Verify(flh, gpu, n, 9001, "F32", draft, kids, seed=60, peak=3.0, chain=False)
    for spare in (0, 1, 70):
        w = Verify(flh, gpu, n, 9001, "F32", draft, kids, seed=60, peak=3.0, chain=False)
        w.rows = v.rows + spare
        more = max(0, w.rows - len(w.token))
        fill = lambda t: torch.cat([t, torch.full((more, w.pitch), float("nan"), dtype=t.dtype)])      # noqa: E731
        w.target, w.draft = fill(w.target), fill(w.draft) if draft else None
        w.token = np.concatenate([w.token, rng.integers(0, 9001, more).astype(np.uint32)])
        w.parent = np.concatenate([w.parent, rng.integers(0, 5, more).astype(np.int32)])
        w.u_accept = np.concatenate([w.u_accept, np.zeros(more, np.float32)])
        w.push().run()
        got = w.check()
        if spare == 0:
            first = got
        for a, b in zip(got, first):
            np.testing.assert_array_equal(a, b)
