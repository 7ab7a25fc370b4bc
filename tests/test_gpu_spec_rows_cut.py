"""Verification where n_tok ends in front of, inside and behind a request's rows."""
import numpy as np
import pytest

from test_gpu_spec_verify import Verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("kids", [1, 3])
@pytest.mark.parametrize("n_tok", [0, 1, 5, 7, 8, 9, 12, 20, 26, 27, 28])
def test_rows_cut_off(flh, gpu, n_tok, kids, draft):
    """Rows that are cut off are not there, but a request's count of tokens has them: len is that without all
    of its rows, and with those of the path."""
    v = Verify(flh, gpu, [5, 3, 0, 12, 1, 6], 700, "F32", draft, kids, seed=n_tok, peak=3.0).push()
    v.p.n_tok = n_tok
    v.p.ws_bytes = flh.spec_verify_ws_bytes(v.p)
    v.run()
    v.start = np.minimum(v.start, n_tok).astype(np.uint32)
    got = v.check()
    for s in range(6):
        assert (got[0][s] > 0) == (v.start[s + 1] > v.start[s])
