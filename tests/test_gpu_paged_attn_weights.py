"""Few rows with 16-bit activations: the weights are not rounded to the type of the cache, so
the results are off by their own rounding."""
import math

import pytest

from paged_cases import attn_oracle, half_step
from test_gpu_paged_attn import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["F16", "BF16"])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("n", [1, 3, 8])
def test_weights_of_few_rows(flh, gpu, dt, d, n):
    """As attn_bound of 16-bit activations, but the weights (two terms, each half a step off what
    is left) add the square of half a step, and 2^-32 of the largest each over f16 (2^-31 is
    the smallest step), not half a step."""
    lens = [(n, 40), (n, 700), (n, 6000), (1, 2500)]
    c = Case(flh, gpu, dt, dt, 8, 2, d, min(d, 192), 16, "head", lens, 90)
    c.run()
    got = c.check()[:c.n_tok, :8 * c.dv].unflatten(1, (8, c.dv)).double()
    out, mag, amp = [t[:c.n_tok] for t in attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, True, 0)]
    keys, u = 6000, half_step(dt)
    e = amp * (4 * math.sqrt(d) * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -22 + 4 * math.sqrt(keys) * 2.0 ** -24
    lim = mag * (2 * e + u * u)[..., None] + out.abs() * u + 2.0 ** -24
    if dt == "F16":
        lim += keys * 2.0 ** -32 * 6.0                 # (|v| < 6)
    bad = (got - out).abs() > lim
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())
