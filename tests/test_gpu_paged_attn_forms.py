"""Every compiled form of the attention kernels: 17 to 32 rows a kv head at all widths and
types, values not seen at the wide heads, single tokens inside a layer."""
import math

import numpy as np
import pytest
import torch

from paged_cases import attn_bound, attn_oracle
from test_gpu_decoder_attention import Layer
from test_gpu_paged_attn import DIMS, TYPES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("n,window", [(5, 0), (8, 0), (7, 70)])
def test_up_to_32_rows(flh, gpu, act, cdt, dk, dv, n, window):
    """Verify steps: two blocks of 16 rows, requests that fill one of them only, contexts
    around the tiles and one that many workgroups share."""
    lens = [(n, n), (n, n + 31), (1, 200), (n - 1, 64), (n, 5000), (0, 9), (2, 129), (n, 777)]
    c = Case(flh, gpu, act, cdt, 8, 2, dk, dv, 16, "token", lens, 80, window=window)
    c.run()
    first = c.check().clone()
    c.run()
    assert torch.equal(c.result(), first)


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("dk,dv", [(128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("n", [1, 7, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_not_seen(flh, gpu, act, cdt, dk, dv, n, value):
    """As for narrow heads: a key or value that is no number is no part of a row that does
    not see it; a split context and one worked on whole."""
    c = Case(flh, gpu, act, cdt, 8, 2, dk, dv, 16, "head", [(n, 150), (n, n + 7), (n, 3000)], 81)
    for s, kv in ((0, 150), (2, 3000)):
        for j in (kv - n // 2 - 1, kv - 1):
            pg = int(c.table[s, j // 16])
            c.cache.view[1][pg, j % 16, 0, dv - 1] = value
            if math.isnan(value):
                c.cache.view[0][pg, j % 16, 1, dk - 1] = value
    c.cache.push()
    c.run()
    out, mag, amp = attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, True, 0)
    have = c.result()[:, :8 * dv].unflatten(1, (8, dv)).double()[:c.n_tok]
    out, mag, amp = out[:c.n_tok], mag[:c.n_tok], amp[:c.n_tok]
    nan, inf = torch.isnan(out), torch.isinf(out)
    assert nan.any() or inf.any()
    assert torch.equal(torch.isnan(have), nan)
    assert torch.equal(have[inf], out[inf])
    fin = ~nan & ~inf
    lim = attn_bound(out, mag, amp, act, dk, 3000)
    assert ((have - out).abs()[fin] <= lim[fin]).all()


@pytest.mark.parametrize("cdt", ["F16", "BF16"])
@pytest.mark.parametrize("captured", [False, True])
def test_layer_of_single_tokens(flh, gpu, orc, cdt, captured):
    """A prompt, then steps of a token a request through the kernel for few rows."""
    rng = np.random.default_rng(82)
    layer = Layer(flh, gpu, cdt)
    layer.inputs((7, 1, 8), rng)
    layer.issue()
    layer.check((7, 1, 8), orc)
    layer.attn.max_q = 1
    layer.attn.ws_bytes = flh.paged_attn_ws_bytes(layer.cache, layer.attn)
    ws = flh.DeviceBuffer(layer.attn.ws_bytes)
    layer.attn.ws = ws.ptr
    graph = None
    if captured:
        with flh.Graph.capture(gpu) as graph:
            layer.issue()
    for add in [(1, 1, 1), (1, 0, 1), (1, 1, 1), (0, 1, 0), (1, 1, 1)]:
        layer.inputs(add, rng)
        graph.launch() if graph else layer.issue()
        layer.check(add, orc)
    if graph:
        graph.close()
