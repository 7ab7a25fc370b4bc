"""Sines and cosines of rotary positions, each to fp32's precision: (0, 1) turns into
(-sin, cos), (1, 0) into (cos, sin)."""
import math

import numpy as np
import pytest
import torch

from paged_cases import get, put
from test_gpu_rope import freqs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("base,n_rot", [(10000.0, 64), (500000.0, 128), (1e7, 256)])
@pytest.mark.parametrize("sign", [1, -1])
def test_angles(flh, gpu, base, n_rot, sign):
    """The angle is off by |pos| 2^-65 of a turn (the rounding of the frequency; the frequency
    itself, a double here, by 2^-52) and by a float's rounding of what is left of it, sincospi by 2 ulp
    (4 * 2^-24), the product by one rounding: 6 * 2^-24 of the value.  Next to a multiple of a quarter
    turn the rest's float rounding (2^-24 of it) is one of the value again."""
    p = n_rot // 2
    pos = sign * np.array([0, 1, 2, 3, 5, 17, 100, 999, 4097, 65537, 1 << 20], np.int64)
    n = len(pos)
    x = torch.zeros(n, 2, n_rot)
    x[:, 0, p:] = 1.0                                  # head 0: (0, 1)
    x[:, 1, :p] = 1.0                                  # head 1: (1, 0)
    bx, bp = put(flh, gpu, x), put(flh, gpu, torch.from_numpy(pos.astype(np.int32)))
    t = flh.RopeTable(n_rot, base=base, layout=flh.RopeLayout.HALVES)
    flh.rope(t, flh.Dtype.F32, bx, 2 * n_rot, n_rot, bx, 2 * n_rot, n_rot, n, 2, n_rot, bp, n, gpu)
    got = get(bx, x, gpu).double().numpy()
    t.close()
    ang = pos[:, None] * freqs(n_rot, base)[None, :]
    sin, cos = np.sin(ang), np.cos(ang)
    off = np.abs(pos)[:, None] * 2.0 ** -65 * 2 * math.pi + np.abs(ang) * 4 * 2.0 ** -52
    for have, want in ((got[:, 0, :p], -sin), (got[:, 0, p:], cos), (got[:, 1, :p], cos), (got[:, 1, p:], sin)):
        err = np.abs(have - want)
        assert (err <= np.abs(want) * 6 * 2.0 ** -24 + off).all(), (err / np.maximum(np.abs(want), 1e-30)).max()
