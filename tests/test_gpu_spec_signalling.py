"""Logits that are no numbers, quiet and signalling ones: -infinity, whatever stands beside them."""
import math

import numpy as np
import pytest
import torch

from test_gpu_spec_verify import Verify
from tree_cases import NONE

pytestmark = pytest.mark.gpu
# quiet and signalling, of both signs, the smallest and the largest payload
BITS = {"F32": (torch.int32, [0x7FC00000, 0x7F800001, 0x7FBFFFFF, 0xFF800001 - (1 << 32), 0xFFFFFFFF - (1 << 32)]),
        "BF16": (torch.int16, [0x7FC0, 0x7F81, 0x7FBF, 0xFF81 - (1 << 16), 0xFFFF - (1 << 16)]),
        "F16": (torch.int16, [0x7E00, 0x7C01, 0x7DFF, 0xFC01 - (1 << 16), 0xFFFF - (1 << 16)])}


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab", [3, 13, 4500, 50257])
def test_no_numbers(flh, gpu, vocab, draft, dtype):
    """Each pattern beside the largest logit, in front of it and behind; drafted tokens that are none; many of them; whole
    rows; greedy requests, too."""
    kind, bits = BITS[dtype]
    for seed in range(2):
        rng = np.random.default_rng(seed)
        v = Verify(flh, gpu, [9] * 6, vocab, dtype, draft, 3, seed=50 + seed, peak=3.0)
        v.inv_temp[[1, 4]] = math.inf
        for t in [v.target] + ([v.draft] if draft else []):
            w = t.view(kind)
            for r in range(v.rows):
                top = int(t[r, :vocab].float().nan_to_num(nan=-math.inf).argmax())
                w[r, [(top + 1) % vocab, (top - 1) % vocab]] = bits[r % len(bits)]
            for r in range(9, v.rows):
                w[r, torch.from_numpy(rng.choice(vocab, max(1, vocab // 3)))] = bits[(r + 1) % len(bits)]
        r0 = int(v.start[2])
        w = v.target.view(kind)
        for j in range(1, 9):                                     # forbidden tokens among the drafted ones
            w[r0 + int(v.parent[r0 + j]), int(v.token[r0 + j])] = bits[j % len(bits)]
        w[int(v.start[3])] = bits[1]
        w[int(v.start[4])] = bits[2]
        v.push().run()
        got = v.check()
        assert got[2][3] == NONE and got[2][4] == NONE
