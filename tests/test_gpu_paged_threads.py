"""Threads that issue on one stream: attention calls that share a workspace, and page plans
over tables of their own."""
import threading

import numpy as np
import pytest
import torch

from test_gpu_kv_plan import Plan, check, make_table, oracle
from test_gpu_paged_attn import Case

pytestmark = pytest.mark.gpu


def at_once(fs):
    errors = []

    def guarded(f):
        try:
            f()
        except Exception as e:
            errors.append(e)
    ts = [threading.Thread(target=guarded, args=(f,)) for f in fs]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("own", [True, False])
def test_attention_calls_that_share_a_workspace(flh, gpu, own):
    cases = [Case(flh, gpu, "F32", "F16", 8, 2, 128, 128, 16, "head", [(1, 5000), (1, 3000)], 60),
             Case(flh, gpu, "BF16", "BF16", 8, 2, 64, 64, 16, "head", [(40, 3000), (30, 1000)], 61),
             Case(flh, gpu, "F16", "F16", 4, 4, 128, 128, 16, "head", [(6, 9000)], 62)]
    ws = flh.DeviceBuffer(max(c.p.ws_bytes for c in cases))
    for c in cases:
        c.p.ws, c.p.ws_bytes = ws.ptr, ws.nbytes
    gpu.sync()
    torch_stream = None if own else torch.cuda.Stream()
    stream = gpu if own else flh.Stream.wrap(torch_stream.cuda_stream)
    for _ in range(5):
        at_once([lambda c=c: [c.run(stream) for _ in range(40)] for c in cases])
        stream.sync()
        for c in cases:
            c.check()


def test_plans_of_two_launches(flh, gpu):
    plans = []
    for seed in (1, 2, 3):
        rng = np.random.default_rng(seed)
        held, add = rng.integers(0, 300, 50).astype(np.uint32), rng.integers(0, 200, 50).astype(np.uint32)
        table, free = make_table(held, 16, 40, rng, 50 * 40)
        p = Plan(flh, gpu, held, add, 16, free, seed, table, 9000 + seed)
        plans.append((p, oracle(held, add, 16, free, seed, table, 9000 + seed, p.slot0, p.pos0)))
    gpu.sync()
    for _ in range(3):
        at_once([lambda p=p: [flh.kv_plan(p.p, gpu) for _ in range(30)] for p, _ in plans])
        for p, want in plans:
            check(p.read(), want)
