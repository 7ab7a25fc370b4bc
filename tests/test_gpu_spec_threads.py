"""Threads that issue the operators of a speculative step on one stream, with one workspace, and on streams of their own."""
import pytest

from test_gpu_paged_threads import at_once
from test_gpu_spec_verify import Verify
from test_gpu_tree_attn import Tree

pytestmark = pytest.mark.gpu


def verifies(flh, gpu):
    return [Verify(flh, gpu, [5, 1, 2, 9, 3, 6], 50257, "F32", True, 1, seed=1).push(),
            Verify(flh, gpu, [1, 30, 7, 0, 13], 9001, "BF16", True, 3, seed=2, peak=3.0).push(),
            Verify(flh, gpu, [4] * 70, 1003, "F16", False, 2, seed=3).push()]


def trees(flh, gpu):
    return [Tree(flh, gpu, "F32", "F16", 8, 2, 128, 128, 16, "head", [(8, 5000), (3, 3000)], 70),
            Tree(flh, gpu, "BF16", "BF16", 8, 2, 64, 64, 16, "head", [(40, 3000), (30, 1000)], 71),
            Tree(flh, gpu, "F32", "BF16", 8, 2, 128, 128, 16, "token", [(16, 9000), (1, 40)], 72, window=500)]


@pytest.mark.parametrize("make", [verifies, trees])
def test_calls_that_share_a_workspace(flh, gpu, make):
    cases = make(flh, gpu)
    ws = flh.DeviceBuffer(max(c.p.ws_bytes for c in cases))
    for c in cases:
        c.p.ws, c.p.ws_bytes = ws.ptr, ws.nbytes
    gpu.sync()
    for _ in range(4):
        at_once([lambda c=c: [c.run() for _ in range(30)] for c in cases])
        gpu.sync()
        for c in cases:
            c.check()


@pytest.mark.parametrize("make", [verifies, trees])
def test_streams_of_their_own(flh, gpu, make):
    cases = make(flh, gpu)
    streams = [flh.Stream() for _ in cases]
    gpu.sync()
    for _ in range(3):
        at_once([lambda c=c, s=s: [c.run(s) for _ in range(30)] for c, s in zip(cases, streams)])
        for s in streams:
            s.sync()
        for c in cases:
            c.check()
    for s in streams:
        s.close()


def test_requests_without_rows(flh, gpu):
    for draft in (False, True):
        v = Verify(flh, gpu, [0, 0, 0], 100, "F32", draft, 2).push()
        for _ in range(2):
            v.run()
            v.check()
