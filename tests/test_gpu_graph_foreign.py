"""Replays by several threads onto one stream that was not made by this library."""
import ctypes
import threading

import numpy as np
import pytest

from oracle import Q4_K, col_stride_floats
from util import activations, sane_rows
from test_gpu_parity import bits, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["foreign", "default"])
@pytest.mark.parametrize("dots", [2, 4])
def test_replays_stay_whole(flh, gpu, kind, dots):
    """Graphs over the same buffers and eager copies of what they leave: each replay is
    whole, so every copy is the result of one."""
    say("graph threads, stream made elsewhere")
    rows, cols, reps, rng = 64, 512, 60, np.random.default_rng(8)
    xb = np.zeros(col_stride_floats(cols), np.float32)
    xb[:cols] = activations(1, cols, rng)[0]
    dx, dw = flh.DeviceBuffer.from_array(xb, gpu), flh.DeviceBuffer.from_array(sane_rows(Q4_K, rows, cols, rng), gpu)
    dy, seen = flh.DeviceBuffer(4 * rows), flh.DeviceBuffer(4 * rows * reps)
    graphs = [flh.Graph.capture(gpu) for _ in range(3)]
    for g in graphs:
        with g:
            dy.zero(gpu)
            flh.act_q8(dx, cols, gpu)
            for _ in range(dots):
                flh.stream_dot(Q4_K, dw, rows, cols, dx, dy, gpu)
    graphs[0].launch(gpu)
    want = dy.download(np.float32, rows, gpu)
    handle, hip = ctypes.c_void_p(), flh.lib()
    if kind == "foreign":
        assert hip.hipStreamCreateWithFlags(ctypes.byref(handle), 1) == 0   # 1: hipStreamNonBlocking
    stream, errors = flh.Stream.wrap(handle.value), []

    def guarded(f):
        def run():
            try:
                f()
            except Exception as e:
                errors.append(e)
        return threading.Thread(target=run)

    ts = [guarded(lambda g=g: [g.launch(stream) for _ in range(100)]) for g in graphs]
    ts.append(guarded(lambda: [flh.copy(seen.ptr + 4 * rows * i, dy, 4 * rows, stream) for i in range(reps)]))
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    stream.sync()
    assert not errors, errors
    got = seen.download(np.float32, rows * reps, stream).reshape(reps, rows)
    assert np.array_equal(bits(got), bits(np.broadcast_to(want, got.shape)))
    assert np.array_equal(bits(dy.download(np.float32, rows, stream)), bits(want))
    for g in graphs:
        g.close()
    if kind == "foreign":
        assert hip.hipStreamDestroy(handle) == 0
