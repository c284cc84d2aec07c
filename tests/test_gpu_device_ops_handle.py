"""Handles that go while a capture is under way."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["another thread", "another stream"])
def test_handle_dropped_elsewhere_while_capturing(fb, where):
    """A handle that goes on a thread or under a stream that captures nothing leaves the capture of another alone."""
    x = torch.arange(300, device="cuda").float().view(3, 100)
    ops, box = fb.DeviceOps(0), [fb.DeviceOps(0)]
    want = ops.f8_quantize(x)
    box[0].f8_quantize(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        if where == "another thread":
            t = threading.Thread(target=box.clear)
            t.start()
            t.join()
        else:
            with torch.cuda.stream(side):
                box.clear()
        q, s = ops.f8_quantize(x)
    del ops   # and the graph outlives its own handle
    gr.replay()
    torch.cuda.synchronize()
    assert (q.view(torch.uint8) == want[0].view(torch.uint8)).all() and (s == want[1]).all()
