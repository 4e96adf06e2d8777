"""The library's first call, in a process of its own (tests/test_gpu_first_call.py): one argument names the case."""
import os
import sys

import torch
from torch._subclasses.fake_tensor import FakeTensorMode

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))), "data-compression_amd"))
import dcamd  # noqa: E402

started = lambda: dcamd.lib().L.dc_get_device()  # noqa: E731


def refused(f, what):
    try:
        f()
    except ValueError as e:
        assert what in str(e), e
    else:
        raise AssertionError("not refused")
    assert started() == -1


case = sys.argv[1]
dcamd.native()
if case == "device":                # a tensor of a device that is not the current one (a stand-in: it has no memory)
    torch.cuda.init()
    torch._subclasses.fake_tensor.init_gpu_context = lambda device: None
    with FakeTensorMode():
        x = torch.empty(4, 8, device="cuda:1")
    refused(lambda: dcamd.act_forward(x, "silu"), "current device")
    assert torch.cuda.current_device() == 0
elif case == "status":              # a status before any call: nothing has run
    assert dcamd.KVCache.status() == 0 and started() == -1
elif case == "capture":
    x = torch.ones(4, 8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        refused(lambda: dcamd.act_forward(x, "silu"), "captured")
    graph.replay()
    torch.cuda.synchronize()
    assert float(y.sum()) == 64
elif case == "threads":             # several at once, from C: one start, the same stream for all
    import ctypes
    import threading
    torch.zeros(1, device="cuda")
    L, gate, got = dcamd.lib().L, threading.Barrier(8), []

    def first():
        word = ctypes.c_uint(7)
        gate.wait()
        rc = L.dc_kv_status(None, ctypes.byref(word), 0)
        got.append((rc, word.value, L.dc_get_stream(), L.dc_get_device()))

    threads = [threading.Thread(target=first) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 8 and len(set(got)) == 1 and got[0][:2] == (0, 0) and got[0][2] and got[0][3] == 0, got
want = torch.nn.functional.silu(torch.ones(4, 8))
got, _ = dcamd.act_forward(torch.ones(4, 8, device="cuda"), "silu")
assert torch.allclose(got.cpu(), want) and started() == 0
print("fine")
