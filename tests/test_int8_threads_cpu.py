"""CPU: int8_linear from several threads on one layer.  The library is a stand-in that lets another thread's call come between a
call's question for its scratch and the call itself."""
import contextlib
import ctypes as C
import threading

import torch

from moe_gen_b200 import MoELayer


class Lib:
    """Answers with rows * cols bytes, and returns only once both threads have asked."""
    def __init__(self):
        self.both = threading.Barrier(2, timeout=20)
        self.given = {}

    def mg_int8_linear_ws_bytes(self, n, n_out, cols, size):
        C.cast(size, C.POINTER(C.c_size_t)).contents.value = n * cols
        self.both.wait()
        return 0

    def mg_int8_linear(self, h, x, ldx, n, wq, ldw, ws, n_out, cols, scratch, ws_bytes, out, ldo, stream):
        self.given[n] = (ws_bytes, bool(scratch))
        return 0

    def mg_destroy(self, h):
        return 0


def test_every_call_has_its_own_scratch():
    layer = MoELayer.__new__(MoELayer)
    layer.lib, layer.device, layer._h = Lib(), torch.device("cpu"), None
    layer._on_device, layer._stream = contextlib.nullcontext, lambda: 0
    w, s = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)

    def call(n):
        layer.int8_linear(torch.zeros(n, 64, dtype=torch.bfloat16), w, s)

    threads = [threading.Thread(target=call, args=(n,)) for n in (20, 300)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert layer.lib.given == {20: (20 * 64, True), 300: (300 * 64, True)}
