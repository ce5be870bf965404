"""Host side of the attention-block operators over one Context: calls of
several threads, on stand-ins for the library and for torch's streams (device
-1 is what host tensors answer with)."""
import ctypes
import threading
import time
import types

import pytest


class Library:
    """Stands for the library's calls: notes the stream that the context has when a call is made, and when it ends."""

    def __init__(self):
        self.stream, self.seen, self.mixed = None, [], 0

    def switch(self, stream):
        self.stream = stream
        time.sleep(0.0005)

    def __call__(self, *args):
        first = self.stream
        time.sleep(0.0005)
        self.mixed += first != self.stream
        self.seen.append((threading.get_ident(), first))
        return 0


@pytest.fixture
def host(t2sc, monkeypatch):
    """(attention module, library stand-in, Context over them)."""
    import t2sc.attention as attention
    library, here = Library(), threading.local()
    monkeypatch.setattr(attention, "_raw_stream", lambda device: here.stream)
    for name in ("_linear", "_rope_apply", "_qk_norm_rope", "_attention"):
        monkeypatch.setattr(attention, name, library)
    beside = types.SimpleNamespace(handle=ctypes.c_void_p(64), stream=None)

    def use(stream):
        library.switch(stream)
        beside.stream = stream

    beside.use = use
    ctx = object.__new__(t2sc.Context)
    ctx.handle, ctx.device, ctx._beside_torch, ctx._lock = None, -1, beside, threading.Lock()
    return attention, library, ctx, here


def test_each_call_runs_on_its_own_threads_stream(host):
    import torch
    attention, library, ctx, here = host
    x, w, q, gain = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(4, 2, 8), torch.ones(2, 8)
    coords = torch.zeros(4, 4, dtype=torch.int32)
    rope = object.__new__(attention.RotaryPositionEmbedder)
    rope.ctx, rope.head_dim, rope.layout, rope.handle = ctx, 8, "pairs", None
    layout = object.__new__(attention.SequenceLayout)
    layout.ctx, layout.q_rows, layout.kv_rows, layout.handle = ctx, 4, 4, None
    streams, errors = {}, []

    def work(stream):
        try:
            here.stream = stream
            streams[threading.get_ident()] = stream
            for _ in range(20):
                attention.dense_linear_device(x, w, ctx=ctx)
                rope.forward_device(q, coords)
                attention.qk_norm_rope_device(q, None, gain, None, ctx=ctx)
                layout.attention_device(q, q, q)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(100 + i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert len(library.seen) == 3 * 20 * 4 and not library.mixed
    assert all(streams[thread] == stream for thread, stream in library.seen)


def test_one_default_context_for_all_threads(t2sc, monkeypatch):
    made = []

    class Slow(t2sc.Context):
        _default = {}

        def __init__(self, device=0):
            time.sleep(0.01)
            made.append(device)

    threads = [threading.Thread(target=Slow.default, args=(0,)) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert made == [0]
