"""Inputs that require gradients under grad mode are refused before the
library is called (host side; device -1 is what host tensors answer with)."""
import ctypes
import threading
import types

import pytest


def test_gradients_are_refused_on_the_host_side(t2sc, monkeypatch):
    import torch
    import t2sc.attention as attention
    called = []
    for name in ("_linear", "_rope_apply", "_qk_norm_rope", "_attention"):
        monkeypatch.setattr(attention, name, lambda *a: called.append(a) or 0)
    monkeypatch.setattr(attention, "_raw_stream", lambda device: 7)
    ctx = object.__new__(t2sc.Context)
    ctx.handle, ctx.device, ctx._lock = None, -1, threading.Lock()
    ctx._beside_torch = types.SimpleNamespace(handle=ctypes.c_void_p(64), stream=7)
    x, q, gain, bias = torch.zeros(4, 16), torch.zeros(4, 2, 8), torch.ones(2, 8), torch.zeros(16)
    w = torch.zeros(16, 16)
    coords = torch.zeros(4, 4, dtype=torch.int32)
    rope = object.__new__(attention.RotaryPositionEmbedder)
    rope.ctx, rope.head_dim, rope.layout, rope.handle = ctx, 8, "pairs", None
    layout = object.__new__(attention.SequenceLayout)
    layout.ctx, layout.q_rows, layout.kv_rows, layout.handle = ctx, 4, 4, None
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda f: attention.dense_linear_device(f(x), w, ctx=ctx), lambda f: attention.dense_linear_device(x, f(w), ctx=ctx),
             lambda f: attention.dense_linear_device(x, w, f(bias), ctx=ctx),
             lambda f: attention.dense_linear_device(x, w, residual=f(x), ctx=ctx),
             lambda f: attention.dense_linear_device(x, w, out=f(x), ctx=ctx),
             lambda f: rope.forward_device(f(q), coords), lambda f: rope.forward_device(q, coords, out=f(q)),
             lambda f: attention.qk_norm_rope_device(f(q), None, gain, None, ctx=ctx),
             lambda f: attention.qk_norm_rope_device(q, f(q), gain, gain, ctx=ctx),
             lambda f: attention.qk_norm_rope_device(q, q, f(gain), gain, ctx=ctx),
             lambda f: attention.qk_norm_rope_device(q, q, gain, f(gain), ctx=ctx),
             lambda f: attention.qk_norm_rope_device(q, q, gain, gain, out_q=f(q), ctx=ctx),
             lambda f: attention.qk_norm_rope_device(q, q, gain, gain, out_k=f(q), ctx=ctx),
             lambda f: layout.attention_device(f(q), q, q), lambda f: layout.attention_device(q, f(q), q),
             lambda f: layout.attention_device(q, q, f(q)), lambda f: layout.attention_device(q, q, q, out=f(q))]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(leaf)
    assert not called
    for call in calls:
        call(torch.clone)
        with torch.no_grad():
            call(leaf)
    assert len(called) == 2 * len(calls)
