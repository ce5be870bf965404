"""Calls on a closed Context do not reach the library."""
import threading
import types

import pytest


def test_a_closed_contexts_handles_are_refused(t2sc, monkeypatch):
    import torch
    import t2sc.attention as attention
    called = []
    for name in ("_linear", "_rope_apply", "_qk_norm_rope", "_attention"):
        monkeypatch.setattr(attention, name, lambda *a: called.append(a) or 0)
    monkeypatch.setattr(attention, "_raw_stream", lambda device: 7)
    ctx = object.__new__(t2sc.Context)
    # as Context.close leaves it, with the stream of the next call already set
    ctx.handle, ctx.device, ctx._lock = None, -1, threading.Lock()
    ctx._beside_torch = types.SimpleNamespace(handle=None, stream=7)
    x, q, gain = torch.zeros(4, 16), torch.zeros(4, 2, 8), torch.ones(2, 8)
    coords = torch.zeros(4, 4, dtype=torch.int32)
    rope = object.__new__(attention.RotaryPositionEmbedder)
    rope.ctx, rope.head_dim, rope.layout, rope.handle = ctx, 8, "pairs", None
    layout = object.__new__(attention.SequenceLayout)
    layout.ctx, layout.q_rows, layout.kv_rows, layout.handle = ctx, 4, 4, None
    for call in (lambda: attention.dense_linear_device(x, x, ctx=ctx), lambda: rope.forward_device(q, coords),
                 lambda: attention.qk_norm_rope_device(q, None, gain, None, coords=coords, rope=rope),
                 lambda: layout.attention_device(q, q, q)):
        with pytest.raises(ValueError, match="closed"):
            call()
    assert not called
    ctx._beside_torch = None   # closed before any such call
    with pytest.raises(ValueError, match="closed"):
        attention.dense_linear_device(x, x, ctx=ctx)
