"""The attention-block entry points refuse bad arguments before they touch a
device, and their host-side checks of layouts and strides behave."""
import ctypes
import types

import numpy as np
import pytest


def _fake_ctx():
    return types.SimpleNamespace(device=0, handle=None, set_stream=lambda s: None)


def test_entry_points_reject_null_handles(t2sc):
    L, E = t2sc.lib, t2sc._lib.ERR_INVALID
    out = ctypes.c_void_p()
    assert L.t2sc_dense_linear_device(None, None, 8, None, 8, None, None, 0, None, 8, 4, 8, 8, 0, 2) == E
    assert L.t2sc_rope_create(None, 64, 10, 10, 10, 1e4, 0, ctypes.byref(out)) == E
    assert L.t2sc_rope_apply_device(None, None, None, 64, None, 64, 4, 1, 2) == E
    assert L.t2sc_qk_norm_rope_device(None, None, None, None, 64, None, 0, None, None, None, 64, None, 0, 4, 1, 64,
                                      1e-6, 2) == E
    assert L.t2sc_seqs_create(None, None, None, 0, ctypes.byref(out)) == E
    assert L.t2sc_attention_device(None, None, 64, None, 64, None, 64, None, 64, 1, 64, 1.0, 2) == E
    assert L.t2sc_rope_destroy(None) == 0 and L.t2sc_seqs_destroy(None) == 0 and not out.value


def test_host_tensors_are_refused(t2sc):
    import torch
    x, w = torch.zeros(4, 16), torch.zeros(8, 16)
    for ctx in (None, _fake_ctx()):
        with pytest.raises(ValueError):
            t2sc.dense_linear_device(x, w, ctx=ctx)
        with pytest.raises(ValueError):
            t2sc.qk_norm_rope_device(x.view(4, 2, 8), None, torch.ones(2, 8), None, ctx=ctx)
    layout = object.__new__(t2sc.SequenceLayout)
    layout.ctx, layout.q_rows, layout.kv_rows = _fake_ctx(), 4, 4
    q = x.view(4, 2, 8)
    with pytest.raises(ValueError):
        layout.attention_device(q, q, q)
    emb = object.__new__(t2sc.RotaryPositionEmbedder)
    emb.ctx, emb.head_dim, emb.layout = _fake_ctx(), 8, "pairs"
    with pytest.raises(ValueError):
        emb.forward_device(q, torch.zeros(4, 4, dtype=torch.int32))


def test_constructor_arguments(t2sc):
    for lens in ([-1, 3], [2, -5]):
        with pytest.raises(ValueError):
            t2sc.SequenceLayout(lens, ctx=_fake_ctx())
    with pytest.raises(ValueError):
        t2sc.SequenceLayout([1, 2], [3], ctx=_fake_ctx())
    with pytest.raises(ValueError):
        t2sc.RotaryPositionEmbedder(64, layout="spiral", ctx=_fake_ctx())
    with pytest.raises(ValueError):
        t2sc.RotaryPositionEmbedder(64, pairs=(8, 8), ctx=_fake_ctx())
    w = (np.zeros((16, 16)), np.zeros(16))
    with pytest.raises(ValueError):
        t2sc.SparseMultiHeadAttention(16, 3, w, to_qkv=(np.zeros((48, 16)), None), ctx=_fake_ctx())   # 16 % 3
    with pytest.raises(ValueError):
        t2sc.SparseMultiHeadAttention(16, 2, w, ctx=_fake_ctx())                                       # no projections
    with pytest.raises(ValueError):
        t2sc.SparseMultiHeadAttention(16, 2, w, to_q=w, to_kv=w, rope=object(), ctx=_fake_ctx())       # rope in cross-attention
    with pytest.raises(ValueError):
        t2sc.SparseFeedForwardNet(w, w, activation="relu", ctx=_fake_ctx())
