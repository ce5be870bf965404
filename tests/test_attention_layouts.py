"""The attention block refuses layouts that are not those of its rows (host side)."""
import types

import numpy as np
import pytest


def _block(t2sc, cross):
    block = object.__new__(t2sc.SparseMultiHeadAttention)
    block.cross, block.channels, block.heads, block.head_dim = cross, 16, 2, 8
    return block


def _layout(q, kv):
    offsets = [np.concatenate([[0], np.cumsum(n)]) for n in (q, kv)]
    return types.SimpleNamespace(q_offsets=offsets[0], kv_offsets=offsets[1], q_rows=sum(q), kv_rows=sum(kv))


@pytest.mark.parametrize("q,kv", [([3, 4], [3, 2]), ([3, 4], [4, 3]), ([5], [4])])
def test_self_attention_refuses_other_keys(t2sc, q, kv):
    import torch
    with pytest.raises(ValueError, match="keys are its queries"):
        _block(t2sc, False).forward_device(torch.zeros(sum(q), 16), _layout(q, kv))


@pytest.mark.parametrize("rows", [4, 6])
def test_cross_attention_refuses_another_contexts_layout(t2sc, rows):
    import torch
    with pytest.raises(ValueError, match="key rows"):
        _block(t2sc, True).forward_device(torch.zeros(7, 16), _layout([3, 4], [3, 2]), context=torch.zeros(rows, 24))
