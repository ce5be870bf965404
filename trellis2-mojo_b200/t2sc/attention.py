"""The attention block over voxel tokens, on the device.

Operators over CUDA tensors of rows, each one C-ABI call on torch's current
stream (the stream of the Context that they are given stays as it was set).
They are for inference: under grad mode, inputs that require gradients are
refused. Several threads may call
them with one Context and its handles, or without one; each call runs on its
own thread's current stream. A kernel that gave up a bounded wait, so that its
result is invalid, is reported by the next call with the Context, or by
Context.synchronize.
  dense_linear_device      act(x @ w^T + bias) + residual   (linear, trellis2_mojo/modules/nn.mojo:27-266)
  RotaryPositionEmbedder   rotary positions over x, y, z    (trellis2_mojo/modules/rope.mojo)
  qk_norm_rope_device      per-head RMS norm + rotation     (bias_rms_rope_qkv, trellis2_mojo/gpu/attention.mojo:507)
  SequenceLayout           a ragged batch; attention inside each sequence (trellis2_mojo/sparse/attention)
and the block's two halves made of them:
  SparseMultiHeadAttention, SparseFeedForwardNet
"""
import ctypes

import numpy as np

import torch

from . import _lib
from ._lib import check, lib
from .sparse import _DTYPES, Context, SparseTensor

_ACTIVATIONS = {None: 0, "silu": _lib.SILU, "gelu": _lib.GELU}
_LAYOUTS = {"pairs": _lib.ROPE_PAIRS, "halves": _lib.ROPE_HALVES}
_CODES = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
_Tensor = torch.Tensor
_linear, _rope_apply = lib.t2sc_dense_linear_device, lib.t2sc_rope_apply_device
_qk_norm_rope, _attention = lib.t2sc_qk_norm_rope_device, lib.t2sc_attention_device


def _code(t, what):
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16")
    return code


def _rows2d(t, device, dtype, what):
    """(rows, width, row stride) of a [rows, width] tensor whose rows are contiguous."""
    if not isinstance(t, _Tensor) or t.get_device() != device:
        raise ValueError(f"{what} must be a CUDA tensor on cuda:{device}")
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 2:
        raise ValueError(f"{what} must be [rows, width] of {dtype}")
    rows, width = shape
    if t.is_contiguous():
        return rows, width, width
    stride, inner = t.stride()
    if width > 1 and inner != 1:
        raise ValueError(f"{what} must have contiguous rows")
    return rows, width, _row_stride(rows, width, stride, what)


def _heads3d(t, device, dtype, what):
    """(rows, heads, head_dim, row stride) of a [rows, heads, head_dim] tensor whose rows are contiguous."""
    if not isinstance(t, _Tensor) or t.get_device() != device:
        raise ValueError(f"{what} must be a CUDA tensor on cuda:{device}")
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 3:
        raise ValueError(f"{what} must be [rows, heads, head_dim] of {dtype}")
    rows, h, d = shape
    if t.is_contiguous():
        return rows, h, d, h * d
    stride, per_head, inner = t.stride()
    if (d > 1 and inner != 1) or (h > 1 and per_head != d):
        raise ValueError(f"{what} must have contiguous rows")
    return rows, h, d, _row_stride(rows, h * d, stride, what)


def _row_stride(rows, width, stride, what):
    if rows <= 1:
        return width
    if stride < width:
        raise ValueError(f"{what}: rows overlap")
    return stride


def _f32(t, device, shape, what):
    if not isinstance(t, _Tensor) or t.get_device() != device or t.dtype is not torch.float32 or \
            t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous float32 {list(shape)} on cuda:{device}")
    return t.data_ptr()


def _coords(t, device, rows):
    if not isinstance(t, _Tensor) or t.get_device() != device or t.dtype is not torch.int32 or \
            t.shape != (rows, 4) or not t.is_contiguous():
        raise ValueError(f"coords must be contiguous int32 [rows, 4] on cuda:{device}")
    return t.data_ptr()


def _no_gradient():
    """Some tensor of the call requires gradients."""
    if torch.is_grad_enabled():
        raise ValueError("the operator has no gradient: call it under torch.no_grad(), or with detached tensors")


def _context(ctx, t):
    if ctx is not None:
        return ctx
    if not isinstance(t, _Tensor) or not t.is_cuda:
        raise ValueError("the operator takes CUDA tensors")
    return Context.default(t.get_device())


def _on_torch_stream(ctx):
    """The library context to call with, its work on torch's current stream of the device. Under the context's lock,
    which is held until the call is made and its error is read (acquired by name: `with` takes twice as long)."""
    stream = torch.cuda.current_stream(ctx.device).cuda_stream if _raw_stream is None else _raw_stream(ctx.device)
    stream = stream or 1    # handle 0 would name the context's own stream, 1 is cudaStreamLegacy
    beside = ctx._beside_torch or ctx.beside_torch()
    handle = beside.handle
    if handle is None:
        raise ValueError("the Context is closed")
    if beside.stream != stream:
        beside.use(stream)
    return handle


# the handle alone, without a Stream object around it (2 us less a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def dense_linear_device(x, weight, bias=None, activation=None, residual=None, out=None, ctx=None):
    """act(x @ weight.T + bias) + residual. x [rows, ci] and weight [co, ci]:
    CUDA tensors of one type (float16, bfloat16 or float32) whose rows may be
    strided; bias float32 [co]; activation None, "silu" or "gelu" (tanh
    form); residual and out [rows, co] of x's type, out may be residual."""
    ctx = _context(ctx, x)
    device, dtype = ctx.device, x.dtype
    if activation not in _ACTIVATIONS:
        raise ValueError('dense_linear: activation must be None, "silu" or "gelu"')
    code, flags = _code(x, "dense_linear: x"), _ACTIVATIONS[activation]
    rows, ci, ldx = _rows2d(x, device, dtype, "dense_linear: x")
    co, wi, ldw = _rows2d(weight, device, dtype, "dense_linear: weight")
    if wi != ci or ci < 1 or co < 1:
        raise ValueError("dense_linear: weight must be [co, ci] with x's ci")
    res, ldr = None, 0
    if residual is not None:
        r, w, ldr = _rows2d(residual, device, dtype, "dense_linear: residual")
        if r != rows or w != co:
            raise ValueError("dense_linear: residual must be [rows, co]")
        res, flags = residual.data_ptr(), flags | _lib.RESIDUAL
    given = out is not None
    if not given:
        out, ldy = x.new_empty((rows, co)), co
    else:
        r, w, ldy = _rows2d(out, device, dtype, "dense_linear: out")
        if r != rows or w != co:
            raise ValueError("dense_linear: out must be [rows, co]")
    b = None if bias is None else _f32(bias, device, (co,), "dense_linear: bias")
    if x.requires_grad or weight.requires_grad or (given and out.requires_grad) or \
            (bias is not None and bias.requires_grad) or (residual is not None and residual.requires_grad):
        _no_gradient()
    if rows:
        ctx._lock.acquire()
        try:
            handle = _on_torch_stream(ctx)
            rc = _linear(handle, x.data_ptr(), ldx, weight.data_ptr(), ldw, b, res, ldr, out.data_ptr(), ldy, rows, co, ci,
                         flags, code)
            if rc:
                check(rc, handle)
        finally:
            ctx._lock.release()
    return out


class RotaryPositionEmbedder:
    """Rotary positions over the voxel axes x, y, z (columns 1..3 of the
    coordinates). Each axis takes pairs[a] of a head's head_dim / 2 pairs
    (default: a third each, rounded down), pair j of an axis turning by
    position * theta^(-j / pairs[a]), theta >= 1; the rest do not turn.
    layout: "pairs" (channels 2p, 2p + 1) or "halves" (channels p, p +
    head_dim / 2). A graph that captured a call with it needs it for as long as
    it is replayed."""

    def __init__(self, head_dim, pairs=None, theta=10000.0, layout="pairs", ctx=None):
        if layout not in _LAYOUTS:
            raise ValueError('RotaryPositionEmbedder: layout must be "pairs" or "halves"')
        self.head_dim, self.theta, self.layout = int(head_dim), float(theta), layout
        self.pairs = tuple(int(p) for p in pairs) if pairs is not None else (self.head_dim // 6,) * 3
        if len(self.pairs) != 3:
            raise ValueError("RotaryPositionEmbedder: pairs are three counts, of x, y and z")
        self.ctx = ctx or Context.default()
        h = ctypes.c_void_p()
        with self.ctx._lock:
            beside = self.ctx.beside_torch().handle
            check(lib.t2sc_rope_create(beside, self.head_dim, *self.pairs, self.theta, _LAYOUTS[layout], ctypes.byref(h)),
                  beside)
        self.handle = h

    def forward_device(self, x, coords, out=None):
        """x [rows, heads, head_dim] (rows may be strided), coords int32 [rows, 4]; out may be x."""
        ctx = self.ctx
        device, dtype = ctx.device, x.dtype
        code = _code(x, "RotaryPositionEmbedder: x")
        rows, heads, d, ldx = _heads3d(x, device, dtype, "RotaryPositionEmbedder: x")
        if d != self.head_dim or heads < 1:
            raise ValueError("RotaryPositionEmbedder: x must be [rows, heads, head_dim]")
        at = _coords(coords, device, rows)
        given = out is not None
        if not given:
            out, ldy = x.new_empty((rows, heads, d)), heads * d
        else:
            r, h, e, ldy = _heads3d(out, device, dtype, "RotaryPositionEmbedder: out")
            if (r, h, e) != (rows, heads, d):
                raise ValueError("RotaryPositionEmbedder: out must have x's shape")
        if x.requires_grad or (given and out.requires_grad):
            _no_gradient()
        if rows:
            ctx._lock.acquire()
            try:
                handle = _on_torch_stream(ctx)
                rc = _rope_apply(self.handle, at, x.data_ptr(), ldx, out.data_ptr(), ldy, rows, heads, code)
                if rc:
                    check(rc, handle)
            finally:
                ctx._lock.release()
        return out

    def __del__(self):
        h = getattr(self, "handle", None)
        if h and lib is not None:   # None: the interpreter is shutting down
            lib.t2sc_rope_destroy(h)
            self.handle = None


def qk_norm_rope_device(q, k, gain_q, gain_k, coords=None, rope=None, eps=1e-6, out_q=None, out_k=None, ctx=None):
    """RMS norm of every head of q and k with its own gains, then the rotation
    of `rope` (None: no rotation) at `coords`, in one pass. q, k [rows, heads,
    head_dim] (rows may be strided), gains float32 [heads, head_dim]. k None:
    q alone. out_q may be q and out_k k. Returns (out_q, out_k)."""
    ctx = rope.ctx if ctx is None and rope is not None else _context(ctx, q)
    device, dtype = ctx.device, q.dtype
    code = _code(q, "qk_norm_rope: q")
    rows, heads, d, ldq = _heads3d(q, device, dtype, "qk_norm_rope: q")
    if heads < 1 or (rope is not None and rope.head_dim != d):
        raise ValueError("qk_norm_rope: q must be [rows, heads, head_dim] with rope's head_dim")
    shape = (rows, heads, d)
    if out_q is None:
        out_q, ldqo = q.new_empty(shape), heads * d
    else:
        *got, ldqo = _heads3d(out_q, device, dtype, "qk_norm_rope: out_q")
        if tuple(got) != shape:
            raise ValueError("qk_norm_rope: out_q must have q's shape")
    gq = _f32(gain_q, device, (heads, d), "qk_norm_rope: gain_q")
    ldk = ldko = 0
    gk = kp = kop = None
    if k is not None:
        *got, ldk = _heads3d(k, device, dtype, "qk_norm_rope: k")
        if tuple(got) != shape:
            raise ValueError("qk_norm_rope: k must have q's shape")
        if out_k is None:
            out_k, ldko = q.new_empty(shape), heads * d
        else:
            *got, ldko = _heads3d(out_k, device, dtype, "qk_norm_rope: out_k")
            if tuple(got) != shape:
                raise ValueError("qk_norm_rope: out_k must have q's shape")
        gk = _f32(gain_k, device, (heads, d), "qk_norm_rope: gain_k")
        kp, kop = k.data_ptr(), out_k.data_ptr()
    elif out_k is not None:
        raise ValueError("qk_norm_rope: out_k without k")
    at = _coords(coords, device, rows) if rope is not None else None
    if q.requires_grad or gain_q.requires_grad or out_q.requires_grad or \
            (k is not None and (k.requires_grad or gain_k.requires_grad or out_k.requires_grad)):
        _no_gradient()
    if rows:
        ctx._lock.acquire()
        try:
            handle = _on_torch_stream(ctx)
            rc = _qk_norm_rope(handle, None if rope is None else rope.handle, at, q.data_ptr(), ldq, kp, ldk, gq, gk,
                               out_q.data_ptr(), ldqo, kop, ldko, rows, heads, d, eps, code)
            if rc:
                check(rc, handle)
        finally:
            ctx._lock.release()
    return out_q, out_k


class SequenceLayout:
    """The sequences of a ragged batch: lengths of each one's queries and of
    its keys (None: the same, self-attention). Built once for a set of
    coordinates (`of` a SparseTensor: one sequence per batch entry) and
    shared by every layer and step. A graph that captured its attention needs
    it for as long as it is replayed."""

    def __init__(self, q_lens, kv_lens=None, ctx=None):
        self.q_offsets = self._offsets(q_lens)
        self.kv_offsets = self.q_offsets if kv_lens is None else self._offsets(kv_lens)
        if len(self.q_offsets) != len(self.kv_offsets):
            raise ValueError("SequenceLayout: as many key lengths as query lengths")
        self.q_rows, self.kv_rows = int(self.q_offsets[-1]), int(self.kv_offsets[-1])
        self.ctx = ctx or Context.default()
        h = ctypes.c_void_p()
        with self.ctx._lock:
            beside = self.ctx.beside_torch().handle
            check(lib.t2sc_seqs_create(beside, self.q_offsets.ctypes.data, self.kv_offsets.ctypes.data,
                                       len(self.q_offsets) - 1, ctypes.byref(h)), beside)
        self.handle = h

    @classmethod
    def of(cls, x, kv_lens=None):
        """One sequence for each batch entry of a SparseTensor."""
        return cls(np.diff(x.offsets), kv_lens, ctx=x.ctx)

    @staticmethod
    def _offsets(lens):
        given = np.asarray(lens).reshape(-1)
        if given.size and given.dtype.kind not in "iu":
            raise ValueError("SequenceLayout: lengths must be whole numbers")
        lens = given.astype(np.int64)
        if len(lens) and lens.min() < 0:
            raise ValueError("SequenceLayout: lengths must not be negative")
        return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)

    def attention_device(self, q, k, v, scale=None, out=None):
        """softmax(scale * q k^T) v inside each sequence. q [rows, heads,
        head_dim] with the layout's query rows, k and v with its key rows
        (more rows may follow; they are left alone); rows may be strided.
        scale defaults to head_dim ** -0.5. out must not overlap an input."""
        ctx = self.ctx
        device, dtype = ctx.device, q.dtype
        code = _code(q, "attention: q")
        rows, heads, d, ldq = _heads3d(q, device, dtype, "attention: q")
        kv_rows, kh, kd, ldk = _heads3d(k, device, dtype, "attention: k")
        v_rows, vh, vd, ldv = _heads3d(v, device, dtype, "attention: v")
        if kh != heads or kd != d or (v_rows, vh, vd) != (kv_rows, kh, kd) or heads < 1 or d < 1:
            raise ValueError("attention: k and v must be [rows, heads, head_dim] with q's heads and head_dim")
        if rows < self.q_rows or kv_rows < self.kv_rows:
            raise ValueError("attention: fewer rows than the layout has")
        given = out is not None
        if not given:
            out, ldo = q.new_empty((rows, heads, d)), heads * d
        else:
            r, h, e, ldo = _heads3d(out, device, dtype, "attention: out")
            if (r, h, e) != (rows, heads, d):
                raise ValueError("attention: out must have q's shape")
        if q.requires_grad or k.requires_grad or v.requires_grad or (given and out.requires_grad):
            _no_gradient()
        ctx._lock.acquire()
        try:
            handle = _on_torch_stream(ctx)
            rc = _attention(self.handle, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo, heads, d,
                            d ** -0.5 if scale is None else scale, code)
            if rc:
                check(rc, handle)
        finally:
            ctx._lock.release()
        return out

    def __del__(self):
        h = getattr(self, "handle", None)
        if h and lib is not None:   # None: the interpreter is shutting down
            lib.t2sc_seqs_destroy(h)
            self.handle = None


def _tensor(a, dtype, device):
    return None if a is None else torch.from_numpy(np.array(a, np.float32)).to(device, dtype)


def _torch_dtype(dtype):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


class SparseMultiHeadAttention:
    """Self- or cross-attention of a SparseTensor's rows, inside each batch
    entry: projections, per-head RMS norm of q and k (qk_norm), rotary
    positions of the voxels (rope, self-attention only), attention, output
    projection (+ residual).

    Self-attention: to_qkv = (weight [3C, C], bias [3C]). Cross-attention
    (ctx_channels given): to_q = (weight [C, C], bias) and to_kv = (weight
    [2C, ctx_channels], bias). to_out = (weight [C, C], bias). gains =
    (gain_q, gain_k), each [heads, head_dim], or None for no norm (then no
    rotation either)."""

    def __init__(self, channels, heads, to_out, to_qkv=None, to_q=None, to_kv=None, gains=None, rope=None, eps=1e-6,
                 dtype="bf16", ctx=None):
        if channels % heads:
            raise ValueError("SparseMultiHeadAttention: channels must be a multiple of heads")
        if (to_qkv is None) == (to_q is None or to_kv is None):
            raise ValueError("SparseMultiHeadAttention: either to_qkv, or to_q and to_kv")
        if rope is not None and (gains is None or to_qkv is None):
            raise ValueError("SparseMultiHeadAttention: rotary positions go with self-attention and q/k gains")
        if dtype not in _DTYPES:
            raise ValueError("SparseMultiHeadAttention: dtype must be f32, f16 or bf16")
        self.ctx = ctx or Context.default()
        self.channels, self.heads, self.head_dim = channels, heads, channels // heads
        self.cross, self.rope, self.eps, self.dtype = to_qkv is None, rope, float(eps), dtype
        dev, dt = f"cuda:{self.ctx.device}", _torch_dtype(dtype)

        def pair(wb, co, ci=None):
            w, b = _tensor(wb[0], dt, dev), _tensor(wb[1], torch.float32, dev)
            if w.dim() != 2 or w.shape[0] != co or (ci is not None and w.shape[1] != ci) or \
                    (b is not None and tuple(b.shape) != (co,)):
                raise ValueError("SparseMultiHeadAttention: projection weights must be [out, in] with bias [out]")
            return w, b

        if self.cross:
            self._q, self._kv = pair(to_q, channels, channels), pair(to_kv, 2 * channels)
        else:
            self._qkv = pair(to_qkv, 3 * channels, channels)
        self._out = pair(to_out, channels, channels)
        self._gains = None
        if gains is not None:
            self._gains = tuple(_tensor(g, torch.float32, dev).reshape(heads, self.head_dim) for g in gains)

    def forward_device(self, x, layout, coords=None, context=None, residual=None):
        """x [rows, C] on the device; layout: the SequenceLayout of its rows
        (and the context's); coords int32 [rows, 4] where rope is set;
        context [context rows, ctx_channels] for cross-attention. Rows behind
        the layout's last are not given a meaning: pass none."""
        h, d, c = self.heads, self.head_dim, self.channels
        rows = x.shape[0]
        if rows != layout.q_rows:
            raise ValueError("SparseMultiHeadAttention: x must have the layout's rows")
        if not self.cross and layout.kv_offsets is not layout.q_offsets and \
                not np.array_equal(layout.kv_offsets, layout.q_offsets):
            raise ValueError("SparseMultiHeadAttention: self-attention needs a layout whose keys are its queries")
        if self.cross:
            if context is None:
                raise ValueError("SparseMultiHeadAttention: cross-attention needs a context")
            if context.shape[0] != layout.kv_rows:
                raise ValueError("SparseMultiHeadAttention: context must have the layout's key rows")
            q = dense_linear_device(x, *self._q, ctx=self.ctx).view(rows, h, d)
            kv = dense_linear_device(context, *self._kv, ctx=self.ctx).view(context.shape[0], 2, h, d)
            k, v = kv[:, 0], kv[:, 1]
            if self._gains:
                qk_norm_rope_device(q, None, self._gains[0], None, eps=self.eps, out_q=q, ctx=self.ctx)
                qk_norm_rope_device(k, None, self._gains[1], None, eps=self.eps, out_q=k, ctx=self.ctx)
        else:
            if context is not None:
                raise ValueError("SparseMultiHeadAttention: a context, but no to_q and to_kv")
            qkv = dense_linear_device(x, *self._qkv, ctx=self.ctx).view(rows, 3, h, d)
            q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
            if self._gains:
                qk_norm_rope_device(q, k, *self._gains, coords=coords, rope=self.rope, eps=self.eps, out_q=q, out_k=k,
                                    ctx=self.ctx)
        a = layout.attention_device(q, k, v)
        return dense_linear_device(a.view(rows, c), *self._out, residual=residual, ctx=self.ctx)

    def forward(self, x, context=None, context_lens=None, residual=False):
        """x: SparseTensor; context: host f32 [rows, ctx_channels] with
        context_lens rows of it for each batch entry. residual: add x."""
        dev, dt = f"cuda:{self.ctx.device}", _torch_dtype(self.dtype)
        xd = _tensor(x.feats, dt, dev)
        if self.cross and context_lens is None:
            raise ValueError("SparseMultiHeadAttention: cross-attention needs context_lens")
        layout = SequenceLayout(np.diff(x.offsets), context_lens if self.cross else None, ctx=self.ctx)
        coords = torch.from_numpy(x.coords).to(dev) if self.rope is not None else None
        y = self.forward_device(xd, layout, coords, _tensor(context, dt, dev), xd if residual else None)
        y = y.float().cpu().numpy()
        self.ctx.synchronize()
        return x.replace(y)

    __call__ = forward


class SparseFeedForwardNet:
    """lin2(GELU(lin1(x))) (+ residual) over rows: lin1 = (weight [H, C], bias
    [H]), lin2 = (weight [C, H], bias [C])."""

    def __init__(self, lin1, lin2, activation="gelu", dtype="bf16", ctx=None):
        if activation not in _ACTIVATIONS:
            raise ValueError('SparseFeedForwardNet: activation must be None, "silu" or "gelu"')
        if dtype not in _DTYPES:
            raise ValueError("SparseFeedForwardNet: dtype must be f32, f16 or bf16")
        self.ctx = ctx or Context.default()
        self.activation, self.dtype = activation, dtype
        dev, dt = f"cuda:{self.ctx.device}", _torch_dtype(dtype)
        self._lin1 = _tensor(lin1[0], dt, dev), _tensor(lin1[1], torch.float32, dev)
        self._lin2 = _tensor(lin2[0], dt, dev), _tensor(lin2[1], torch.float32, dev)

    def forward_device(self, x, residual=None):
        h = dense_linear_device(x, *self._lin1, activation=self.activation, ctx=self.ctx)
        return dense_linear_device(h, *self._lin2, residual=residual, ctx=self.ctx)

    def forward(self, x, residual=False):
        """x: SparseTensor or host f32 [rows, C]; residual: add x."""
        st = x if isinstance(x, SparseTensor) else None
        xd = _tensor(st.feats if st is not None else x, _torch_dtype(self.dtype), f"cuda:{self.ctx.device}")
        y = self.forward_device(xd, xd if residual else None).float().cpu().numpy()
        self.ctx.synchronize()
        return st.replace(y) if st is not None else y

    __call__ = forward
