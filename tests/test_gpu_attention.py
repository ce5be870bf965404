"""The attention-block operators on the GPU against their plain 64-bit forms
(_attention_ref.py, which derives the bounds), at the sizes, strides and
lengths where tiles end, and the block made of them."""
import ctypes

import numpy as np
import pytest

import _attention_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16", "float32"]
NAN = float("nan")


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype="float32"):
    import torch
    return (torch.randn(shape, generator=g, device="cuda") * std).to(getattr(torch, dtype))


def _inside(rows, width, dtype, pad_rows=3, pad_cols=8, fill=NAN):
    """A [rows, width] view into a larger buffer filled with `fill`, and the buffer."""
    import torch
    buf = torch.full((rows + pad_rows, width + pad_cols), fill, device="cuda", dtype=getattr(torch, dtype))
    return buf[:rows, :width], buf


def _untouched(buf, rows, width):
    import torch
    return torch.isnan(buf[rows:]).all() and torch.isnan(buf[:, width:]).all()


# ---- dense linear ----

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ci,co", [(1, 8, 8), (1, 1536, 264), (2, 64, 7), (5, 200, 64), (8, 72, 129), (9, 512, 96),
                                        (17, 1024, 512), (64, 40, 200), (127, 64, 64), (128, 128, 256), (129, 136, 257),
                                        (300, 328, 520), (1000, 64, 24)])
def test_linear_shapes(t2sc, dtype, rows, ci, co):
    g = _gen(rows * 7 + ci + co)
    x, w = _normal(g, rows, ci, dtype=dtype), _normal(g, co, ci, std=ci ** -0.5, dtype=dtype)
    b = _normal(g, co, std=0.5)
    out, buf = _inside(rows, co, dtype)
    y = t2sc.dense_linear_device(x, w, b, out=out)
    assert y is out and _untouched(buf, rows, co)
    ref.assert_close(y, *ref.linear(x, w, b))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("rows,ci,co", [(3, 96, 80), (200, 96, 80)])
def test_linear_epilogue(t2sc, dtype, act, rows, ci, co):
    g = _gen(3)
    x, w = _normal(g, rows, ci, std=3.0, dtype=dtype), _normal(g, co, ci, std=ci ** -0.5, dtype=dtype)
    b, r = _normal(g, co, std=2.0), _normal(g, rows, co, dtype=dtype)
    for bias in (b, None):
        for res in (r, None):
            y = t2sc.dense_linear_device(x, w, bias, activation=act, residual=res)
            ref.assert_close(y, *ref.linear(x, w, bias, act, res))


def test_linear_saturated_activations(t2sc):
    """Pre-activations far out on both sides: zeros and the value itself, no NaN."""
    import torch
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.tensor([[-1e4], [-300.0], [-90.0], [90.0], [300.0], [1e4]], device="cuda", dtype=dtype).repeat(1, 8)
        w = torch.zeros(8, 8, device="cuda", dtype=dtype)
        w[:, 0] = 1
        for act in ("silu", "gelu"):
            ref.assert_close(t2sc.dense_linear_device(x, w, activation=act), *ref.linear(x, w, None, act))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 6, 33, 260])
def test_linear_strided_and_in_place(t2sc, dtype, rows):
    """x a slice of a packed buffer with NaN around it, w a slice of a wider one, y = residual in place."""
    g = _gen(11)
    xv, _ = _inside(rows, 256, dtype)
    wv, _ = _inside(136, 256, dtype)
    xv.copy_(_normal(g, rows, 256, dtype=dtype))
    wv.copy_(_normal(g, 136, 256, std=1 / 16, dtype=dtype))
    rv, buf = _inside(rows, 136, dtype, pad_cols=16)
    rv.copy_(_normal(g, rows, 136, dtype=dtype))
    want = ref.linear(xv, wv, None, "gelu", rv.clone())
    y = t2sc.dense_linear_device(xv, wv, activation="gelu", residual=rv, out=rv)
    assert y is rv and _untouched(buf, rows, 136)
    ref.assert_close(y, *want)


@pytest.mark.parametrize("shift_x,shift_w,shift_y,ci", [(1, 0, 0, 64), (0, 1, 0, 64), (0, 0, 1, 64), (0, 0, 0, 61), (4, 4, 4, 64)])
@pytest.mark.parametrize("rows", [3, 150])
def test_linear_unaligned(t2sc, shift_x, shift_w, shift_y, ci, rows):
    """Bases off 16 bytes and odd row widths."""
    import torch
    g = _gen(5)

    def at(n, width, shift, std):
        flat = torch.empty(n * width + 8, device="cuda", dtype=torch.bfloat16)[shift:shift + n * width].view(n, width)
        return flat.copy_(_normal(g, n, width, std=std))

    x, w = at(rows, ci, shift_x, 1.0), at(48, ci, shift_w, ci ** -0.5)
    out = at(rows, 48, shift_y, 0.0)
    ref.assert_close(t2sc.dense_linear_device(x, w, out=out), *ref.linear(x, w))


@pytest.mark.parametrize("rows,ci,co", [(1, 4096, 1024), (2, 1000, 517), (3, 4096, 1024), (4, 1024, 4608), (17, 2000, 300), (40, 4096, 1024),
                                        (64, 4096, 130), (100, 1040, 777), (128, 8192, 128), (1941, 1536, 768), (2500, 512, 2304)])
def test_linear_larger(t2sc, rows, ci, co):
    g = _gen(9)
    x, w, b = _normal(g, rows, ci, dtype="bfloat16"), _normal(g, co, ci, std=ci ** -0.5, dtype="bfloat16"), _normal(g, co)
    y = t2sc.dense_linear_device(x, w, b, activation="silu")
    ref.assert_close(y, *ref.linear(x, w, b, "silu"))
    import torch
    assert torch.equal(y, t2sc.dense_linear_device(x, w, b, activation="silu"))   # no order-dependent sums


def test_linear_long_rows_offset(t2sc):
    """Rows far enough apart that element offsets pass 2^31."""
    import torch
    g = _gen(13)
    rows, stride = 2200, 1 << 20
    big = torch.empty(rows * stride, device="cuda", dtype=torch.bfloat16)
    x, y = big.view(rows, stride)[:, :64], big.view(rows, stride)[:, 128:192]
    x.copy_(_normal(g, rows, 64))
    w = _normal(g, 64, 64, std=1 / 8, dtype="bfloat16")
    t2sc.dense_linear_device(x, w, out=y)
    ref.assert_close(y, *ref.linear(x, w))


# ---- rotary positions, norm + rotation ----

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("rows,heads,d,pairs", [(1, 1, 2, (1, 0, 0)), (3, 2, 6, None), (257, 12, 128, None), (130, 16, 64, None),
                                                (77, 5, 80, (3, 17, 20)), (33, 24, 96, (0, 48, 0)), (9, 3, 40, None),
                                                (65, 1, 256, None), (19, 40, 32, (0, 0, 0)), (21, 7, 72, (36, 0, 0))])
def test_rope(t2sc, dtype, layout, rows, heads, d, pairs):
    import torch
    g = _gen(d + rows)
    x = _normal(g, rows, heads, d, dtype=dtype)
    coords = torch.randint(-512, 1536, (rows, 4), generator=g, device="cuda", dtype=torch.int32)
    emb = t2sc.RotaryPositionEmbedder(d, pairs, theta=10000.0, layout=layout)
    y = emb.forward_device(x, coords)
    want = ref.rope(x, coords, emb.pairs, 10000.0, layout)
    ref.assert_close(y, *want)
    keep = x.clone()
    assert emb.forward_device(x, coords, out=x) is x and torch.equal(x, y)   # in place
    packed = torch.full((rows, 3, heads, d), NAN, device="cuda", dtype=x.dtype)
    packed[:, 1] = keep
    out = packed[:, 2]
    emb.forward_device(packed[:, 1], coords, out=out)   # one slice of a packed buffer into another
    assert torch.equal(out, y) and torch.isnan(packed[:, 0]).all() and torch.equal(packed[:, 1], keep)


def test_rope_far_positions(t2sc):
    """Any int32 position turns by its exact angle."""
    import torch
    g = _gen(1)
    x = _normal(g, 6, 2, 12)
    coords = torch.tensor([[0, v, -v, v // 3] for v in (0, 1, 10 ** 6, 2 ** 30, 2 ** 31 - 1, -2 ** 31 + 1)], device="cuda",
                          dtype=torch.int32)
    emb = t2sc.RotaryPositionEmbedder(12)
    # at 2^31 a 64-bit angle in turns is itself off by 2^31 * 2^-53 * 2 pi * 2 < 2^-18
    want, tol = ref.rope(x, coords, emb.pairs, 10000.0, "pairs")
    ref.assert_close(emb.forward_device(x, coords), want, tol + 2.0 ** -18 * x.abs().max().item())


def test_rope_leaves_unturned_channels(t2sc):
    """Channels without an axis pass through exactly, infinities and NaN too, and stay apart from the others."""
    import torch
    x = torch.ones(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    x[:, :, 62], x[:, :, 63] = float("inf"), NAN
    coords = torch.full((4, 4), 7, device="cuda", dtype=torch.int32)
    y = t2sc.RotaryPositionEmbedder(64).forward_device(x, coords)
    assert torch.equal(y[:, :, 60:63], x[:, :, 60:63]) and torch.isnan(y[:, :, 63]).all()
    assert torch.isfinite(y[:, :, :60]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("rows,heads,d", [(1, 1, 8), (300, 12, 128), (131, 16, 64), (70, 24, 96), (41, 3, 80), (13, 5, 36), (5, 2, 256)])
def test_qk_norm_rope(t2sc, dtype, layout, rows, heads, d):
    import torch
    g = _gen(d * 3 + rows)
    qkv = _normal(g, rows, 3, heads, d, std=1.7, dtype=dtype)
    qkv[rows // 2, 0] *= 1e-3          # a row near eps
    qkv[rows // 2, 1] = 0              # a row of zeros stays zero
    gq, gk = 1 + _normal(g, heads, d, std=0.3), _normal(g, heads, d)
    coords = torch.randint(0, 1024, (rows, 4), generator=g, device="cuda", dtype=torch.int32)
    emb = t2sc.RotaryPositionEmbedder(d, layout=layout)
    q, k = qkv[:, 0], qkv[:, 1]
    want = [ref.rope(t, coords, emb.pairs, 10000.0, layout, gain, 1e-6) for t, gain in ((q, gq), (k, gk))]
    oq, ok = t2sc.qk_norm_rope_device(q, k, gq, gk, coords, emb, eps=1e-6)
    ref.assert_close(oq, *want[0])
    ref.assert_close(ok, *want[1])
    assert (ok[rows // 2] == 0).all()
    alone, none = t2sc.qk_norm_rope_device(q, None, gq, None, coords, emb, eps=1e-6)
    assert none is None and torch.equal(alone, oq)
    plain, _ = t2sc.qk_norm_rope_device(q, None, gq, None, eps=1e-6)      # no rotation
    ref.assert_close(plain, *ref.rope(q, coords, (0, 0, 0), 1.0, layout, gq, 1e-6))
    v = qkv[:, 2].clone()
    t2sc.qk_norm_rope_device(q, k, gq, gk, coords, emb, eps=1e-6, out_q=q, out_k=k)   # in place in the packed buffer
    assert torch.equal(q, oq) and torch.equal(k, ok) and torch.equal(qkv[:, 2], v)


# ---- attention ----

LENGTHS = [([2, 1, 0, 2], [700, 0, 5, 129]), ([4, 3, 1], [9000, 1, 64]), ([1, 1], [5000, 20000]), ([8, 5], [2100, 77]), ([1], [1]), ([1], [300]), ([3], [2048]), ([17], [0]), ([64], [64]), ([127], [129]), ([128], [128]), ([129], [127]),
           ([255, 1, 0, 300], [255, 1, 0, 300]), ([5, 0, 200, 40], [0, 77, 1, 513]), ([700], [1029]), ([256, 257], [1, 640])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,kv_lens", LENGTHS)
@pytest.mark.parametrize("heads,d", [(2, 64), (3, 128)])
def test_attention_lengths(t2sc, dtype, q_lens, kv_lens, heads, d):
    import torch
    g = _gen(sum(q_lens) + d)
    q = _normal(g, sum(q_lens), heads, d, std=1.5, dtype=dtype)
    k, v = _normal(g, sum(kv_lens), heads, d, std=1.5, dtype=dtype), _normal(g, sum(kv_lens), heads, d, dtype=dtype)
    layout = t2sc.SequenceLayout(q_lens, kv_lens)
    y = layout.attention_device(q, k, v)
    ref.assert_close(y, *ref.attention(q, k, v, q_lens, kv_lens, d ** -0.5))
    assert torch.equal(y, layout.attention_device(q, k, v))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 72, 80, 96, 104, 120, 136, 256, 7, 33])
def test_attention_head_dims(t2sc, dtype, d):
    g = _gen(d)
    lens = [130, 1, 77]
    q, k, v = (_normal(g, sum(lens), 2, d, dtype=dtype) for _ in range(3))
    y = t2sc.SequenceLayout(lens).attention_device(q, k, v, scale=0.21)
    ref.assert_close(y, *ref.attention(q, k, v, lens, lens, 0.21))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("q_lens,kv_lens", [([150, 90], [200, 61]), ([2, 1], [900, 333])])
def test_attention_packed_and_bounded(t2sc, dtype, q_lens, kv_lens):
    """q and packed k, v with NaN and infinities in every row and column that
    belongs to no sequence: neither read into a result nor written."""
    import torch
    g = _gen(21)
    h, d = 3, 64
    nq, nk = sum(q_lens), sum(kv_lens)
    tdt = getattr(torch, dtype)
    qb = torch.full((nq + 40, h * d + 24), NAN, device="cuda", dtype=tdt)
    kvb = torch.full((nk + 300, 3, h, d), float("inf"), device="cuda", dtype=tdt)
    ob = torch.full((nq + 40, h * d + 8), NAN, device="cuda", dtype=tdt)
    q, out = qb[:, :h * d].unflatten(1, (h, d)), ob[:, :h * d].unflatten(1, (h, d))
    q[:nq] = _normal(g, nq, h, d, dtype=dtype)
    k, v = kvb[:, 0], kvb[:, 2]
    k[:nk], v[:nk] = _normal(g, nk, h, d, dtype=dtype), _normal(g, nk, h, d, dtype=dtype)
    t2sc.SequenceLayout(q_lens, kv_lens).attention_device(q, k, v, out=out)
    assert _untouched(ob, nq, h * d)
    ref.assert_close(out[:nq], *ref.attention(q[:nq], k[:nk], v[:nk], q_lens, kv_lens, d ** -0.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")])
@pytest.mark.parametrize("q_len", [3, 140])
def test_attention_bad_values_stay_in_their_sequence(t2sc, dtype, bad, q_len):
    """What one sequence holds never reaches another's rows."""
    import torch
    g = _gen(4)
    lens_q, lens_k = [q_len, q_len, q_len], [100, 156, 37]
    q, k, v = (_normal(g, n, 2, 64, dtype=dtype) for n in (sum(lens_q), sum(lens_k), sum(lens_k)))
    want = ref.attention(q, k, v, lens_q, lens_k, 0.125)
    q[q_len:2 * q_len], k[100:256], v[100:256] = bad, bad, bad
    y = t2sc.SequenceLayout(lens_q, lens_k).attention_device(q, k, v)
    for rows in (slice(0, q_len), slice(2 * q_len, None)):
        ref.assert_close(y[rows], want[0][rows], want[1][rows])
    assert not torch.isfinite(y[q_len:2 * q_len]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,kv_len", [(2, 1500), (150, 1500)])
def test_attention_rising_and_peaked_scores(t2sc, dtype, q_len, kv_len):
    """The running maximum moves in every block of keys, up to scores of a
    few hundred; one key takes nearly all the weight of its row."""
    import torch
    g = _gen(8)
    d = 64
    q, k, v = (_normal(g, n, 1, d, dtype=dtype) for n in (q_len, kv_len, kv_len))
    q[:] = 1
    k[:] = (torch.linspace(-6, 6, kv_len, device="cuda")[:, None, None] + 0.1 * k.float()).to(k.dtype)
    y = t2sc.SequenceLayout([q_len], [kv_len]).attention_device(q, k, v, scale=1.0)
    ref.assert_close(y, *ref.attention(q, k, v, [q_len], [kv_len], 1.0))
    k = k.flip(0).contiguous()   # falling: all later keys weigh next to nothing
    y = t2sc.SequenceLayout([q_len], [kv_len]).attention_device(q, k, v, scale=1.0)
    ref.assert_close(y, *ref.attention(q, k, v, [q_len], [kv_len], 1.0))


@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
@pytest.mark.parametrize("q_len", [1, 130])
def test_attention_scales(t2sc, scale, q_len):
    g = _gen(6)
    q, k, v = (_normal(g, n, 2, 64, dtype="bfloat16") for n in (q_len, 300, 300))
    y = t2sc.SequenceLayout([q_len], [300]).attention_device(q, k, v, scale=scale)
    ref.assert_close(y, *ref.attention(q, k, v, [q_len], [300], scale))


@pytest.mark.parametrize("q_len", [1, 129])
def test_attention_long_offsets(t2sc, q_len):
    """Key rows whose element offsets pass 2^31."""
    import torch
    g = _gen(2)
    n, stride, h, d = 2300, 1 << 20, 2, 64
    big = torch.empty(n * stride, device="cuda", dtype=torch.bfloat16).view(n, stride)
    k, v = big[:, :h * d].unflatten(1, (h, d)), big[:, 256:256 + h * d].unflatten(1, (h, d))
    k.copy_(_normal(g, n, h, d))
    v.copy_(_normal(g, n, h, d))
    q = _normal(g, q_len, h, d, dtype="bfloat16")
    y = t2sc.SequenceLayout([q_len], [n]).attention_device(q, k, v)
    ref.assert_close(y, *ref.attention(q, k, v, [q_len], [n], d ** -0.5))


def test_attention_first_offset_above_zero(t2sc):
    """Through the C ABI: sequences that start behind row 0 leave the rows before them alone."""
    import torch
    g = _gen(12)
    h, d, dt = 2, 64, t2sc._lib.DT_BF16
    ctx = t2sc.Context.default(0)
    q, k, v = (_normal(g, n, h, d, dtype="bfloat16") for n in (240, 190, 190))
    for q_off, kv_off in (([20, 170, 200], [30, 130, 180]), ([3, 5, 6], [30, 130, 180])):
        out = torch.full_like(q, NAN)
        off = [np.array(o, np.int64) for o in (q_off, kv_off)]
        seqs = ctypes.c_void_p()
        t2sc._lib.check(t2sc.lib.t2sc_seqs_create(ctx.handle, off[0].ctypes.data, off[1].ctypes.data, 2, ctypes.byref(seqs)),
                        ctx.handle)
        torch.cuda.synchronize()
        t2sc._lib.check(t2sc.lib.t2sc_attention_device(seqs, q.data_ptr(), h * d, k.data_ptr(), h * d, v.data_ptr(), h * d,
                                                       out.data_ptr(), h * d, h, d, 0.125, dt), ctx.handle)
        ctx.synchronize()
        t2sc.lib.t2sc_seqs_destroy(seqs)
        a, b = q_off[0], q_off[-1]
        assert torch.isnan(out[:a]).all() and torch.isnan(out[b:]).all()
        ql, kl = np.diff(q_off).tolist(), np.diff(kv_off).tolist()
        ref.assert_close(out[a:b], *ref.attention(q[a:b], k[kv_off[0]:], v[kv_off[0]:], ql, kl, 0.125))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_very_many_sequences(t2sc, dtype):
    """100,000 sequences of none to four tokens: finding a block's sequence stays cheap."""
    import torch
    g = _gen(34)
    lens = np.random.default_rng(6).integers(0, 5, 100000)
    q, k, v = (_normal(g, int(lens.sum()), 1, 16, dtype=dtype) for _ in range(3))
    y = t2sc.SequenceLayout(lens).attention_device(q, k, v)
    # tokens of sequences of one get their own v; a sample of the others against the formula
    off = np.concatenate([[0], np.cumsum(lens)])
    ones = torch.from_numpy(off[:-1][lens == 1]).cuda()
    assert torch.equal(y[ones], v[ones])
    for b in np.nonzero(lens > 1)[0][::9973]:
        r = slice(int(off[b]), int(off[b + 1]))
        ref.assert_close(y[r], *ref.attention(q[r], k[r], v[r], [int(lens[b])], [int(lens[b])], 0.25))


def test_attention_many_sequences(t2sc):
    """More sequences than SMs, most of them short, some empty."""
    g = _gen(33)
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 40, 700)]
    lens[350] = 1500
    q, k, v = (_normal(g, sum(lens), 2, 64, dtype="bfloat16") for _ in range(3))
    y = t2sc.SequenceLayout(lens).attention_device(q, k, v)
    ref.assert_close(y, *ref.attention(q, k, v, lens, lens, 0.125))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("d", [128, 96, 64, 40])
def test_attention_two_blocks_a_cta(t2sc, dtype, d):
    """Enough heads that a CTA takes 256 queries: with one block, two blocks
    and a part of the second, keys from none to many blocks."""
    g = _gen(60 + d)
    q_lens, kv_lens = [700, 1, 0, 257, 128, 30], [650, 700, 90, 3, 129, 0]
    q, k, v = (_normal(g, n, 40, d, dtype=dtype) for n in (sum(q_lens), sum(kv_lens), sum(kv_lens)))
    y = t2sc.SequenceLayout(q_lens, kv_lens).attention_device(q, k, v)
    ref.assert_close(y, *ref.attention(q, k, v, q_lens, kv_lens, d ** -0.5))


# ---- how they are called ----

def _block(t2sc, dtype, c=128, heads=2, hidden=384, cross=None, seed=50, ctx=None):
    S = t2sc.synth
    d = c // heads
    w = lambda i, co, ci: (S.normal(seed + i, (co, ci)) * ci ** -0.5, S.normal(seed + i + 1, (co,), std=0.1))  # noqa: E731
    rope = None if cross else t2sc.RotaryPositionEmbedder(d, ctx=ctx)
    gains = (1 + 0.2 * S.normal(seed + 20, (heads, d)), 1 + 0.2 * S.normal(seed + 21, (heads, d)))
    proj = dict(to_q=w(0, c, c), to_kv=w(2, 2 * c, cross)) if cross else dict(to_qkv=w(0, 3 * c, c))
    attn = t2sc.SparseMultiHeadAttention(c, heads, w(4, c, c), gains=gains, rope=rope, dtype=dtype, ctx=ctx, **proj)
    ffn = t2sc.SparseFeedForwardNet(w(6, hidden, c), w(8, c, hidden), dtype=dtype, ctx=ctx)
    return attn, ffn, gains, proj, w(4, c, c), w(6, hidden, c), w(8, c, hidden)


def _block_ref(x, coords, lens, heads, gains, proj, to_out, lin1, lin2, context=None, context_lens=None):
    """The block in 64 bits without intermediate roundings."""
    import torch
    t = lambda a: torch.from_numpy(np.asarray(a, np.float64)).cuda()  # noqa: E731
    lin = lambda h, wb: h @ t(wb[0]).T + t(wb[1])  # noqa: E731
    x = t(x)
    n, c = x.shape
    d = c // heads
    if context is None:
        qkv = lin(x, proj["to_qkv"]).view(n, 3, heads, d)
        q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
        pairs = (d // 6,) * 3
    else:
        kv = lin(t(context), proj["to_kv"]).view(-1, 2, heads, d)
        q, k, v = lin(x, proj["to_q"]).view(n, heads, d), kv[:, 0], kv[:, 1]
        pairs = (0, 0, 0)
    cq = torch.from_numpy(coords).cuda()
    ck = cq if context is None else torch.zeros(len(k), 4, device="cuda", dtype=torch.int32)
    q = _rope64(q, cq, pairs, t(gains[0]))
    k = _rope64(k, ck, pairs, t(gains[1]))
    out, q0, k0 = [], 0, 0
    for a, b in zip(lens, context_lens or lens):
        s = torch.einsum("ihd,jhd->hij", q[q0:q0 + a], k[k0:k0 + b]) * d ** -0.5
        out.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[k0:k0 + b]))
        q0, k0 = q0 + a, k0 + b
    h = x + lin(torch.cat(out).reshape(n, c), to_out)
    return (h + lin(torch.nn.functional.gelu(lin(h, lin1), approximate="tanh"), lin2)).cpu().numpy()


def _rope64(x, coords, pairs, gain):
    import torch
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain
    n = pairs[0]
    if n == 0:
        return x
    f = 10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
    ang = (coords[:, 1:, None].double() * f).reshape(len(x), 1, 3 * n)
    z = torch.view_as_complex(x[..., :6 * n].contiguous().view(*x.shape[:2], 3 * n, 2)) * torch.polar(torch.ones_like(ang), ang)
    return torch.cat((torch.view_as_real(z).flatten(-2), x[..., 6 * n:]), -1)


@pytest.mark.parametrize("dtype,tol", [("bf16", 3 * 2.0 ** -8), ("f16", 3 * 2.0 ** -11), ("f32", 1e-5)])
@pytest.mark.parametrize("cross", [None, 72])
def test_block_end_to_end(t2sc, dtype, tol, cross):
    """Attention + residual, then feed-forward + residual over a SparseTensor
    of two shapes. Seven roundings to the type lie in a row on the way to an
    output (x, qkv, q/k, weights of v, a, h, hidden), each off by at most u =
    2^-8 or 2^-11 relative to values of the output's order, evenly spread:
    u / sqrt(3) each in the 2-norm, sqrt(7 / 3) u = 1.5 u together, and as much
    again for the five weight matrices, which are rounded too: 3 u. f32: sums
    of at most 400 products, 400 * 2^-24 * (sum |x w| / |sum x w| of about
    0.4) = 1e-5."""
    S = t2sc.synth
    shells = [S.shell(32, 12.0, 0.6), S.shell(32, 9.0, 0.5, seed=1)]
    shells[1][:, 0] = 1
    coords = np.concatenate(shells)
    lens = [len(s) for s in shells]
    x = S.normal(1, (sum(lens), 128))
    attn, ffn, gains, proj, to_out, lin1, lin2 = _block(t2sc, dtype, cross=cross)
    ctx_lens = [70, 33]
    context = S.normal(2, (sum(ctx_lens), cross)) if cross else None
    st = t2sc.SparseTensor(x, coords)
    h = attn.forward(st, context, ctx_lens if cross else None, residual=True)
    y = ffn.forward(h, residual=True).feats
    want = _block_ref(x, coords, lens, 2, gains, proj, to_out, lin1, lin2, context, ctx_lens if cross else None)
    assert np.linalg.norm(y - want) <= tol * np.linalg.norm(want)


def _chain(t2sc, attn, ffn, layout, x, coords):
    return ffn.forward_device(*(2 * (attn.forward_device(x, layout, coords, residual=x),)))


def test_block_in_a_graph_and_on_streams(t2sc):
    """The block captured and replayed on new inputs, two graphs replayed on
    two streams, and a side stream: the same bits as eager."""
    import torch
    attn, ffn, *_ = _block(t2sc, "bf16")
    g = _gen(70)
    lens = [300, 5, 41]
    layout = t2sc.SequenceLayout(lens)
    few = t2sc.SequenceLayout([1, 2], [200, 146])
    coords = torch.randint(0, 64, (sum(lens), 4), generator=g, device="cuda", dtype=torch.int32)
    xs = [_normal(g, sum(lens), 128, dtype="bfloat16") for _ in range(3)]
    kv = [_normal(g, sum(lens), 2, 64, dtype="bfloat16") for _ in range(2)]

    def both(x):
        y = _chain(t2sc, attn, ffn, layout, x, coords)
        return y, few.attention_device(y[:3].unflatten(1, (2, 64)), kv[0], kv[1])

    eager = [[t.clone() for t in both(x)] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = both(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, eager[0]))
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = both(x)
        graphs.append((graph, x, y))
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(4):
        for i, ((graph, x, y), st) in enumerate(zip(graphs, streams)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                x.copy_(xs[(rep + i) % 3])
                graph.replay()
        torch.cuda.synchronize()
        for i, (graph, x, y) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(y, eager[(rep + i) % 3]))
    assert all(torch.equal(a, b) for a, b in zip(both(xs[1]), eager[1]))   # eager again after the captures
    t2sc.Context.default(0).synchronize()


def test_two_contexts(t2sc):
    """A second context of the device with its own handles, interleaved with the first."""
    import torch
    c2 = t2sc.Context(0)
    g = _gen(80)
    lens = [150, 33]
    q, k, v = (_normal(g, sum(lens), 2, 64, dtype="float16") for _ in range(3))
    l1, l2 = t2sc.SequenceLayout(lens), t2sc.SequenceLayout(lens, ctx=c2)
    ys = [l.attention_device(q, k, v) for l in (l1, l2, l1, l2)]
    assert all(torch.equal(y, ys[0]) for y in ys)
    del l2
    c2.synchronize()
    c2.close()


# ---- refusals that need device tensors ----

def test_refusals(t2sc):
    import torch
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, device="cuda", dtype=dt)  # noqa: E731
    x, w = z(8, 64), z(16, 64)
    lin = t2sc.dense_linear_device
    emb = t2sc.RotaryPositionEmbedder(64)
    coords = z(8, 4, dt=torch.int32)
    q = z(8, 2, 64)
    layout = t2sc.SequenceLayout([8])
    gain = z(2, 64, dt=torch.float32)
    packed = z(10, 2, 2, 64)
    bad = [
        lambda: lin(x, z(16, 56)), lambda: lin(x, z(16, 64, dt=torch.float16)), lambda: lin(x, w, activation="relu"),
        lambda: lin(x, w, z(16)), lambda: lin(x, w, residual=z(8, 15)), lambda: lin(x, w, out=z(7, 16)),
        lambda: lin(x, w.cpu()), lambda: lin(x.cpu(), w), lambda: lin(x.t(), w), lambda: lin(z(8, 64, dt=torch.int16), w),
        lambda: lin(x[:, :16], z(16, 16), out=x[:, 8:24]),                      # y overlaps x
        lambda: lin(x, w, out=w[:8, :16]),                                       # y overlaps w
        lambda: lin(x[:1].expand(8, 64), w),                                     # rows that share memory
        lambda: emb.forward_device(z(8, 2, 32), coords), lambda: emb.forward_device(q, z(7, 4, dt=torch.int32)),
        lambda: emb.forward_device(q, z(8, 4, dt=torch.int64)), lambda: emb.forward_device(q.transpose(0, 1), coords),
        lambda: emb.forward_device(packed.view(-1)[:1024].view(8, 2, 64), coords,
                                   out=packed.view(-1)[64:1088].view(8, 2, 64)),   # half over the input
        lambda: t2sc.qk_norm_rope_device(q, q, gain, gain, coords, emb, eps=0.0),
        lambda: t2sc.qk_norm_rope_device(q, z(8, 2, 64), gain, gain, coords, emb, out_q=q, out_k=q),
        lambda: t2sc.qk_norm_rope_device(q, None, gain[:1], None, coords, emb),
        lambda: t2sc.qk_norm_rope_device(q, None, gain, None, None, emb),
        lambda: layout.attention_device(q[:7], q, q), lambda: layout.attention_device(q, q[:7], q[:7]),
        lambda: layout.attention_device(q, q, z(8, 2, 32)), lambda: layout.attention_device(q, q, q, out=q),
        lambda: layout.attention_device(q, q, q, scale=NAN), lambda: layout.attention_device(q, q, q.half()),
        lambda: layout.attention_device(z(8, 1, 264), z(8, 1, 264), z(8, 1, 264)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, AttributeError, t2sc.T2SCError)):
            call()
            print("not refused:", i)
    # and nothing of it broke the context; empty calls are fine
    assert lin(z(0, 64), w).shape == (0, 16)
    assert emb.forward_device(z(0, 2, 64), z(0, 4, dt=torch.int32)).shape == (0, 2, 64)
    assert t2sc.SequenceLayout([]).attention_device(z(0, 2, 64), z(0, 2, 64), z(0, 2, 64)).shape == (0, 2, 64)
    assert t2sc.SequenceLayout([3, 2], [0, 0]).attention_device(q, q[:0], q[:0])[:5].abs().max().item() == 0
    t2sc.Context.default(0).synchronize()


# ---- calls at the edges of what is allowed ----

@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows", [1, 5, 150])
def test_linear_activations_of_huge_values(t2sc, dtype, rows):
    """SiLU and GELU go to 0 on the left and to the value on the right, however far out."""
    import torch
    dt = getattr(torch, dtype)
    x = torch.zeros(rows, 16, device="cuda", dtype=dt)
    x[:, 0] = 1
    w = torch.zeros(8, 16, device="cuda", dtype=dt)
    w[:, 0] = torch.tensor([-3e38, -1e30, -1e20, -200.0, 200.0, 1e12, 1e30, 3e38], device="cuda")
    for act in ("silu", "gelu"):
        y = t2sc.dense_linear_device(x, w, activation=act)
        want = torch.where(w[:, 0] > 0, w[:, 0], 0).expand(rows, 8)
        assert torch.equal(y.abs(), want)


def test_linear_more_outputs_than_a_grid_axis(t2sc):
    """f32 with more column tiles than the 65535 of a grid's second axis."""
    import torch
    g = _gen(15)
    co = 65537 * 64 + 3
    x, w, b = _normal(g, 70, 4), _normal(g, co, 4), _normal(g, co)
    y = t2sc.dense_linear_device(x, w, b)
    for c in (slice(0, 70), slice(co // 2, co // 2 + 70), slice(co - 70, co)):
        ref.assert_close(y[:, c], *ref.linear(x, w[c], b[c]))
    ones = torch.ones(70, 4, device="cuda")
    w.fill_(0.25)
    assert torch.equal(t2sc.dense_linear_device(ones, w), torch.ones(70, co, device="cuda"))


def test_layouts_dropped_at_once(t2sc):
    """A layout that is dropped right after its call, its memory given to the next ones, while the kernel still waits
    behind other work on its stream."""
    import torch
    g = _gen(16)
    lens = [13 * (i % 7) for i in range(40)]
    q, k, v = (_normal(g, sum(lens), 2, 64, dtype="bfloat16") for _ in range(3))
    want = t2sc.SequenceLayout(lens).attention_device(q, k, v)
    torch.cuda.synchronize()
    got = []
    for rep in range(8):
        torch.cuda._sleep(20_000_000)
        got.append(t2sc.SequenceLayout(lens).attention_device(q, k, v))
        t2sc.SequenceLayout([1] * 40, [0] * 40)
    assert all(torch.equal(y, want) for y in got)


def test_attention_head_dims_in_turn_and_extreme_scales(t2sc):
    """CUDA-core calls of large and small heads in turn; scales whose product with log2(e) overflows; scores of zero."""
    g = _gen(17)
    for d in (256, 8, 200, 33):
        q, k, v = (_normal(g, 50, 2, d) for _ in range(3))
        ref.assert_close(t2sc.SequenceLayout([50]).attention_device(q, k, v), *ref.attention(q, k, v, [50], [50], d ** -0.5))
    import torch
    for n in (2, 130):
        q = torch.zeros(n, 2, 64, device="cuda", dtype=torch.bfloat16)
        v = _normal(g, n, 2, 64, dtype="bfloat16")
        y = t2sc.SequenceLayout([n]).attention_device(q, q, v, scale=3e38)
        ref.assert_close(y, *ref.attention(q, q, v, [n], [n], 1.0))


def test_the_contexts_stream_stays_as_set(t2sc):
    """Another operator of the same context, called after one of these, runs on the stream that the program gave the
    context: it sees rows that are written there late."""
    import torch
    ctx = t2sc.Context(0)
    g = _gen(18)
    mine = torch.cuda.Stream()
    ctx.set_stream(mine.cuda_stream)
    norm = t2sc.LayerNorm32(64, ctx=ctx)
    new = _normal(g, 40, 64)
    want = norm.forward_device(new)
    rows, y = torch.zeros(40, 64, device="cuda"), torch.zeros(40, 64, device="cuda")
    x, w = _normal(g, 40, 64, dtype="bfloat16"), _normal(g, 48, 64, dtype="bfloat16")
    torch.cuda.synchronize()
    before = ctx.launch_count()
    with torch.cuda.stream(mine):
        torch.cuda._sleep(100_000_000)
        rows.copy_(new)
    z = t2sc.dense_linear_device(x, w, ctx=ctx)
    norm.forward_device(rows, y)
    ref.assert_close(z, *ref.linear(x, w))
    assert ctx.launch_count() == before + 2
    ctx.synchronize()
    assert torch.equal(y, want)
    ctx.close()


def test_handles_made_and_dropped_during_a_capture(t2sc):
    """The first calls of a context, and handles that come and go, while a graph is captured: replays give the same bits."""
    import gc
    import torch
    g = _gen(19)
    lens = [70, 3, 200]
    n = sum(lens)
    q, k, v = (_normal(g, n, 2, 64, dtype="bfloat16") for _ in range(3))
    x, w = _normal(g, n, 128, dtype="bfloat16"), _normal(g, 128, 128, std=0.1, dtype="bfloat16")
    coords = torch.randint(0, 64, (n, 4), generator=g, device="cuda", dtype=torch.int32)
    layout, rope = t2sc.SequenceLayout(lens), t2sc.RotaryPositionEmbedder(64)
    want = [layout.attention_device(rope.forward_device(q, coords), k, v), t2sc.dense_linear_device(x, w)]
    dropped = [t2sc.SequenceLayout([5, 6]), t2sc.RotaryPositionEmbedder(32)]
    torch.cuda.synchronize()
    graph, held = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        ctx = t2sc.Context(0)
        held += [t2sc.SequenceLayout(lens, ctx=ctx), t2sc.RotaryPositionEmbedder(64, ctx=ctx), ctx]
        got = [held[0].attention_device(held[1].forward_device(q, coords), k, v), t2sc.dense_linear_device(x, w, ctx=ctx)]
        dropped.clear()
        gc.collect()
    for y in got:
        y.fill_(NAN)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del graph, got
    held[2].synchronize()


def test_two_threads_with_contexts_of_their_own(t2sc):
    """Two threads, a context and a stream each, calling at once."""
    import threading
    import torch
    g = _gen(21)
    cases = []
    for i, (lens, d) in enumerate((([130, 20], 64), ([40, 7, 300], 128))):
        q, k, v = (_normal(g, sum(lens), 3, d, dtype="float16") for _ in range(3))
        x, w = _normal(g, 90, 256, dtype="bfloat16"), _normal(g, 200, 256, std=1 / 16, dtype="bfloat16")
        f = _normal(g, 33, 2, 24 if i else 200)
        cases.append((lens, q, k, v, x, w, f))
    torch.cuda.synchronize()
    errors = []

    def work(lens, q, k, v, x, w, f):
        try:
            ctx, stream = t2sc.Context(0), torch.cuda.Stream()
            layout, few = t2sc.SequenceLayout(lens, ctx=ctx), t2sc.SequenceLayout([33], ctx=ctx)
            rope = t2sc.RotaryPositionEmbedder(q.shape[2], ctx=ctx)
            coords = torch.arange(4 * len(q), device="cuda", dtype=torch.int32).view(-1, 4)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for rep in range(30):
                    ys = [layout.attention_device(rope.forward_device(q, coords), k, v), few.attention_device(f, f, f),
                          t2sc.dense_linear_device(x, w, activation="gelu", ctx=ctx)]
                    stream.synchronize()
                    first = ys if rep == 0 else first
                    assert all(torch.equal(a, b) for a, b in zip(ys, first))
            ref.assert_close(ys[1], *ref.attention(f, f, f, [33], [33], f.shape[2] ** -0.5))
            ref.assert_close(ys[2], *ref.linear(x, w, None, "gelu"))
            ctx.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_more_refusals(t2sc):
    import torch
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, device="cuda", dtype=dt)  # noqa: E731
    w = (np.zeros((16, 16), np.float32), None)
    attn = t2sc.SparseMultiHeadAttention(16, 2, w, to_qkv=(np.zeros((48, 16), np.float32), None))
    layout = t2sc.SequenceLayout([4])
    bad = [
        lambda: t2sc.RotaryPositionEmbedder(64, theta=0.5), lambda: t2sc.RotaryPositionEmbedder(64, theta=float("inf")),
        lambda: t2sc.SequenceLayout([2.5, 1.0]), lambda: t2sc.SequenceLayout([2 ** 31 - 1]),
        lambda: t2sc.SequenceLayout([3], [2 ** 31 - 1000]),
        lambda: attn.forward_device(z(4, 16), layout, context=z(4, 16)),
    ]
    for call in bad:
        with pytest.raises((ValueError, t2sc.T2SCError)):
            call()
    assert attn.forward_device(z(4, 16), layout).shape == (4, 16)
    t2sc.Context.default(0).synchronize()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,ci,co", [(200, 8192, 128), (300, 4100, 130), (129, 6152, 260), (513, 8192, 4), (700, 9000, 33)])
def test_linear_few_tiles_over_a_long_axis(t2sc, dtype, rows, ci, co):
    """Several tiles of rows with the K axis split, ragged in every direction, in place and with an unaligned result."""
    import torch
    g = _gen(rows + ci)
    x, w, b = _normal(g, rows, ci, dtype=dtype), _normal(g, co, ci, std=ci ** -0.5, dtype=dtype), _normal(g, co)
    for pad in (8, 5):
        rv, buf = _inside(rows, co, dtype, pad_cols=pad)
        rv.copy_(_normal(g, rows, co, dtype=dtype))
        want = ref.linear(x, w, b, "gelu", rv.clone())
        first = t2sc.dense_linear_device(x, w, b, activation="gelu", residual=rv)
        t2sc.dense_linear_device(x, w, b, activation="gelu", residual=rv, out=rv)
        assert torch.equal(first, rv) and _untouched(buf, rows, co)
        ref.assert_close(rv, *want)


def test_calls_in_a_row_see_each_others_results(t2sc):
    """Kernels begin while the one before them ends: chains of small calls that read what the last one wrote and
    overwrite what it read, each kind behind each other, in a graph and eagerly."""
    import torch
    g = _gen(23)
    h, d = 2, 64
    c = h * d
    w = [_normal(g, c, c, std=c ** -0.5, dtype="bfloat16") for _ in range(4)]
    gain = torch.ones(h, d, device="cuda")
    coords = torch.randint(0, 64, (512, 4), generator=g, device="cuda", dtype=torch.int32)
    rope = t2sc.RotaryPositionEmbedder(d)
    layouts = {m: (t2sc.SequenceLayout([m]), t2sc.SequenceLayout([1, 1], [m - m // 4, m // 4]),
                   t2sc.SequenceLayout([0, 0], [m, 0])) for m in (1, 4, 24, 300)}

    def chain(bufs, m):
        a, b = (t[:m] for t in bufs)
        one, few, none = layouts[m]
        heads = lambda t: t.view(m, h, d)  # noqa: E731
        for i in range(6):
            t2sc.dense_linear_device(a, w[i % 4], activation="silu", out=b)
            t2sc.qk_norm_rope_device(heads(b), None, gain, None, coords=coords[:m], rope=rope, out_q=heads(b))
            one.attention_device(heads(b), heads(b), heads(b), out=heads(a))
            none.attention_device(heads(b), heads(b), heads(b), out=heads(a))
            t2sc.dense_linear_device(a, w[(i + 1) % 4], residual=b, out=b)
            rope.forward_device(heads(b), coords[:m], out=heads(b))
            if m > 3:
                few.attention_device(heads(b), heads(b), heads(b), out=heads(a))
            t2sc.dense_linear_device(b, w[(i + 2) % 4], residual=a, out=a)
        return a

    for m in (1, 4, 24, 300):
        start = _normal(g, 300, c, dtype="bfloat16")
        slow = [start.clone(), torch.zeros_like(start)]
        # the same chain with the device idle between any two calls
        sync = torch.cuda.synchronize
        patched = [(t2sc, "dense_linear_device"), (t2sc, "qk_norm_rope_device"), (type(rope), "forward_device"),
                   (t2sc.SequenceLayout, "attention_device")]
        kept = [getattr(o, name) for o, name in patched]

        def waiting(f):
            def call(*args, **kw):
                y = f(*args, **kw)
                sync()
                return y
            return call

        for (o, name), f in zip(patched, kept):
            setattr(o, name, waiting(f))
        try:
            want = chain(slow, m).clone()
        finally:
            for (o, name), f in zip(patched, kept):
                setattr(o, name, f)
        for _ in range(5):
            bufs = [start.clone(), torch.zeros_like(start)]
            assert torch.equal(chain(bufs, m), want)
        bufs = [start.clone(), torch.zeros_like(start)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = chain(bufs, m)
        for _ in range(5):
            bufs[0].copy_(start)
            graph.replay()
            assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("q_len", [1, 2, 4])
def test_attention_more_short_calls_than_sms(t2sc, dtype, d, q_len):
    """Few queries of more sequences and heads than SMs, keys of none, of one and of many blocks, bad values behind them."""
    import torch
    g = _gen(24 + d + q_len)
    kv_lens = [0, 1, 33, 64, 65, 700, 129, 2, 0, 5] * 3
    q_lens = [q_len if i % 7 else 1 for i in range(len(kv_lens))]
    n = sum(kv_lens)
    q = _normal(g, sum(q_lens), 12, d, dtype=dtype)
    k, v = (torch.full((n + 64, 12, d), NAN, device="cuda", dtype=getattr(torch, dtype)) for _ in range(2))
    k[:n], v[:n] = (_normal(g, n, 12, d, dtype=dtype) for _ in range(2))
    y = t2sc.SequenceLayout(q_lens, kv_lens).attention_device(q, k, v)
    ref.assert_close(y, *ref.attention(q, k[:n], v[:n], q_lens, kv_lens, d ** -0.5))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,ci,co", [(1000, 136, 2143), (777, 64, 321), (4000, 40, 65), (300, 72, 4100)])
def test_linear_odd_rows_of_many_tiles(t2sc, dtype, rows, ci, co):
    """Tiles whose rows start anywhere: odd widths, the last columns and rows of a tile, in place and not."""
    import torch
    g = _gen(rows + co)
    x, w, b = _normal(g, rows, ci, dtype=dtype), _normal(g, co, ci, std=ci ** -0.5, dtype=dtype), _normal(g, co)
    for pad in (0, 3, 8):
        rv, buf = _inside(rows, co, dtype, pad_cols=pad)
        rv.copy_(_normal(g, rows, co, dtype=dtype))
        want = ref.linear(x, w, b, "silu", rv.clone())
        first = t2sc.dense_linear_device(x, w, b, activation="silu", residual=rv)
        t2sc.dense_linear_device(x, w, b, activation="silu", residual=rv, out=rv)
        assert torch.equal(first, rv) and _untouched(buf, rows, co)
        ref.assert_close(rv, *want)
        plain, buf = _inside(rows, co, dtype, pad_cols=pad)
        t2sc.dense_linear_device(x, w, out=plain)
        assert _untouched(buf, rows, co)
        ref.assert_close(plain, *ref.linear(x, w))
