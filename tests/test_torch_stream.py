"""A context on torch's current stream, and the cases of perf/operators.py
through the framework's entry points."""
import ctypes
import importlib.util
import os
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cases():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("torch_handle,want", [(0, 1), (4711, 4711)])
def test_use_torch_stream_sets_torchs_stream(t2sc, monkeypatch, torch_handle, want):
    """Torch's default stream has handle 0, which would name the context's own stream: it is given as cudaStreamLegacy."""
    import torch
    ctx = object.__new__(t2sc.Context)
    ctx.handle, ctx.device, ctx._beside_torch = ctypes.c_void_p(64), 3, None
    asked, given = [], []
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device=None: asked.append(device) or types.SimpleNamespace(cuda_stream=torch_handle))
    monkeypatch.setattr(ctx, "_switch_stream", given.append)
    ctx.use_torch_stream()
    assert asked == [3] and given == [want]


@pytest.mark.gpu
def test_use_torch_stream_orders_work(t2sc):
    """A call by device pointers sees rows that torch's current stream writes late, on a stream of torch's and on its default one."""
    import torch
    ctx = t2sc.Context(0)
    new = torch.randn(40, 64, device="cuda")
    want = t2sc.LayerNorm32(64, eps=1e-6, affine=False, ctx=ctx).forward_device(new)
    for stream in (torch.cuda.Stream(), torch.cuda.default_stream()):
        rows, y = torch.zeros(40, 64, device="cuda"), torch.zeros(40, 64, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            ctx.use_torch_stream()
            torch.cuda._sleep(100_000_000)
            rows.copy_(new)
            t2sc._lib.check(t2sc.lib.t2sc_layernorm_device(ctx.handle, rows.data_ptr(), y.data_ptr(), 40, 64, None, None, 1e-6, 0,
                                                           t2sc._lib.DT_F32), ctx.handle)
            got = y.clone()
        stream.synchronize()
        assert torch.equal(got, want)
    ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear one row", "linear qkv 1941", "rope 509", "rope 49152 f32", "qk norm rope 1941",
                                  "attention 1 x 49152", "attention 1203+738", "attention cross f16"])
def test_listed_case_through_the_entry_points(t2sc, name):
    """Every kind of listed case runs through the framework's calls and agrees with its plain form: f32 sums rounded once on both
    sides, and in attention the weights rounded to the type, whose errors are independent and average out."""
    import torch
    cases = _cases()
    case = next(c for c in cases.listed() if c["name"] == name)
    got = {}
    for cases.own in (True, False):
        y = cases.run(cases.prepare(case, 5))
        got[cases.own] = list(y) if isinstance(y, (tuple, list)) else [y]
    u = torch.finfo(cases.DTYPES[case["dtype"]]).eps / 2
    assert len(got[True]) == len(got[False])
    for a, b in zip(got[True], got[False]):
        assert a.shape == b.shape and a.dtype == b.dtype
        a, b = a.double(), b.double()
        assert ((a - b).norm() / b.norm()).item() <= 2 * u
