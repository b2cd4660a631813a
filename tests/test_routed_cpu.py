"""Routed row movements without a GPU: every refusal comes before a launch, the fake implementations give the shapes and
types of the outputs, and the C entry points reject bad arguments on the host."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import magicompiler_b200 as mb
from magicompiler_b200 import _loader

I32, I64, BF = torch.int32, torch.int64, torch.bfloat16


def maps(tokens=3, k=2):
    return torch.zeros(tokens * k, dtype=I32), torch.zeros(tokens, k, dtype=I32)


def test_sort_refuses():
    for form in (mb.expert_sort, mb.expert_sort_out):
        with pytest.raises(TypeError, match="int32 or int64"):
            form(torch.zeros(3, 2), 4)
        with pytest.raises(ValueError, match=r"\[tokens, choices\]"):
            form(torch.zeros(3, dtype=I64), 4)
        with pytest.raises(ValueError, match=r"\[tokens, choices\]"):
            form(torch.zeros(3, 0, dtype=I64), 4)
        for experts in (0, -1, 1025):
            with pytest.raises(ValueError, match="num_experts"):
                form(torch.zeros(3, 2, dtype=I64), experts)
        with pytest.raises(TypeError, match="CUDA tensors only"):
            form(torch.zeros(3, 2, dtype=I64), 4)


def test_gather_refuses():
    rs, sr = maps()
    for form in (mb.expert_gather, mb.expert_gather_out, mb.expert_gather_fp8, mb.expert_gather_fp8_out):
        with pytest.raises(TypeError, match="bf16 rows only"):
            form(torch.zeros(3, 16), rs, sr)
        with pytest.raises(ValueError, match="x must be"):
            form(torch.zeros(4, 16, dtype=BF), rs, sr)
        with pytest.raises(ValueError, match="x must be"):
            form(torch.zeros(1, 3, 16, dtype=BF), rs, sr)
        with pytest.raises(ValueError, match="multiple of"):
            form(torch.zeros(3, 12, dtype=BF), rs, sr)
        with pytest.raises(ValueError, match="multiple of"):
            form(torch.zeros(3, 0, dtype=BF), rs, sr)
        with pytest.raises(TypeError, match="row_slot must be an int32"):
            form(torch.zeros(3, 16, dtype=BF), rs.long(), sr)
        with pytest.raises(TypeError, match="slot_row must be an int32"):
            form(torch.zeros(3, 16, dtype=BF), rs, sr.long())
        with pytest.raises(ValueError, match="row_slot has 5 rows"):
            form(torch.zeros(3, 16, dtype=BF), rs[:5], sr)
        with pytest.raises(ValueError, match="contiguous 2-D"):
            form(torch.zeros(3, 16, dtype=BF), rs, torch.zeros(2, 3, dtype=I32).t())
        with pytest.raises(TypeError, match="CUDA tensors only"):
            form(torch.zeros(3, 16, dtype=BF), rs, sr)
    with pytest.raises(ValueError, match="multiple of 16"):  # 8 is enough for bf16 rows, not for fp8 ones
        mb.expert_gather_fp8(torch.zeros(3, 24, dtype=BF), rs, sr)


def test_combine_refuses():
    rs, sr = maps()
    y, w = torch.zeros(6, 16, dtype=BF), torch.zeros(3, 2)
    for form in (mb.expert_combine, mb.expert_combine_out):
        with pytest.raises(TypeError, match="bf16 rows only"):
            form(y.float(), w, rs, sr)
        with pytest.raises(ValueError, match="y must be"):
            form(y[:5], w, rs, sr)
        with pytest.raises(TypeError, match="fp32"):
            form(y, w.to(BF), rs, sr)
        with pytest.raises(ValueError, match="weights must be"):
            form(y, w.t(), rs, sr)
        for weights in (w, None):
            with pytest.raises(TypeError, match="CUDA tensors only"):
                form(y, weights, rs, sr)
    with pytest.raises(ValueError, match="row length"):
        mb.expert_combine_backward(torch.zeros(3, 24, dtype=BF), y, w, rs, sr, True, True)


def test_quantise_refuses():
    for form in (mb.quantize_fp8_block, mb.quantize_fp8_block_out):
        with pytest.raises(TypeError, match="bf16 rows only"):
            form(torch.zeros(3, 16))
        with pytest.raises(ValueError, match="x must be"):
            form(torch.zeros(16, dtype=BF))
        with pytest.raises(ValueError, match="multiple of 16"):
            form(torch.zeros(3, 8, dtype=BF))
        with pytest.raises(TypeError, match="CUDA tensors only"):
            form(torch.zeros(3, 16, dtype=BF))


def test_fake_implementations():
    with FakeTensorMode():
        ids = torch.empty(5, 3, dtype=I64, device="cuda")
        rs, sr, off = torch.ops.magi_swiglu.expert_sort(ids, 7)
        assert [(tuple(t.shape), t.dtype) for t in (rs, sr, off)] == [((15,), I32), ((5, 3), I32), ((8,), I32)]
        x = torch.empty(5, 144, dtype=BF, device="cuda")
        xs = torch.ops.magi_swiglu.expert_gather(x, rs, sr)
        assert tuple(xs.shape) == (15, 144) and xs.dtype == BF
        q, s = torch.ops.magi_swiglu.expert_gather_fp8(x, rs, sr)
        assert tuple(q.shape) == (15, 144) and q.dtype == torch.float8_e4m3fn
        assert tuple(s.shape) == (15, 2) and s.dtype == torch.float32
        q, s = torch.ops.magi_swiglu.quantize_fp8_block(x)
        assert tuple(q.shape) == (5, 144) and tuple(s.shape) == (5, 2)
        w = torch.empty(5, 3, device="cuda")
        for weights in (w, None):
            assert tuple(torch.ops.magi_swiglu.expert_combine(xs, weights, rs, sr).shape) == (5, 144)
        dy, dw = torch.ops.magi_swiglu.expert_combine_backward(x, xs, w, rs, sr, True, False)
        assert tuple(dy.shape) == (15, 144) and dy.dtype == BF and tuple(dw.shape) == (0,)


@pytest.mark.parametrize("shift", [1, 4, 8])
@pytest.mark.parametrize("rows", [1, 4])
def test_rows_that_start_off_a_16_byte_boundary_are_copied(rows, shift):
    from magicompiler_b200 import ops, routed

    whole = torch.arange(4 * 64 + 16, dtype=torch.float32).to(BF)
    whole = whole[(-whole.data_ptr() % 16) // 2:]
    t = whole[shift:shift + rows * 64].view(rows, 64)
    assert t.is_contiguous() and (t.data_ptr() % 16 == 0) == (shift == 8)
    for view in (ops._rows_view, routed._rows):
        got = view(t, 64)
        assert got.data_ptr() % 16 == 0 and torch.equal(got, t) and (got.data_ptr() == t.data_ptr()) == (shift == 8)


class _NoKernels:
    """In the place of the library: every entry point succeeds and writes nothing."""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def without_kernels(monkeypatch):
    """Operator bodies that run on CPU tensors up to the launch."""
    from magicompiler_b200 import fp8_block, routed

    monkeypatch.setattr(_loader, "load_library", lambda: _NoKernels())
    for module in (routed, fp8_block):
        monkeypatch.setattr(module, "_check_device", lambda *a: 0)
        monkeypatch.setattr(module, "_raw_stream", lambda dev: 0)


def recorded(fn, *args):
    """The package's operators in the graph that ``torch.jit.trace`` makes of ``fn``."""
    graph = torch.jit.trace(fn, args, check_trace=False).inlined_graph
    return [n.kind() for n in graph.nodes() if n.kind().startswith("magi_swiglu::")]


@pytest.mark.parametrize("grad", [False, True])
def test_a_tracer_records_the_operators(without_kernels, grad):
    rs, sr = maps()
    x, y, w = torch.zeros(3, 16, dtype=BF, requires_grad=grad), torch.zeros(6, 16, dtype=BF, requires_grad=grad), torch.zeros(3, 2)
    assert recorded(lambda *a: mb.expert_gather(*a), x, rs, sr) == ["magi_swiglu::expert_gather"]
    assert recorded(lambda *a: mb.expert_combine(*a), y, w, rs, sr) == ["magi_swiglu::expert_combine"]


def test_a_tracer_records_the_operators_of_the_routed_block(without_kernels):
    mlp = mb.RoutedSwiGLUMLP(torch.zeros(4, 64, 16, dtype=BF), torch.zeros(4, 16, 32, dtype=BF), precision="fp8")
    assert recorded(mlp, torch.zeros(3, 16, dtype=BF), torch.zeros(3, 2, dtype=I64), torch.zeros(3, 2)) == [
        "magi_swiglu::expert_sort", "magi_swiglu::expert_gather_fp8", "magi_swiglu::gemm_swiglu_fp8_block",
        "magi_swiglu::gemm_fp8_block", "magi_swiglu::expert_combine"]


class _Wrapped(torch.Tensor):
    """A tensor without memory of its own; operators get the tensor inside."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    seen = []

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(str(func))
        return func(*[a.inner if isinstance(a, cls) else a for a in args], **(kwargs or {}))


class _Watch(torch.overrides.TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_any_operand_may_be_a_subclass(without_kernels, which):
    rs, sr = maps()
    args = [torch.zeros(6, 16, dtype=BF), torch.zeros(3, 2), rs, sr]
    args[which] = _Wrapped(args[which])
    _Wrapped.seen.clear()
    mb.expert_combine(*args)
    assert any("expert_combine" in f for f in _Wrapped.seen)
    if which != 1:
        args = [torch.zeros(3, 16, dtype=BF), None, rs, sr]
        args[which] = _Wrapped(args[which])
        _Wrapped.seen.clear()
        mb.expert_gather(args[0], args[2], args[3])
        assert any("expert_gather" in f for f in _Wrapped.seen)


def test_a_torch_function_mode_sees_the_operators(without_kernels):
    rs, sr = maps()
    mlp = mb.RoutedSwiGLUMLP(torch.zeros(4, 64, 16, dtype=BF), torch.zeros(4, 16, 32, dtype=BF), precision="fp8")
    with _Watch() as watch:
        mb.expert_gather(torch.zeros(3, 16, dtype=BF), rs, sr)
        mlp(torch.zeros(3, 16, dtype=BF), torch.zeros(3, 2, dtype=I64), torch.zeros(3, 2))
    for op in ("expert_sort", "expert_gather", "expert_gather_fp8", "gemm_swiglu_fp8_block", "gemm_fp8_block", "expert_combine"):
        assert {f"magi_swiglu.{op}", f"magi_swiglu.{op}.default"} & set(watch.seen), op


def test_a_default_device_does_not_send_calls_through_the_dispatcher(without_kernels):
    from magicompiler_b200 import routed

    x = torch.zeros(3, 16, dtype=BF)
    with torch.device("cpu"):
        assert routed._plain(x) and routed._plain(x, None, x)
        mb.expert_gather(x, *maps())
        with _Watch():
            assert not routed._plain(x)
    with _Watch(), torch.device("cpu"):
        assert not routed._plain(x)
    assert routed._plain(x) and not routed._plain(x, _Wrapped(x))


def test_the_row_movements_split_graphs():
    for op in ("expert_sort", "expert_gather", "expert_combine", "expert_gather_fp8"):
        assert f"magi_swiglu::{op}" in mb.SPLITTING_OPS


def test_c_entry_points_reject_on_the_host():
    lib = mb.load_library()
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    p += -p % 16
    sort = lambda **o: lib.magi_swiglu_expert_sort(*{**dict(ids=p, wide=1, slots=4, e=4, rs=p, sr=p, off=p, dev=0, st=None), **o}.values())  # noqa: E731
    assert sort(slots=-1) == -2 and sort(slots=1 << 30) == -2 and sort(e=0) == -2 and sort(e=1025) == -2
    assert sort(ids=None) == -1 and sort(off=None) == -1 and sort(ids=p + 4) == -3 and sort(rs=p + 2) == -3
    assert sort(dev=1000) == -5 and "not available" in _loader.last_error()
    gat = lambda **o: lib.magi_swiglu_expert_gather_bf16(*{**dict(x=p, rs=p, sr=p, xs=p, T=2, k=2, H=16, ld=16, dev=0, st=None), **o}.values())  # noqa: E731
    assert gat(T=-1) == -2 and gat(k=0) == -2 and gat(H=12) == -2 and gat(ld=8) == -2 and gat(T=1 << 30, k=2) == -2
    assert gat(ld=20) == -3 and gat(x=p + 8) == -3 and gat(xs=None) == -1 and gat(T=0, x=None) == 0
    com = lambda **o: lib.magi_swiglu_expert_combine_bf16(*{**dict(y=p, w=p, sr=p, out=p, T=2, k=2, H=16, ld=16, dev=0, st=None), **o}.values())  # noqa: E731
    assert com(H=0) == -2 and com(y=None) == -1 and com(out=p + 4) == -3 and com(T=0) == 0
    bwd = lambda **o: lib.magi_swiglu_expert_combine_backward_bf16(*{**dict(d=p, y=p, w=p, rs=p, sr=p, dy=p, dw=p, T=2, k=2, H=16, ldd=16, ldy=16, dev=0, st=None), **o}.values())  # noqa: E731
    assert bwd(w=None) == -1 and bwd(y=None) == -1 and bwd(ldy=12) == -2 and bwd(dy=None, dw=None) == 0
    assert bwd(ldd=24 + 4) == -3 and bwd(dy=p + 8) == -3
    qua = lambda **o: lib.magi_swiglu_quantize_fp8_block(*{**dict(x=p, c=p, s=p, M=2, K=16, ld=16, dev=0, st=None), **o}.values())  # noqa: E731
    assert qua(K=24, ld=24) == -2 and qua(s=None) == -1 and qua(c=p + 8) == -3 and qua(M=0) == 0
    gf8 = lambda **o: lib.magi_swiglu_expert_gather_fp8_block(*{**dict(x=p, rs=p, sr=p, c=p, s=p, T=2, k=2, K=16, ld=16, dev=0, st=None), **o}.values())  # noqa: E731
    assert gf8(rs=None) == -1 and gf8(K=8, ld=8) == -2
