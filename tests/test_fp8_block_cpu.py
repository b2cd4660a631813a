"""Block-scaled fp8 products without a GPU: refusals, fake implementations, the load-time weight quantisers and the host
checks of the C entry points."""
import copy
import ctypes

import pytest
import torch
from hypothesis import given, settings, strategies as st
from torch._subclasses.fake_tensor import FakeTensorMode

import magicompiler_b200 as mb
from magicompiler_b200 import _loader

F8, F32, I32 = torch.float8_e4m3fn, torch.float32, torch.int32


def operands(m=4, n=256, k=272, experts=0, halves=1):
    lead = (experts,) if experts else ()
    nb, kb = -(-n // 128), -(-k // 128)
    t = dict(a=torch.zeros(m, k).to(F8), a_scale=torch.zeros(m, kb), b=torch.zeros(*lead, halves * n, k).to(F8),
             b_scale=torch.zeros(*lead, halves * nb, kb))
    if experts:
        t["offsets"] = torch.zeros(experts + 1, dtype=I32)
    return t


FORMS = [(mb.gemm_fp8_block, 1), (mb.gemm_fp8_block_out, 1), (mb.gemm_swiglu_fp8_block, 2), (mb.gemm_swiglu_fp8_block_out, 2)]


@pytest.mark.parametrize("form,halves", FORMS)
def test_refusals(form, halves):
    def call(error, match, experts=0, **changes):
        t = operands(experts=experts, halves=halves)
        t.update(changes)
        with pytest.raises(error, match=match):
            form(t["a"], t["a_scale"], t["b"], t["b_scale"], t.get("offsets"))

    t = operands(halves=halves)
    call(TypeError, "CUDA tensors only")
    call(TypeError, "CUDA tensors only", experts=3)
    call(TypeError, "a must be", a=t["a"].to(torch.float8_e5m2))
    call(TypeError, "a must be", a=t["a"].to(torch.bfloat16))
    call(TypeError, "b must be", b=t["b"].view(torch.uint8))
    call(TypeError, "a_scale must be", a_scale=t["a_scale"].double())
    call(TypeError, "b_scale must be", b_scale=t["b_scale"].to(torch.bfloat16))
    call(TypeError, "offsets must be", experts=3, offsets=torch.zeros(4, dtype=torch.int64))
    call(ValueError, "2-D", a=t["a"][None])
    call(ValueError, "without offsets", b=t["b"][None])
    call(ValueError, "with offsets", experts=3, b=t["b"])
    call(ValueError, "offsets must be a contiguous", experts=3, offsets=torch.zeros(5, dtype=I32))
    call(ValueError, "inner dimensions", a=torch.zeros(4, 256).to(F8))
    call(ValueError, "a_scale must be", a_scale=torch.zeros(4, 2))
    call(ValueError, "scales must be", b_scale=torch.zeros(1, 3))
    call(ValueError, "must be contiguous", b=torch.zeros(halves * 256, 288).to(F8)[:, :272])
    call(ValueError, "multiple of", **{k: v for k, v in operands(n=256, k=264, halves=halves).items()})
    call(ValueError, "multiple of", **{k: v for k, v in operands(n=252, k=272, halves=halves).items()})
    call(ValueError, "multiple of", a=torch.zeros(4, 0).to(F8), b=torch.zeros(halves * 256, 0).to(F8))


def test_an_odd_number_of_packed_rows_is_refused():
    t = operands(n=256, halves=1)
    with pytest.raises(ValueError, match="N gate rows"):
        mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"][:255], t["b_scale"])
    with pytest.raises(ValueError, match="N gate rows"):
        mb.quantize_fp8_gate_up(torch.zeros(255, 64))
    with pytest.raises(ValueError, match="a weight is"):
        mb.quantize_fp8_weight(torch.zeros(64))


def test_fake_implementations():
    with FakeTensorMode():
        for experts in (0, 3):
            t = {k: torch.empty(v.shape, dtype=v.dtype, device="cuda") for k, v in operands(experts=experts).items()}
            c = torch.ops.magi_swiglu.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t.get("offsets"))
            assert tuple(c.shape) == (4, 256) and c.dtype == torch.bfloat16
            t = {k: torch.empty(v.shape, dtype=v.dtype, device="cuda") for k, v in operands(n=272, experts=experts, halves=2).items()}
            q, s = torch.ops.magi_swiglu.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t.get("offsets"))
            assert tuple(q.shape) == (4, 272) and q.dtype == F8 and tuple(s.shape) == (4, 3) and s.dtype == F32


@pytest.mark.parametrize("n,k", [(128, 128), (130, 144), (1, 16), (300, 500)])
def test_weight_quantiser(n, k):
    """Each code times its scale is within half an e4m3 step of the weight: 2^-4 of its size, or half the smallest code
    (2^-10) of the scale."""
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n))
    codes, scales = mb.quantize_fp8_weight(w)
    assert codes.dtype == F8 and tuple(scales.shape) == (-(-n // 128), -(-k // 128))
    full = scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    err = (codes.float() * full - w).abs()
    assert (err <= w.abs() * 2.0 ** -4 * (1 + 1e-6) + full * 2.0 ** -10).all()
    two = torch.stack([w, -2 * w])
    c2, s2 = mb.quantize_fp8_weight(two)
    assert torch.equal(c2[0].float(), codes.float()) and torch.equal(s2[1], 2 * scales)


def test_gate_up_halves_are_blocked_from_their_own_first_row():
    w = torch.randn(2 * 200, 136, generator=torch.Generator().manual_seed(1))
    codes, scales = mb.quantize_fp8_gate_up(w)
    g, gs = mb.quantize_fp8_weight(w[:200])
    u, us = mb.quantize_fp8_weight(w[200:])
    assert torch.equal(codes.float(), torch.cat([g.float(), u.float()])) and torch.equal(scales, torch.cat([gs, us]))
    assert tuple(mb.quantize_fp8_gate_up(torch.zeros(3, 400, 136))[1].shape) == (3, 4, 2)
    assert (mb.quantize_fp8_weight(torch.zeros(8, 16))[1] == 2.0 ** -126).all()


def row_groups(offsets, M, rows, running_maximum):
    """The kernels' count of groups of `rows` rows: every offset clamped to [0, M] and, with `running_maximum`, one below an
    earlier one taken for that one."""
    starts = []
    for o in offsets:
        o = min(max(o, 0), M)
        starts.append(max(o, starts[-1]) if running_maximum and starts else o)
    return sum(-(-max(hi - lo, 0) // rows) for lo, hi in zip(starts, starts[1:]))


@settings(max_examples=300, deadline=None)
@given(st.integers(1, 3000), st.sampled_from([16, 32, 64, 128, 256]), st.lists(st.integers(-10, 4000), min_size=2, max_size=70))
def test_no_offsets_make_more_row_groups_than_a_launch_has_room_for(M, rows, offsets):
    """The host counts on at most M / rows whole groups and one partial one for each expert with rows; a cluster that shares a
    tile's K blocks relies on it (a second tile would put its barriers out of step)."""
    room = M // rows + min(M, len(offsets))
    assert row_groups(offsets, M, rows, True) <= room


def test_clamping_alone_would_let_falling_offsets_make_more_row_groups():
    assert row_groups([0, 1100, 0, 1100], 1100, 256, False) == 10 > 1100 // 256 + 4
    assert row_groups([0, 1100, 0, 1100], 1100, 256, True) == 5


def test_c_entry_points_reject_on_the_host():
    lib = mb.load_library()
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    p += -p % 16
    base = dict(a=p, asc=p, b=p, bsc=p, off=None, e=1, c=p, M=4, N=16, K=32, lda=32, lds=1, zt=1, dev=0, st=None)
    gemm = lambda **o: lib.magi_swiglu_gemm_fp8_block(*{**base, **o}.values())  # noqa: E731
    assert gemm(M=-1) == -2 and gemm(N=12) == -2 and gemm(K=24) == -2 and gemm(e=2) == -2 and gemm(e=0) == -2
    assert gemm(off=p, e=1025) == -2 and gemm(lda=16) == -2 and gemm(lds=0) == -2
    assert gemm(lda=40) == -3 and gemm(a=p + 8) == -3 and gemm(c=p + 2) == -3 and gemm(bsc=p + 2) == -3
    assert gemm(b=None) == -1 and gemm(c=None) == -1 and gemm(M=0, a=None) == 0
    assert gemm(dev=1000) == -5 and "not available" in _loader.last_error()
    base = dict(a=p, asc=p, b=p, bsc=p, off=None, e=1, c=p, s=p, M=4, N=16, K=32, lda=32, lds=1, zt=1, dev=0, st=None)
    fused = lambda **o: lib.magi_swiglu_gemm_swiglu_fp8_block(*{**base, **o}.values())  # noqa: E731
    assert fused(N=8) == -2 and fused(s=None) == -1 and fused(c=p + 4) == -3 and fused(M=0) == 0


@pytest.mark.parametrize("lead", [(), (3,)])
def test_quantised_parameters_keep_no_graph(lead):
    w = torch.nn.Parameter(torch.randn(*lead, 64, 48))
    for quantiser in (mb.quantize_fp8_weight, mb.quantize_fp8_gate_up):
        for got, want in zip(quantiser(w), quantiser(w.detach())):
            assert not got.requires_grad and torch.equal(got.float(), want.float())


def test_a_routed_block_made_from_parameters_can_be_copied():
    w13, w2 = (torch.nn.Parameter(torch.randn(s).to(torch.bfloat16)) for s in ((3, 64, 48), (3, 48, 32)))
    mlp = mb.RoutedSwiGLUMLP(w13, w2, precision="fp8")
    assert not any(b.requires_grad for b in mlp.buffers())
    for a, b in zip(copy.deepcopy(mlp).buffers(), mlp.buffers()):
        assert torch.equal(a.float(), b.float())


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16),
                                  lambda m: torch.nn.Sequential(m).to(torch.float16)[0], lambda m: m.type(torch.float64)])
def test_a_cast_of_the_module_leaves_codes_and_scales(cast):
    w13, w2 = torch.randn(3, 64, 48).to(torch.bfloat16), torch.randn(3, 48, 32).to(torch.bfloat16)
    mlp = mb.RoutedSwiGLUMLP(w13, w2, precision="fp8")
    before = {k: v.clone() for k, v in mlp.named_buffers()}
    assert len(before) == 4
    for k, v in cast(mlp).named_buffers():
        assert v.dtype == before[k].dtype == (F8 if k.endswith("codes") else F32) and torch.equal(v.float(), before[k].float())
    moved = mlp.to("meta", torch.bfloat16)
    assert all(b.device.type == "meta" and b.dtype == before[k].dtype for k, b in moved.named_buffers())
    trainable = mb.RoutedSwiGLUMLP(w13, w2).float()
    assert all(p.dtype == F32 for p in trainable.parameters())


def plan(*args, form=0, **kw):
    prev = _loader.set_tuning("fp8_form", form)
    try:
        return tuple(_loader.fp8_block_plan(*args, sm_count=148, **kw).values())
    finally:
        assert _loader.set_tuning("fp8_form", prev) == form


def test_plans_of_the_sizes_that_the_kernels_are_for():
    assert plan(8192, 4096, 14336) == plan(8192, 14336, 4096, halves=2) == (0, 2, 1)  # long prompts: CTA pairs
    assert plan(15200, 1424, 2064, halves=2, experts=64) == (0, 2, 1)
    assert plan(15200, 1408, 2048, halves=2, experts=64) == (0, 1, 1)  # many rows an expert, K a multiple of 32: single CTAs
    assert plan(4096, 2048, 768, experts=128) == (0, 1, 1)
    for tokens, ctas, splits in (plan(1, 4096, 14336), plan(16, 28672, 8192, halves=2), plan(74, 4096, 14336, experts=8)):
        assert tokens in (16, 32, 64) and ctas == 1 and splits in (1, 2, 4, 8)


def test_a_form_asked_for_is_the_one_planned_or_refused():
    for form in (16, 32, 64):
        assert plan(300, 256, 2048, form=form) == (form, 1, 1) and plan(300, 256, 2048, form=form + 1024, experts=3) == (form, 1, 4)
    for form, ctas, splits in ((1, 1, 1), (2, 2, 1), (4, 2, 2), (8, 2, 4)):
        for halves in (1, 2):
            assert plan(300, 256, 2048, form=form, halves=halves) == (0, ctas, splits)
    for form, args, kw in ((64, (300, 256, 2048), dict(halves=2)), (8, (300, 256, 384), {}), (16 + 2048, (300, 256, 896), {}),
                           (8, (8192, 4096, 4096), {}), (4, (8192, 4096, 4096), {}), (16, (2 ** 21, 256, 256), {}),
                           (16 + 768, (300, 256, 2048), {}), (3, (300, 256, 2048), {}), (128, (300, 256, 2048), {}),
                           (258, (300, 256, 2048), {})):
        with pytest.raises(ValueError, match="cannot serve"):
            plan(*args, form=form, **kw)
    for args, kw in (((0, 16, 16), {}), ((1, 12, 16), {}), ((1, 8, 16), dict(halves=2)), ((1, 8, 24), {}), ((1, 8, 16), dict(halves=3)),
                     ((1, 8, 16), dict(experts=1025))):
        with pytest.raises(ValueError, match="out of range"):
            plan(*args, **kw)


def test_watchdog_selftest_rejects_on_the_host():
    selftest = mb.load_library().magi_swiglu_fp8_block_watchdog_selftest
    assert selftest(0, None, 10) == -2 and selftest(0, None, 10 ** 10) == -2 and selftest(1000, None, 2000) == -5


@pytest.mark.parametrize("shape", [(32,), (), (1, 2, 32, 32)])
def test_weights_of_other_ranks_are_refused(shape):
    for quantiser in (mb.quantize_fp8_weight, mb.quantize_fp8_gate_up):
        with pytest.raises(ValueError, match="a weight is"):
            quantiser(torch.zeros(shape))
