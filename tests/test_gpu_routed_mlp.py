"""``RoutedSwiGLUMLP``: the routed operators and the experts' products as a user runs them, forward, gradients, fp8, graph."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import magicompiler_b200 as mb

ROOT = Path(__file__).resolve().parent.parent
BF = torch.bfloat16


def weights(E, N, K, K_out, seed, device):
    g = torch.Generator().manual_seed(seed)
    w13 = (torch.randn(E, 2 * N, K, generator=g) * K ** -0.5).to(BF)
    w2 = (torch.randn(E, K_out, N, generator=g) * N ** -0.5).to(BF)
    return w13.to(device), w2.to(device)


def batch(shape, k, E, K, seed, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, K, generator=g).to(BF)
    logits = torch.randn(*shape, E, generator=g)
    top, ids = torch.topk(logits, k, dim=-1)
    ids[torch.rand(*shape, k, generator=g) < drop] = -1
    return x.cuda(), ids.cuda(), torch.softmax(top, -1).cuda()


def plain(x, ids, w, w13, w2):
    """The formula in 64 bits, differentiable, masked instead of sorted."""
    N = w2.shape[2]
    out = 0
    for e in range(w13.shape[0]):
        h = x @ w13[e].t()
        y = (torch.nn.functional.silu(h[..., :N]) * h[..., N:]) @ w2[e].t()
        out = out + y * (w * (ids == e)).sum(-1, keepdim=True)
    return out


def test_refusals():
    w13, w2 = weights(2, 64, 32, 32, 0, "cpu")
    with pytest.raises(ValueError, match="precision"):
        mb.RoutedSwiGLUMLP(w13, w2, precision="int8")
    with pytest.raises(ValueError, match="must be"):
        mb.RoutedSwiGLUMLP(w13, w2[:1])
    with pytest.raises(ValueError, match="must be"):
        mb.RoutedSwiGLUMLP(w13[:, :100], w2)
    with pytest.raises(TypeError, match="bf16"):
        mb.RoutedSwiGLUMLP(w13.float(), w2.float())
    mlp = mb.RoutedSwiGLUMLP(w13, w2)
    x = torch.zeros(3, 32, dtype=BF)
    with pytest.raises(ValueError, match="agree"):
        mlp(x, torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 1))
    with pytest.raises(ValueError, match="agree"):
        mlp(x, torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2))
    with pytest.raises(TypeError, match="CUDA tensors only"):
        mlp(x, torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,k,E,K,N,drop", [((1,), 2, 4, 64, 128, 0), ((3, 17), 2, 4, 256, 272, 0.2), ((300,), 3, 8, 128, 64, 0),
                                                ((40,), 2, 40, 64, 48, 0), ((5,), 2, 3, 64, 64, 1.0)])
def test_training_step(shape, k, E, K, N, drop):
    """bf16: the four roundings to bf16 of the chain (y, h, the experts' outputs, the result; a gradient has as many again)
    are 2^-8 of a value each with random signs: 2-norm errors stay under 8 * 2^-8 of the norm."""
    w13, w2 = weights(E, N, K, K, 1, "cuda")
    x, ids, w = batch(shape, k, E, K, 2, drop)
    mlp = mb.RoutedSwiGLUMLP(w13, w2)
    x.requires_grad_(), w.requires_grad_()
    out = mlp(x, ids, w)
    leaves = [t.detach().double().requires_grad_() for t in (x, w, w13, w2)]
    want = plain(leaves[0], ids, leaves[1], leaves[2], leaves[3])
    d = torch.randn(*shape, K, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    out.backward(d)
    want.backward(d.double())
    assert out.shape == (*shape, K) and out.dtype == BF
    for name, got, ref in (("out", out, want), ("x", x.grad, leaves[0].grad), ("w", w.grad, leaves[1].grad),
                           ("gate_up", mlp.w_gate_up.grad, leaves[2].grad), ("down", mlp.w_down.grad, leaves[3].grad)):
        got, ref = got.detach().double(), ref.detach()
        assert (got - ref).norm() <= 8 * 2.0 ** -8 * ref.norm() + 1e-30, (name, ((got - ref).norm() / ref.norm()).item())


@pytest.mark.gpu
@pytest.mark.parametrize("shape,k,E,K,N,drop", [((1,), 2, 8, 256, 272, 0), ((2, 33), 2, 4, 272, 256, 0.2), ((600,), 4, 6, 512, 384, 0)])
def test_fp8_forward(shape, k, E, K, N, drop):
    """Three quantisations at 2^-4 of a value at most each, uniform in their step: 3 * 2^-4 / sqrt(3) ~ 0.11 of the norm."""
    w13, w2 = weights(E, N, K, K, 4, "cuda")
    x, ids, w = batch(shape, k, E, K, 5, drop)
    mlp = mb.RoutedSwiGLUMLP(w13, w2, precision="fp8")
    out = mlp(x, ids, w)
    want = plain(x.double(), ids, w.double(), w13.double(), w2.double())
    assert out.shape == (*shape, K) and (out.double() - want).norm() <= 0.11 * want.norm()
    with pytest.raises(RuntimeError, match="inference"):
        mlp(x.clone().requires_grad_(), ids, w)
    assert set(mlp.state_dict()) == {"gate_up_codes", "gate_up_scales", "down_codes", "down_scales"}


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_no_tokens(precision):
    mlp = mb.RoutedSwiGLUMLP(*weights(3, 64, 128, 128, 1, "cuda"), precision=precision)
    out = mlp(*batch((0,), 2, 3, 128, 1))
    assert out.shape == (0, 128) and out.dtype == BF


@pytest.mark.gpu
def test_compiled_fp8_forward():
    """Under torch.compile the block is made of the registered ops: the same bits as the direct calls."""
    mlp = mb.RoutedSwiGLUMLP(*weights(4, 128, 256, 256, 2, "cuda"), precision="fp8")
    args = batch((30,), 2, 4, 256, 3, 0.1)
    compiled = torch.compile(mlp, backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        assert torch.equal(compiled(*args), mlp(*args))


@pytest.mark.gpu
def test_fp8_forward_captured_on_a_stream():
    w13, w2 = weights(8, 256, 256, 256, 6, "cuda")
    mlp = mb.RoutedSwiGLUMLP(w13, w2, precision="fp8")
    x, ids, w = batch((24,), 2, 8, 256, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(x, ids, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(x, ids, w)
    for seed in (8, 9):
        for dst, src in zip((x, ids, w), batch((24,), 2, 8, 256, seed, 0.3)):
            dst.copy_(src)
        graph.replay()
        assert torch.equal(out, mlp(x, ids, w))


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_back_to_back_calls_that_reuse_every_buffer(captured):
    """Kernels may be scheduled while the previous one drains: each has to see its writes, and must not write too early."""
    E, k, T, H, N = 8, 2, 24, 512, 256
    w13, w2 = weights(E, N, H, H, 7, "cuda")
    qw, qws = mb.quantize_fp8_weight(w13)
    qd, qds = mb.quantize_fp8_weight(w2)
    inputs = [batch((T,), k, E, H, 100 + i, drop=0.1) for i in range(6)]
    R = T * k
    f8 = torch.float8_e4m3fn
    xq, hq = torch.empty(R, H, dtype=f8, device="cuda"), torch.empty(R, N, dtype=f8, device="cuda")
    xs, hs = torch.empty(R, H // 128, device="cuda"), torch.empty(R, N // 128, device="cuda")
    y, x, ids, rw = (torch.empty(R, H, dtype=BF, device="cuda"), torch.empty_like(inputs[0][0]),
                     torch.empty_like(inputs[0][1]), torch.empty_like(inputs[0][2]))
    index = [torch.empty(R, dtype=torch.int32, device="cuda"), torch.empty(T, k, dtype=torch.int32, device="cuda"),
             torch.empty(E + 1, dtype=torch.int32, device="cuda")]
    out = [torch.empty(T, H, dtype=BF, device="cuda") for _ in inputs]

    def run(i, wait=lambda: None):
        for d, s in zip((x, ids, rw), inputs[i]):
            d.copy_(s)
        wait()
        rs, sr, off = mb.expert_sort_out(ids, E, out=index)
        wait()
        mb.expert_gather_fp8_out(x, rs, sr, out=(xq, xs))
        wait()
        mb.gemm_swiglu_fp8_block_out(xq, xs, qw, qws, off, out=(hq, hs))
        wait()
        mb.gemm_fp8_block_out(hq, hs, qd, qds, off, out=y)
        wait()
        mb.expert_combine_out(y, rw, rs, sr, out=out[i])
        wait()

    for b in (xq, hq, xs, hs, y):
        b.zero_()
    want = []
    for i in range(len(inputs)):
        run(i, torch.cuda.synchronize)
        want.append(out[i].clone())
    steps = lambda: [run(i) for i in range(len(inputs))]
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            steps()
        steps = graph.replay
    for _ in range(20):
        for o in out:
            o.zero_()
        steps()
        for o, r in zip(out, want):
            assert torch.equal(o, r)


@pytest.mark.gpu
def test_first_call_of_a_process_inside_a_capture():
    """Whatever the library looks up once per device it may look up while a stream is being captured."""
    code = """
import torch, magicompiler_b200 as mb
torch.manual_seed(0)
w13, w2 = torch.randn(4, 512, 2048).bfloat16().cuda(), torch.randn(4, 2048, 256).bfloat16().cuda()
mlp = mb.RoutedSwiGLUMLP(w13 * 0.02, w2 * 0.05, precision="fp8")
for T in (5, 1200):
    x, w = torch.randn(T, 2048).bfloat16().cuda(), torch.rand(T, 2).cuda()
    ids = torch.randint(0, 4, (T, 2)).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(x, ids, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, mlp(x, ids, w))
assert mb.device_status(0)["code"] == 0
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@pytest.mark.gpu
def test_traced_and_compiled_calls_go_through_the_ops():
    """make_fx and autograd formulas of the registered ops: the same values as the direct calls."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, ids, w = batch((20,), 2, 4, 64, 1)
    row_slot, slot_row, _ = mb.expert_sort(ids, 4)

    def block(x, w):
        return mb.expert_combine(mb.expert_gather(x, row_slot, slot_row), w, row_slot, slot_row)

    graph = make_fx(block)(x, w)
    targets = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    assert {"magi_swiglu.expert_gather.default", "magi_swiglu.expert_combine.default"} <= targets
    assert torch.equal(graph(x, w), block(x, w))
    grads = []
    for gather, combine in ((mb.expert_gather, mb.expert_combine),
                            (torch.ops.magi_swiglu.expert_gather, torch.ops.magi_swiglu.expert_combine)):
        lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
        combine(gather(lx, row_slot, slot_row), lw, row_slot, slot_row).sum().backward()
        grads.append((lx.grad, lw.grad))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


@pytest.mark.gpu
def test_registered_ops_keep_their_contracts():
    """Schema, fake implementation (shapes, strides, types) and autograd registration of every new op against real calls."""
    x, ids, w = batch((9,), 2, 4, 144, 2, 0.2)
    row_slot, slot_row, offsets = mb.expert_sort(ids, 4)
    xs, ops = mb.expert_gather(x, row_slot, slot_row), torch.ops.magi_swiglu
    a, a_scale = mb.quantize_fp8_block(xs)
    w13, w2 = weights(4, 64, 144, 144, 3, "cuda")
    q13, q2 = mb.quantize_fp8_gate_up(w13), mb.quantize_fp8_weight(w2)
    h, h_scale = mb.gemm_swiglu_fp8_block(a, a_scale, *q13, offsets)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    every = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    with_fp8 = every[1:3]  # torch's schema check multiplies the values, which float8 tensors cannot do
    for op, args, tests in (
            (ops.expert_sort, (ids, 4), every), (ops.expert_gather, (grad(x), row_slot, slot_row), every),
            (ops.expert_combine, (grad(xs), grad(w), row_slot, slot_row), every),
            (ops.expert_combine, (grad(xs), None, row_slot, slot_row), every),
            (ops.expert_combine_backward, (x, xs, w, row_slot, slot_row, True, True), every[:3]),
            (ops.quantize_fp8_block, (x,), with_fp8), (ops.expert_gather_fp8, (x, row_slot, slot_row), with_fp8),
            (ops.gemm_swiglu_fp8_block, (a, a_scale, *q13, offsets), with_fp8),
            (ops.gemm_fp8_block, (h, h_scale, *q2, offsets), with_fp8), (ops.gemm_fp8_block, (a, a_scale, q13[0][0], q13[1][0][:1]), with_fp8)):
        torch.library.opcheck(op.default, args, test_utils=tests)


@pytest.mark.gpu
def test_traced_calls_follow_their_inputs():
    """torch.jit.trace records the operators: the traced functions answer other inputs, of other lengths, like eager calls."""
    E, k, H = 6, 2, 64

    def inputs(T, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return (torch.randn(T, H, generator=g, device="cuda").to(BF), torch.randint(-1, E, (T, k), generator=g, device="cuda"),
                torch.rand(T, k, generator=g, device="cuda"))

    def there_and_back(x, ids, w):
        row_slot, slot_row, _ = mb.expert_sort(ids, E)
        return mb.expert_combine(mb.expert_gather(x, row_slot, slot_row), w, row_slot, slot_row)

    g = torch.Generator(device="cuda").manual_seed(1)
    mlp = mb.RoutedSwiGLUMLP((0.1 * torch.randn(E, 64, H, generator=g, device="cuda")).to(BF),
                             (0.1 * torch.randn(E, H, 32, generator=g, device="cuda")).to(BF), precision="fp8")
    for fn in (there_and_back, mlp):
        with torch.no_grad():
            traced = torch.jit.trace(fn, inputs(20, 0), check_trace=False)
            for T, seed in ((20, 2), (7, 3), (300, 4)):
                args = inputs(T, seed)
                assert torch.equal(traced(*args), fn(*args))
