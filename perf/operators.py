"""Cases of the routed (mixture-of-experts) feed-forward operators and of the block-scaled fp8 products under them.

A routed SwiGLU block sorts its tokens by expert, gathers them (in bf16 for training, quantised for serving), runs the
experts' gate/up and down projections over contiguous row ranges, and adds each token's weighted results up again.
Every case is one of those steps, in the direction and type that a training step or a serving step uses it.

``own`` False: elementary torch operations in 32 bits, rounded once.  ``own`` True: the package's operators."""
import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
TINY = 2.0 ** -126


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoded token finds its experts' rows: pure latency
        dict(name="dispatch_one_token", op="dispatch", T=1, k=2, E=8, H=4096, grad=False, valid=1),
        # a training step of an 8-expert block with the Llama-3-8B width: sorted, gathered, and the gradient back
        dict(name="dispatch_train", op="dispatch", T=8192, k=2, E=8, H=4096, grad=True, valid=8192),
        # many small experts, an odd token count and a padded batch tail that belongs to no expert
        dict(name="dispatch_fine_grained", op="dispatch", T=4099, k=8, E=128, H=2048, grad=False, valid=3900),
        # one decoded token's results come back with their router weights
        dict(name="combine_one_token", op="combine", T=1, k=2, E=8, H=4096, grad=False, valid=1),
        # a training step: weighted sum, gradients of the experts' outputs and of the router weights
        dict(name="combine_train", op="combine", T=8192, k=8, E=64, H=2048, grad=True, valid=8192),
        # activations quantised in front of a dense fp8 projection (Llama-3-8B width)
        dict(name="quantize_rows", op="quantize", M=8192, K=4096, routed=False),
        # activations quantised on the way to their experts, ragged
        dict(name="quantize_routed", op="quantize", T=2005, k=8, E=64, K=2064, routed=True, valid=2005),
        # the dense down projection of the Llama-3-8B block over a prompt
        dict(name="down_prompt", op="gemm", M=8192, N=4096, K=14336, E=0, k=1, valid=8192),
        # the down projection of eight experts for a handful of decoded tokens: the weights' bytes are everything
        dict(name="down_experts_decode", op="gemm", M=37, N=4096, K=14336, E=8, k=2, valid=37),
        # the fused gate/up projection of the Llama-3-8B block over a prompt
        dict(name="gate_up_prompt", op="swiglu", M=8192, N=14336, K=4096, E=0, k=1, valid=8192),
        # the same projection of the 70B-class decode weight, a batch of 16 tokens
        dict(name="gate_up_decode", op="swiglu", M=16, N=28672, K=8192, E=0, k=1, valid=16),
        # fine-grained experts over an odd number of prompt tokens, ragged widths and a padded tail
        dict(name="gate_up_experts_prompt", op="swiglu", M=2005, N=1424, K=2064, E=64, k=8, valid=1900),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, lo, hi, m):
    return max(m, _log(rng, lo, hi) // m * m)


def draw(rng):
    op = rng.choice(("dispatch", "combine", "quantize", "gemm", "swiglu"))
    E = _log(rng, 4, 256)
    k = rng.randint(1, min(E, 8))
    if op in ("dispatch", "combine"):
        H = _mult(rng, 256, 8192, 8)
        T = _log(rng, 1, max(1, min(16384, 33_000_000 // (H * k))))
        return dict(op=op, T=T, k=k, E=E, H=H, grad=rng.random() < 0.5, valid=T if rng.random() < 0.6 else rng.randint(0, T))
    if op == "quantize":
        K = _mult(rng, 128, 14336, 16)
        if rng.random() < 0.5:
            return dict(op=op, M=_log(rng, 1, max(1, min(16384, 33_000_000 // K))), K=K, routed=False)
        T = _log(rng, 1, max(1, min(16384, 33_000_000 // (K * k))))
        return dict(op=op, T=T, k=k, E=E, K=K, routed=True, valid=T if rng.random() < 0.6 else rng.randint(0, T))
    N, K = _mult(rng, 128, 16384, 16), _mult(rng, 128, 16384, 16)
    if rng.random() < 0.5:
        M = _log(rng, 1, max(1, min(8192, int(4.0e11 // (N * K)))))
        return dict(op=op, M=M, N=N, K=K, E=0, k=1, valid=M)
    E = min(E, max(1, 900_000_000 // (2 * N * K)))
    k = min(k, E)
    M = _log(rng, 1, max(1, min(8192, int(4.0e11 // (N * K * k)))))
    return dict(op=op, M=M, N=N, K=K, E=E, k=k, valid=M if rng.random() < 0.6 else rng.randint(0, M))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _route(T, k, E, valid, g):
    """Expert ids [T, k] (distinct per token, some experts more popular than others; -1 in a padded tail) and softmax weights."""
    logits = torch.randn(T, E, generator=g, device="cuda") + 0.7 * torch.randn(1, E, generator=g, device="cuda")
    top, ids = torch.topk(logits, k, dim=1)
    ids[valid:] = -1
    return ids, torch.softmax(top, dim=1)


def _hidden(rows, cols, g):
    """Activations: unit scale with a few strong channels, bf16."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= 1.0 + 7.0 * (torch.rand(1, cols, generator=g, device="cuda") < 0.01)
    return x.to(torch.bfloat16)


def _weight(shape, g):
    """An fp8 weight [.., N, K] with one fp32 scale per 128 x 128 block, as a checkpoint holds it."""
    N, K = shape[-2:]
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    amax = 0.02 * (3.0 + 2.0 * torch.rand(*shape[:-2], nb, kb, generator=g, device="cuda"))
    scale = amax / FP8_MAX
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat, sflat = codes.view(-1, N, K), scale.view(-1, nb, kb)
    for e in range(flat.shape[0]):  # one expert at a time: bounded memory
        full = sflat[e].repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
        flat[e] = (0.02 * torch.randn(N, K, generator=g, device="cuda") / full).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return codes, scale


def _gate_up_weight(E, N, K, g):
    """Packed [.., 2N, K] codes (gate rows first); the two halves were quantised one by one: scales [.., 2 * ceil(N / 128), ceil(K / 128)]."""
    lead = (E,) if E else ()
    wg, sg = _weight((*lead, N, K), g)
    wu, su = _weight((*lead, N, K), g)
    return torch.cat([wg.view(torch.uint8), wu.view(torch.uint8)], dim=-2).view(torch.float8_e4m3fn), torch.cat([sg, su], dim=-2)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case)
    if op in ("dispatch", "combine") or (op == "quantize" and case["routed"]):
        ids, w = _route(case["T"], case["k"], case["E"], case["valid"], g)
        if op == "dispatch":
            s["ids"], s["x"] = ids, _hidden(case["T"], case["H"], g)
            if case["grad"]:
                s["dxs"] = _hidden(case["T"] * case["k"], case["H"], g)
            return s
        s["row_slot"], s["slot_row"], s["offsets"] = _sort(ids, case["E"])
        if op == "combine":
            s["w"], s["y"] = w, _hidden(case["T"] * case["k"], case["H"], g)
            if case["grad"]:
                s["dout"] = _hidden(case["T"], case["H"], g)
        else:
            s["x"] = _hidden(case["T"], case["K"], g)
        return s
    if op == "quantize":
        s["x"] = _hidden(case["M"], case["K"], g)
        return s
    E, N, K, rows = case["E"], case["N"], case["K"], case["M"] * case["k"]
    s["offsets"], s["bounds"] = None, [0, rows]
    if E:
        ids, _ = _route(case["M"], case["k"], E, case["valid"], g)
        s["offsets"] = _sort(ids, E)[2]
        s["bounds"] = s["offsets"].tolist()  # the plain form's loop over experts needs them on the host
    s["a"], s["a_scale"] = _quantize(_hidden(rows, K, g).float())
    if op == "gemm":
        s["b"], s["b_scale"] = _weight(((E,) if E else ()) + (N, K), g)
    else:
        s["b"], s["b_scale"] = _gate_up_weight(E, N, K, g)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _sort(ids, E):
    T, k = ids.shape
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True)[1]
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.cumsum(torch.bincount(key, minlength=E + 1)[:E], 0)
    here = torch.arange(T * k, device=ids.device)
    row_slot = torch.where(here < offsets[E], order, -1).to(torch.int32)
    slot_row = torch.empty_like(here)
    slot_row[order] = here
    slot_row = torch.where(key < E, slot_row, -1).to(torch.int32).reshape(T, k)
    return row_slot, slot_row, offsets


def _gather(x, row_slot, k):
    src = torch.div(row_slot.long(), k, rounding_mode="floor").clamp_min(0)
    return torch.where((row_slot >= 0).unsqueeze(1), x[src], torch.zeros((), dtype=x.dtype, device=x.device))


def _combine(y, w, slot_row):
    rows = y[slot_row.long().clamp_min(0)].float()  # [T, k, H]
    w = torch.where(slot_row >= 0, w, torch.zeros((), device=w.device))
    return (rows * w.unsqueeze(2)).sum(1)


def _quantize(x):
    """(codes, scales) of fp32 rows: s = max(amax / 448, 2^-126) per 128 columns, q = e4m3(x / s)."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    xp = torch.nn.functional.pad(x, (0, kb * BLOCK - K)).view(M, kb, BLOCK)
    top = xp.abs().amax(2)
    scale = (top / torch.full_like(top, FP8_MAX)).clamp_min(TINY)  # by a tensor: by a number it would be a product with 1 / 448
    codes = (xp / scale.unsqueeze(2)).to(torch.float8_e4m3fn)
    return codes.view(M, kb * BLOCK)[:, :K].contiguous(), scale


def _rows_f32(a, scale):
    return a.float() * scale.repeat_interleave(BLOCK, 1)[:, :a.shape[1]]


def _weight_f32(b, scale):
    return b.float() * scale.repeat_interleave(BLOCK, 0)[:b.shape[0]].repeat_interleave(BLOCK, 1)[:, :b.shape[1]]


def _halves_f32(b, scale):
    n, nb = b.shape[0] // 2, scale.shape[0] // 2
    return torch.cat([_weight_f32(b[:n], scale[:nb]), _weight_f32(b[n:], scale[nb:])])


def _product(s, weight):
    """fp32 rows of every expert's product; rows behind the last expert's are zero."""
    a = _rows_f32(s["a"], s["a_scale"])
    if s["offsets"] is None:
        return a @ weight(s["b"], s["b_scale"]).t()
    out = torch.zeros(a.shape[0], s["b"].shape[1], device=a.device)
    for e in range(s["E"]):
        lo, hi = s["bounds"][e], s["bounds"][e + 1]
        if hi > lo:
            out[lo:hi] = a[lo:hi] @ weight(s["b"][e], s["b_scale"][e]).t()
    return out


def _run_plain(s):
    op = s["op"]
    if op == "dispatch":
        row_slot, slot_row, offsets = _sort(s["ids"], s["E"])
        out = dict(row_slot=row_slot, slot_row=slot_row, offsets=offsets, xs=_gather(s["x"], row_slot, s["k"]))
        if s["grad"]:
            ones = torch.ones(s["T"], s["k"], device="cuda")
            out["dx"] = _combine(s["dxs"], ones, slot_row).to(torch.bfloat16)
        return out
    if op == "combine":
        out = dict(out=_combine(s["y"], s["w"], s["slot_row"]).to(torch.bfloat16))
        if s["grad"]:
            used = (s["row_slot"] >= 0).unsqueeze(1)
            slot = s["row_slot"].long().clamp_min(0)
            dout_rows = s["dout"][torch.div(slot, s["k"], rounding_mode="floor")].float()
            out["dy"] = torch.where(used, dout_rows * s["w"].reshape(-1)[slot].unsqueeze(1), 0.0).to(torch.bfloat16)
            dots = (dout_rows * s["y"].float()).sum(1)
            out["dw"] = torch.where(s["slot_row"] >= 0, dots[s["slot_row"].long().clamp_min(0)], 0.0)
        return out
    if op == "quantize":
        x = _gather(s["x"], s["row_slot"], s["k"]) if s["routed"] else s["x"]
        codes, scale = _quantize(x.float())
        return dict(codes=codes, scale=scale)
    if op == "gemm":
        return dict(c=_product(s, _weight_f32).to(torch.bfloat16))
    h = _product(s, _halves_f32)
    n = s["N"]
    g, u = h[:, :n], h[:, n:]
    codes, scale = _quantize(g / (1.0 + torch.exp(-g)) * u)
    return dict(codes=codes, scale=scale)


def _run_own(s):
    import magicompiler_b200 as mb

    op = s["op"]
    if op == "dispatch":
        row_slot, slot_row, offsets = mb.expert_sort_out(s["ids"], s["E"])
        out = dict(row_slot=row_slot, slot_row=slot_row, offsets=offsets)
        if s["grad"]:
            x = s["x"].detach().requires_grad_()
            xs = mb.expert_gather(x, row_slot, slot_row)
            out["xs"], (out["dx"],) = xs.detach(), torch.autograd.grad(xs, x, s["dxs"])
        else:
            out["xs"] = mb.expert_gather_out(s["x"], row_slot, slot_row)
        return out
    if op == "combine":
        if not s["grad"]:
            return dict(out=mb.expert_combine_out(s["y"], s["w"], s["row_slot"], s["slot_row"]))
        y, w = s["y"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        out = mb.expert_combine(y, w, s["row_slot"], s["slot_row"])
        dy, dw = torch.autograd.grad(out, (y, w), s["dout"])
        return dict(out=out.detach(), dy=dy, dw=dw)
    if op == "quantize":
        if s["routed"]:
            codes, scale = mb.expert_gather_fp8_out(s["x"], s["row_slot"], s["slot_row"])
        else:
            codes, scale = mb.quantize_fp8_block_out(s["x"])
        return dict(codes=codes, scale=scale)
    if op == "gemm":
        return dict(c=mb.gemm_fp8_block_out(s["a"], s["a_scale"], s["b"], s["b_scale"], s["offsets"]))
    codes, scale = mb.gemm_swiglu_fp8_block_out(s["a"], s["a_scale"], s["b"], s["b_scale"], s["offsets"])
    return dict(codes=codes, scale=scale)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    op = case["op"]
    if op in ("dispatch", "combine"):
        T, k, E, H = case["T"], case["k"], case["E"], case["H"]
        R = T * k
        live = case["valid"] * k
        if op == "dispatch":
            b = 8 * R + 8 * R + 4 * (E + 1) + 2 * case["valid"] * H + 2 * R * H
            return dict(bytes=b + (2 * live * H + 2 * T * H if case["grad"] else 0), flops=live * H if case["grad"] else 0)
        b = 4 * R + 4 * R + 2 * live * H + 2 * T * H
        # the training step: one read of y serves the sum and the router's gradient only if the two directions were one
        # pass; they are not (the loss lies between), so y is read in each
        return dict(bytes=b + (2 * live * H + 2 * case["valid"] * H + 2 * R * H + 12 * R if case["grad"] else 0),
                    flops=2 * live * H + (3 * live * H if case["grad"] else 0))
    if op == "quantize":
        K, kb = case["K"], -(-case["K"] // BLOCK)
        rows, src = (case["T"] * case["k"], case["valid"]) if case["routed"] else (case["M"], case["M"])
        return dict(bytes=2 * src * K + rows * (K + 4 * kb) + (8 * rows if case["routed"] else 0), flops=2 * rows * K)
    N, K, rows = case["N"], case["K"], case["M"] * case["k"]
    live = case["valid"] * case["k"]
    kb, nb = -(-K // BLOCK), -(-N // BLOCK)
    halves = 2 if op == "swiglu" else 1
    used = min(case["E"], live) if case["E"] else 1  # experts that can have rows
    b = live * (K + 4 * kb) + used * halves * (N * K + 4 * nb * kb)
    b += rows * (N + 4 * nb) if op == "swiglu" else 2 * rows * N
    return dict(bytes=b, flops=2 * live * N * K * halves)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(case, s):
    """Each row's product in 64 bits, straight from the definition: block sums of the codes, then the two scales."""
    E, K = case["E"], case["K"]
    n = s["b"].shape[-2]
    out = torch.zeros(s["a"].shape[0], n, dtype=torch.float64, device="cuda")
    bounds = s["bounds"]
    per_half = n // (2 if case["op"] == "swiglu" else 1)
    col = torch.arange(n, device="cuda")
    col_block = col % per_half // BLOCK + col // per_half * (-(-per_half // BLOCK))
    k_block = torch.arange(K, device="cuda") // BLOCK
    a = s["a"].to(torch.float64) * s["a_scale"].to(torch.float64)[:, k_block]
    for e in range(max(E, 1)):
        lo, hi = bounds[e], bounds[e + 1]
        if hi == lo:
            continue
        b, bs = (s["b"][e], s["b_scale"][e]) if E else (s["b"], s["b_scale"])
        for c in range(0, n, 8192):  # bounded memory
            cols = slice(c, min(n, c + 8192))
            w = b[cols].to(torch.float64) * bs.to(torch.float64)[col_block[cols]][:, k_block]
            out[lo:hi, cols] = a[lo:hi] @ w.t()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("dispatch", "combine") or (op == "quantize" and case["routed"]):
        if op == "dispatch":
            s["row_slot"], s["slot_row"], _ = _sort(s["ids"], case["E"])
        slot_row, k = s["slot_row"].long(), case["k"]
        token, j = torch.nonzero(slot_row >= 0, as_tuple=True)  # every slot that has an expert, and its row
        row = slot_row[token, j]
        R = case["T"] * k
    if op == "dispatch":
        xs = torch.zeros(R, case["H"], dtype=torch.float64, device="cuda")
        xs[row] = s["x"].double()[token]
        out = dict(row_slot=None, slot_row=None, offsets=None, xs=xs)
        if case["grad"]:
            dx = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
            out["dx"] = dx.index_add_(0, token, s["dxs"].double()[row])
        return out
    if op == "combine":
        w, y = s["w"].double(), s["y"].double()
        res = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
        out = dict(out=res.index_add_(0, token, y[row] * w[token, j].unsqueeze(1)))
        if case["grad"]:
            dout = s["dout"].double()
            dy = torch.zeros(R, case["H"], dtype=torch.float64, device="cuda")
            dy[row] = dout[token] * w[token, j].unsqueeze(1)
            dw = torch.zeros(case["T"], k, dtype=torch.float64, device="cuda")
            dw[token, j] = torch.einsum("rh,rh->r", dout[token], y[row])
            out.update(dy=dy, dw=dw)
        return out
    if op == "gemm":
        return dict(c=_exact_rows(case, s))
    if op == "quantize":
        v = s["x"].double()
        if case["routed"]:
            rows = torch.zeros(R, case["K"], dtype=torch.float64, device="cuda")
            rows[row] = v[token]
            v = rows
    else:
        h = _exact_rows(case, s)
        v = h[:, :case["N"]] * torch.sigmoid(h[:, :case["N"]]) * h[:, case["N"]:]
    scales, codes = [], torch.empty_like(v)
    for c in range(0, v.shape[1], BLOCK):
        part = v[:, c:c + BLOCK]
        top = torch.clamp(part.abs().max(1, keepdim=True)[0] / FP8_MAX, min=TINY)
        scales.append(top)
        codes[:, c:c + BLOCK] = part / top
    return dict(codes=codes, scale=torch.cat(scales, 1))
