"""Routed row movements and the block quantiser on the GPU, against plain formulas in 64 bits (the sort and the codes:
exactly).  Tolerances: a bf16 result of an fp32 sum is off by half a bf16 step of its value (2^-8) plus the fp32 sum's own
error, k or H terms at 2^-24 of their magnitudes each."""
import pytest
import torch

import magicompiler_b200 as mb

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def routing(T, k, E, seed=0, drop=0.0, skew=False, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 1 if skew else E, (T, k), generator=g)
    ids[torch.rand(T, k, generator=g) < drop] = -1
    return ids.to(dtype).cuda()


def sorted_plain(ids, E):
    flat = ids.cpu().long().reshape(-1)
    rows = [[] for _ in range(E)]
    for s, e in enumerate(flat.tolist()):
        if 0 <= e < E:
            rows[e].append(s)
    row_slot = [s for r in rows for s in r]
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    slot_row = [-1] * len(flat)
    for r, s in enumerate(row_slot):
        slot_row[s] = r
    row_slot += [-1] * (len(flat) - len(row_slot))
    return (torch.tensor(row_slot, dtype=torch.int32), torch.tensor(slot_row, dtype=torch.int32).view(ids.shape),
            torch.tensor(offsets, dtype=torch.int32))


def rows_of(n, h, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(n, h, generator=g)).to(BF).cuda()


def close_bf16(got, want64, magnitude64, terms):
    """|got - want| within half a bf16 step of want plus `terms` fp32 roundings of the summed magnitudes."""
    err = (got.double() - want64).abs()
    lim = want64.abs() * 2.0 ** -8 + magnitude64 * (terms + 1) * 2.0 ** -24 * (1 + 2.0 ** -8) + 2.0 ** -133
    assert (err <= lim).all(), (err - lim).max().item()


@pytest.mark.parametrize("T,k,E,drop", [
    (0, 2, 8, 0), (1, 1, 1, 0), (1, 2, 8, 0), (1, 8, 1024, 0), (5, 3, 4, 0.5), (33, 1, 2, 0), (128, 1, 1, 0),
    (257, 7, 130, 0.1), (1000, 8, 256, 0.9), (1024, 8, 8, 0), (1025, 8, 63, 0), (3000, 6, 1024, 0.2), (4099, 8, 128, 0.05),
    (16384, 8, 256, 0), (20001, 9, 33, 0.3)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort_is_the_stable_order(T, k, E, drop, dtype):
    ids = routing(T, k, E, seed=T + k, drop=drop, dtype=dtype)
    got = mb.expert_sort(ids, E)
    for g, w in zip(got, sorted_plain(ids, E)):
        assert g.dtype == torch.int32 and g.shape == w.shape and torch.equal(g.cpu(), w)


@pytest.mark.parametrize("case", ["all_one", "none", "out_of_range", "last_only", "strided"])
def test_sort_of_odd_ids(case):
    T, k, E = 700, 4, 16
    ids = routing(T, k, E, seed=3)
    if case == "all_one":
        ids[:] = 5
    elif case == "none":
        ids[:] = -1
    elif case == "out_of_range":
        ids[::3, 0], ids[1::3, 1], ids[2::3, 2] = E, 2 ** 40, -(2 ** 62)
    elif case == "last_only":
        ids[:], ids[-1, -1] = -1, E - 1
    else:
        ids = routing(k, T, E, seed=4).t()
    for g, w in zip(mb.expert_sort(ids, E), sorted_plain(ids, E)):
        assert torch.equal(g.cpu(), w)


MOVES = [(1, 1, 8, 1, 0), (1, 2, 4096, 8, 0), (3, 8, 136, 4, 0.4), (130, 3, 256, 7, 0.2), (257, 2, 8200, 3, 0), (31, 9, 512, 5, 0.1),
         (64, 17, 264, 30, 0), (2049, 8, 2048, 64, 0.05), (16, 4, 512, 8, 1.0)]


@pytest.mark.parametrize("T,k,H,E,drop", MOVES)
def test_gather_and_its_gradient(T, k, H, E, drop):
    ids = routing(T, k, E, seed=H, drop=drop)
    row_slot, slot_row, _ = mb.expert_sort(ids, E)
    x = rows_of(T, H, 1).requires_grad_()
    xs = mb.expert_gather(x, row_slot, slot_row)
    src = row_slot.long()
    want = torch.where((src >= 0)[:, None], x.detach()[src.clamp_min(0) // k], torch.zeros((), dtype=BF, device="cuda"))
    assert torch.equal(xs, want)
    assert torch.equal(mb.expert_gather_out(x.detach(), row_slot, slot_row), want)
    d = rows_of(T * k, H, 2)
    xs.backward(d)
    live = (slot_row >= 0)[:, :, None].double()
    terms = d.double()[slot_row.long().clamp_min(0)] * live
    close_bf16(x.grad, terms.sum(1), terms.abs().sum(1), k)


@pytest.mark.parametrize("T,k,H,E,drop", MOVES)
def test_combine_and_its_gradients(T, k, H, E, drop):
    ids = routing(T, k, E, seed=H + 1, drop=drop)
    row_slot, slot_row, _ = mb.expert_sort(ids, E)
    y = rows_of(T * k, H, 3).requires_grad_()
    w = torch.randn(T, k, generator=torch.Generator().manual_seed(4)).cuda().requires_grad_()
    out = mb.expert_combine(y, w, row_slot, slot_row)
    live = slot_row >= 0
    rows = y.detach().double()[slot_row.long().clamp_min(0)] * live[:, :, None]
    terms = rows * w.detach().double()[:, :, None]
    close_bf16(out, terms.sum(1), terms.abs().sum(1), k)
    assert torch.equal(out, mb.expert_combine_out(y.detach(), w.detach(), row_slot, slot_row))
    d = rows_of(T, H, 5)
    out.backward(d)
    slot = row_slot.long()
    dy = torch.where((slot >= 0)[:, None], w.detach().double().reshape(-1)[slot.clamp_min(0)][:, None] * d.double()[slot.clamp_min(0) // k], 0.0)
    close_bf16(y.grad, dy, dy.abs(), 1)
    prod = rows * d.double()[:, None, :]
    err = (w.grad.double() - prod.sum(2)).abs()
    assert w.grad.dtype == torch.float32
    assert (err <= prod.abs().sum(2) * (H + 1) * 2.0 ** -24).all()
    assert (w.grad[~live] == 0).all()


def test_gradients_agree_with_differences():
    """Both operators are linear in each argument: a difference quotient along a random direction has no truncation error.
    The outputs are exact here (small integers), so the quotient equals the gradient's inner product exactly."""
    T, k, H, E = 7, 3, 64, 4
    g = torch.Generator().manual_seed(0)
    small = lambda *s: torch.randint(-3, 4, s, generator=g).float().cuda()  # noqa: E731
    row_slot, slot_row, _ = mb.expert_sort(routing(T, k, E, seed=9, drop=0.2), E)
    x, dx, cot = small(T, H).to(BF), small(T, H).to(BF), small(T * k, H).to(BF)
    leaf = x.clone().requires_grad_()
    mb.expert_gather(leaf, row_slot, slot_row).backward(cot)
    diff = mb.expert_gather(x + dx, row_slot, slot_row).double() - mb.expert_gather(x, row_slot, slot_row).double()
    assert (diff * cot.double()).sum() == (leaf.grad.double() * dx.double()).sum()
    y, w, cot = small(T * k, H).to(BF), small(T, k), small(T, H).to(BF)
    ly, lw = y.clone().requires_grad_(), w.clone().requires_grad_()
    mb.expert_combine(ly, lw, row_slot, slot_row).backward(cot)
    base = mb.expert_combine(y, w, row_slot, slot_row).double()
    dy, dw = small(T * k, H).to(BF), small(T, k)
    diff = mb.expert_combine(y + dy, w, row_slot, slot_row).double() - base
    assert (diff * cot.double()).sum() == (ly.grad.double() * dy.double()).sum()
    diff = mb.expert_combine(y, w + dw, row_slot, slot_row).double() - base
    assert (diff * cot.double()).sum() == (lw.grad.double() * dw.double()).sum()


def test_only_the_gradient_that_is_asked_for():
    T, k, H, E = 40, 2, 128, 4
    row_slot, slot_row, _ = mb.expert_sort(routing(T, k, E), E)
    y, w, d = rows_of(T * k, H, 1), torch.rand(T, k, device="cuda"), rows_of(T, H, 2)
    both_y, both_w = y.clone().requires_grad_(), w.clone().requires_grad_()
    mb.expert_combine(both_y, both_w, row_slot, slot_row).backward(d)
    one = y.clone().requires_grad_()
    mb.expert_combine(one, w, row_slot, slot_row).backward(d)
    assert torch.equal(one.grad, both_y.grad)
    one = w.clone().requires_grad_()
    mb.expert_combine(y, one, row_slot, slot_row).backward(d)
    assert torch.equal(one.grad, both_w.grad)
    one = y.clone().requires_grad_()  # no weights: the adjoint of the sum is the gather
    mb.expert_combine(one, None, row_slot, slot_row).backward(d)
    assert torch.equal(one.grad, mb.expert_gather(d, row_slot, slot_row))


def test_broadcast_and_strided_operands():
    T, k, H, E = 50, 2, 256, 4
    row_slot, slot_row, _ = mb.expert_sort(routing(T, k, E, drop=0.1), E)
    wide = rows_of(T, H + 64, 1)
    assert torch.equal(mb.expert_gather(wide[:, 32:32 + H], row_slot, slot_row),
                       mb.expert_gather(wide[:, 32:32 + H].contiguous(), row_slot, slot_row))
    odd = rows_of(T, H + 3, 2)[:, 3:]  # neither the base nor the stride is aligned: copied
    assert torch.equal(mb.expert_gather(odd, row_slot, slot_row), mb.expert_gather(odd.contiguous(), row_slot, slot_row))
    y = rows_of(T * k, H, 3).requires_grad_()
    mb.expert_combine(y, None, row_slot, slot_row).sum().backward()  # an expanded, stride-0 gradient
    assert torch.equal(y.grad, (row_slot >= 0)[:, None].to(BF).expand(-1, H))
    w = torch.rand(k, T, device="cuda").t()
    assert torch.equal(mb.expert_combine(y.detach(), w, row_slot, slot_row),
                       mb.expert_combine(y.detach(), w.contiguous(), row_slot, slot_row))


def unaligned(t):
    """The same values, contiguous, two bytes past a 16-byte boundary."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)[1:1 + t.numel()]
    assert flat.data_ptr() % 16 == 2
    return flat.copy_(t.reshape(-1)).view(t.shape)


def test_contiguous_operands_and_gradients_off_a_16_byte_boundary():
    T, k, H, E = 50, 2, 256, 4
    row_slot, slot_row, _ = mb.expert_sort(routing(T, k, E, drop=0.1), E)
    x, y, w, dx, dy = rows_of(T, H, 1), rows_of(T * k, H, 2), torch.rand(T, k, device="cuda"), rows_of(T * k, H, 3), rows_of(T, H, 4)
    for form in (mb.expert_gather, mb.expert_gather_fp8, torch.ops.magi_swiglu.expert_gather):
        got, want = form(unaligned(x), row_slot, slot_row), form(x, row_slot, slot_row)
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a.float(), b.float())
    for a, b in zip(mb.quantize_fp8_block(unaligned(x)), mb.quantize_fp8_block(x)):
        assert torch.equal(a.float(), b.float())
    assert torch.equal(mb.expert_combine(unaligned(y), w, row_slot, slot_row), mb.expert_combine(y, w, row_slot, slot_row))

    def gradients(ddx, ddy):
        lx, ly, lw = x.clone().requires_grad_(), y.clone().requires_grad_(), w.clone().requires_grad_()
        return (*torch.autograd.grad(mb.expert_gather(lx, row_slot, slot_row), lx, ddx),
                *torch.autograd.grad(mb.expert_combine(ly, lw, row_slot, slot_row), (ly, lw), ddy))

    for a, b in zip(gradients(unaligned(dx), unaligned(dy)), gradients(dx, dy)):
        assert torch.equal(a, b)


def test_masked_slots_may_hold_anything():
    T, k, H, E = 20, 4, 128, 4
    ids = routing(T, k, E, drop=0.5, seed=8)
    ids[3] = -1  # a token without any expert
    row_slot, slot_row, offsets = mb.expert_sort(ids, E)
    y, w = rows_of(T * k, H, 1), torch.rand(T, k, device="cuda")
    clean = mb.expert_combine(y, w, row_slot, slot_row)
    y2, w2 = y.clone(), w.clone()
    y2[offsets[-1]:] = float("nan")
    w2[slot_row < 0] = float("inf")
    assert torch.equal(mb.expert_combine(y2, w2, row_slot, slot_row), clean) and (clean[3] == 0).all()
    d = rows_of(T, H, 2)
    got = mb.expert_combine_backward(d, y2, w2, row_slot, slot_row, True, True)
    want = mb.expert_combine_backward(d, y, w, row_slot, slot_row, True, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (want[1][3] == 0).all()
    dg = rows_of(T * k, H, 3)
    dg2 = dg.clone()
    dg2[offsets[-1]:] = float("nan")
    assert torch.equal(mb.expert_combine(dg2, None, row_slot, slot_row), mb.expert_combine(dg, None, row_slot, slot_row))


def test_indices_out_of_range_touch_nothing_outside():
    """Bad index arrays are no-expert entries: guard rows around the output stay as they were."""
    T, k, H = 6, 2, 64
    slot_row = torch.tensor([[0, 99], [-7, 1], [2, 12], [3, 4], [5, 6], [2 ** 31 - 1, 7]], dtype=torch.int32, device="cuda")
    row_slot = torch.arange(12, dtype=torch.int32, device="cuda")
    guard = torch.full((14, H), 7.0, dtype=BF, device="cuda")
    x = rows_of(T, H, 1)
    mb.expert_gather_out(x, row_slot, slot_row, out=guard[1:13])
    assert (guard[0] == 7).all() and (guard[13] == 7).all()
    for t, j, r in ((0, 0, 0), (1, 1, 1), (2, 0, 2), (5, 1, 7)):
        assert torch.equal(guard[1 + r], x[t]), (t, j)
    y = rows_of(T * k, H, 2)
    assert torch.equal(mb.expert_combine(y, None, row_slot, slot_row)[0], y[0])


def test_a_row_whose_slot_is_out_of_range_holds_none():
    """As for -1: zero rows, zero codes and the smallest scale, zero gradients, also in memory that held something else."""
    T, k, H = 6, 2, 256
    ids = torch.arange(T * k, device="cuda").view(T, k) % 3
    ids[4:] = -1
    row_slot, slot_row, offsets = mb.expert_sort(ids, 3)
    n, bad = int(offsets[-1]), row_slot.clone()
    bad[n:] = torch.tensor([T * k, 2 ** 31 - 1, -1, -(2 ** 31)], dtype=torch.int32, device="cuda")
    x, y, w, d = rows_of(T, H, 1), rows_of(T * k, H, 2), torch.rand(T, k, device="cuda"), rows_of(T, H, 3)
    xs = mb.expert_gather_out(x, bad, slot_row, out=torch.full((T * k, H), 7.0, dtype=BF, device="cuda"))
    assert torch.equal(xs, mb.expert_gather(x, row_slot, slot_row)) and (xs[n:] == 0).all()
    filled = (torch.full((T * k, H), 7.0, device="cuda").to(torch.float8_e4m3fn), torch.full((T * k, 2), 7.0, device="cuda"))
    codes, scales = mb.expert_gather_fp8_out(x, bad, slot_row, out=filled)
    assert (codes[n:].float() == 0).all() and (scales[n:] == 2.0 ** -126).all()
    assert torch.equal(codes.float(), mb.expert_gather_fp8(x, row_slot, slot_row)[0].float())
    torch.full((T * k, H), float("nan"), dtype=BF, device="cuda")  # the block that dy is likely to get
    dy, _ = mb.expert_combine_backward(d, y, w, bad, slot_row, True, False)
    assert torch.equal(dy, mb.expert_combine_backward(d, y, w, row_slot, slot_row, True, False)[0]) and (dy[n:] == 0).all()


def plain_quantise(x):
    """The formula in fp32, element by element (IEEE divisions)."""
    M, K = x.shape
    kb = -(-K // 128)
    v = torch.zeros(M, kb * 128, device=x.device)
    v[:, :K] = x.float()
    v = v.view(M, kb, 128)
    s = v.abs().amax(2)
    s = s / torch.full_like(s, 448.0)  # by a tensor: on a GPU torch turns a division by a number into a product with 1 / 448
    s = torch.where(s < 2.0 ** -126, torch.full_like(s, 2.0 ** -126), s)
    return (v / s[:, :, None]).to(torch.float8_e4m3fn).view(M, kb * 128)[:, :K], s


def same_codes(a, b):
    fa, fb = a.float(), b.float()
    return bool(((fa == fb) | (fa.isnan() & fb.isnan())).all())


@pytest.mark.parametrize("M,K", [(0, 128), (1, 16), (1, 128), (3, 144), (7, 2064), (130, 4096), (300, 8208), (1023, 512)])
def test_quantiser_is_the_formula_bit_for_bit(M, K):
    x = rows_of(M, K, M + K, scale=3.0)
    x *= torch.exp2(torch.randint(-20, 20, (1, K), generator=torch.Generator().manual_seed(1)).float()).cuda().to(BF)
    codes, scales = mb.quantize_fp8_block(x)
    wc, ws = plain_quantise(x)
    assert codes.dtype == torch.float8_e4m3fn and torch.equal(scales, ws)
    assert torch.equal(codes.float(), wc.float())


def test_quantiser_of_every_bf16_value():
    """Each finite bf16 value against every power-of-two and odd block maximum near it: ties at e4m3 midpoints included."""
    bits = torch.arange(0x0001, 0x7f80, dtype=torch.int32).to(torch.int16)
    vals = bits.view(BF).cuda()
    n = vals.numel() // 127 * 127
    x = torch.empty(n // 127, 128, dtype=BF, device="cuda")
    x[:, :127] = vals[:n].view(-1, 127) * -1
    for top in (1, 28, 448, 3, 251):  # the last column sets the maximum of rows that are below it
        x[:, 127] = top
        codes, scales = mb.quantize_fp8_block(x)
        wc, ws = plain_quantise(x)
        assert torch.equal(scales, ws) and torch.equal(codes.float(), wc.float())


def test_quantiser_of_every_bf16_value_with_a_maximum_near_it():
    """Each positive finite bf16 value in a block whose maximum is a multiple of it: powers of two, odd ones, and those that put
    the quotient at the middle between two codes (448 / c for c = 17, 19, .. 31 sixteenths)."""
    vals = torch.arange(0x0001, 0x7f80, dtype=torch.int32).to(torch.int16).view(BF).cuda()
    factors = [1, 2, 4, 64, 2 ** 9, 2 ** 17, 2 ** 19, 3, 5, 7, 28, 251, 448] + [448 * 16 / c for c in range(17, 32, 2)]
    tops = (vals.float()[:, None] * torch.tensor(factors, device="cuda")).to(BF)
    for sign in (1, -1):
        x = torch.zeros(vals.numel(), len(factors), 128, dtype=BF, device="cuda")
        x[:, :, 5], x[:, :, 127] = sign * vals[:, None], tops
        x = x.view(vals.numel(), -1)
        codes, scales = mb.quantize_fp8_block(x)
        wc, ws = plain_quantise(x)
        assert torch.equal(scales, ws) and same_codes(codes, wc)


def test_quantiser_of_every_pair_of_mantissas():
    """The quotient x / s takes one correction step instead of a division: each of the 128 bf16 mantissas of x against each
    of the 128 of the block's maximum, at every distance of exponents that gives a code other than zero, at scales near
    both ends of the corrected range, in the middle and outside."""
    mant = (1.0 + torch.arange(128) / 128.0).cuda()
    for power in (-118, -100, -92, -91, 0, 100, 119, 126):
        for down in range(1, 20):
            x = torch.zeros(128, 256, device="cuda")
            x[:, 0] = x[:, 128] = mant * 2.0 ** power
            x[:, 1:128], x[:, 129] = mant[:127] * 2.0 ** (power - down), mant[127] * 2.0 ** (power - down)
            x = x.to(BF)
            codes, scales = mb.quantize_fp8_block(x)
            wc, ws = plain_quantise(x)
            assert torch.equal(scales, ws) and torch.equal(codes.float(), wc.float()), (power, down)


@pytest.mark.parametrize("power", [-73, -72, -71, -70])
def test_quantiser_where_corrected_products_take_over_from_divisions(power):
    """Blocks whose scale lies on either side of 2^-80: every pair of mantissas again."""
    mant = (1.0 + torch.arange(128) / 128.0).cuda()
    for down in range(1, 20):
        x = torch.zeros(128, 128, device="cuda")
        x[:, :] = mant * 2.0 ** (power - down)
        x[:, 0] = mant * 2.0 ** power
        x = x.to(BF)
        codes, scales = mb.quantize_fp8_block(x)
        wc, ws = plain_quantise(x)
        assert torch.equal(scales, ws) and torch.equal(codes.float(), wc.float())


def test_quantiser_of_special_values():
    x = rows_of(8, 256, 1)
    x[0, 3], x[1, 200], x[2, 5], x[3], x[4, :128] = float("nan"), float("inf"), float("-inf"), 0, 1e-40
    x[5, 0], x[6, 0] = 3.38e38, -3.38e38
    codes, scales = mb.quantize_fp8_block(x)
    wc, ws = plain_quantise(x)
    assert torch.equal(scales.isnan(), ws.isnan()) and torch.equal(scales.nan_to_num(1), ws.nan_to_num(1))
    assert same_codes(codes, wc)
    assert codes[0, :128].float().isnan().all() and not codes[0, 128:].float().isnan().any()
    assert (codes[3].float() == 0).all() and (scales[3] == 2.0 ** -126).all()


@pytest.mark.parametrize("T,k,K,E,drop", [(1, 1, 16, 1, 0), (1, 8, 2048, 64, 0), (5, 3, 144, 4, 0.5), (130, 2, 4112, 8, 0.1),
                                          (1001, 6, 512, 33, 0.2), (9, 2, 256, 3, 1.0)])
def test_quantised_gather_is_the_gather_quantised(T, k, K, E, drop):
    row_slot, slot_row, _ = mb.expert_sort(routing(T, k, E, seed=K, drop=drop), E)
    x = rows_of(T, K, 6)
    codes, scales = mb.expert_gather_fp8(x, row_slot, slot_row)
    wc, ws = mb.quantize_fp8_block(mb.expert_gather(x, row_slot, slot_row))
    assert torch.equal(codes.view(torch.uint8), wc.view(torch.uint8)) and torch.equal(scales, ws)


def test_captured_and_replayed_with_new_routing():
    """Sort, gather and combine in one CUDA graph, replayed on new ids, rows and weights; two graphs alternate."""
    T, k, H, E = 65, 4, 512, 8

    def build(seed):
        s = dict(ids=routing(T, k, E, seed=seed), x=rows_of(T, H, seed), w=torch.rand(T, k, device="cuda"))

        def step():
            row_slot, slot_row, off = mb.expert_sort_out(s["ids"], E)
            s["xs"] = mb.expert_gather_out(s["x"], row_slot, slot_row)
            s["q"] = mb.expert_gather_fp8_out(s["x"], row_slot, slot_row)
            s["out"], s["off"] = mb.expert_combine_out(s["xs"], s["w"], row_slot, slot_row), off

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        return s, graph

    a, b = build(1), build(2)
    for turn in range(3):
        for i, (s, graph) in enumerate((a, b)):
            s["ids"].copy_(routing(T, k, E, seed=50 + 7 * turn + i, drop=0.2))
            s["x"].copy_(rows_of(T, H, 90 + turn + i))
            graph.replay()
        for s, _ in (a, b):
            row_slot, slot_row, off = mb.expert_sort(s["ids"], E)
            xs = mb.expert_gather(s["x"], row_slot, slot_row)
            assert torch.equal(s["off"], off) and torch.equal(s["xs"], xs)
            assert torch.equal(s["out"], mb.expert_combine(xs, s["w"], row_slot, slot_row))
            assert torch.equal(s["q"][0].float(), mb.quantize_fp8_block(xs)[0].float())


def test_on_a_side_stream():
    T, k, H, E = 513, 2, 1024, 8
    ids, x, w = routing(T, k, E), rows_of(T, H, 1), torch.rand(T, k, device="cuda")
    want = None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            row_slot, slot_row, _ = mb.expert_sort(ids, E)
            got = mb.expert_combine(mb.expert_gather(x, row_slot, slot_row), w, row_slot, slot_row)
        torch.cuda.current_stream().wait_stream(stream)
        want = got if want is None else want
        assert torch.equal(got, want)


def test_a_captured_step_with_its_gradients():
    """Forward and backward in one graph, replayed with new routing, rows and weights; leaves are made inside the capture."""
    T, k, H, E = 40, 3, 256, 6
    static = dict(ids=routing(T, k, E), x=rows_of(T, H, 1), w=torch.rand(T, k, device="cuda"), dout=rows_of(T, H, 2))

    def step(ids, x, w, dout):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        row_slot, slot_row, _ = mb.expert_sort_out(ids, E)
        out = mb.expert_combine(mb.expert_gather(x, row_slot, slot_row), w, row_slot, slot_row)
        return (out.detach(), *torch.autograd.grad(out, (x, w), dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(**static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(**static)
    for seed in (5, 6):
        new = dict(ids=routing(T, k, E, seed=seed, drop=0.2), x=rows_of(T, H, seed), w=torch.rand(T, k, device="cuda"),
                   dout=rows_of(T, H, seed + 10))
        want = step(**new)
        for name, t in new.items():
            static[name].copy_(t)
        graph.replay()
        for g, r in zip(got, want):
            assert torch.equal(g, r)


def test_out_arguments():
    T, k, H, E = 12, 2, 64, 4
    ids = routing(T, k, E)
    out = (torch.empty(T * k, dtype=torch.int32, device="cuda"), torch.empty(T, k, dtype=torch.int32, device="cuda"),
           torch.empty(E + 1, dtype=torch.int32, device="cuda"))
    got = mb.expert_sort_out(ids, E, out=out)
    assert all(a is b for a, b in zip(got, out))
    x = rows_of(T, H, 1)
    for bad in (torch.empty(T * k, H, device="cuda"), torch.empty(T, H, dtype=BF, device="cuda"),
                torch.empty(T * k, 2 * H, dtype=BF, device="cuda")[:, :H],
                torch.empty(T * k * H + 1, dtype=BF, device="cuda")[1:].view(T * k, H)):
        with pytest.raises(ValueError, match="out must be"):
            mb.expert_gather_out(x, out[0], out[1], out=bad)
    codes, scales = torch.empty(T, H, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(T, 1, device="cuda")
    assert mb.quantize_fp8_block_out(x, out=(codes, scales))[0] is codes
    with pytest.raises(TypeError, match="CUDA tensors only"):
        mb.expert_gather_out(x, out[0].cpu(), out[1])


def test_results_that_overlap_operands_are_refused():
    """With one choice a token the shapes agree, so an in-place permutation looks possible: the kernels read after they write."""
    T, k, H, E = 12, 1, 128, 4
    ids = routing(T, k, E).int()
    row_slot, slot_row, offsets = mb.expert_sort(ids, E)
    x = rows_of(T, H, 1)
    new = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="cuda")
    codes, scales = mb.quantize_fp8_block(x)
    w, ws = mb.quantize_fp8_weight(rows_of(H, H, 2))
    w13, w13s = mb.quantize_fp8_gate_up(rows_of(2 * H, H, 3))
    raw = codes.view(torch.uint8)
    shared = torch.empty(T * H * 2, dtype=torch.uint8, device="cuda")
    for call in (lambda: mb.expert_sort_out(ids, E, out=(row_slot, ids, offsets)),
                 lambda: mb.expert_sort_out(ids, T - 1, out=(row_slot, new(T, k), row_slot)),
                 lambda: mb.expert_gather_out(x, row_slot, slot_row, out=x),
                 lambda: mb.expert_combine_out(x, None, row_slot, slot_row, out=x),
                 lambda: mb.expert_gather_fp8_out(x, row_slot, slot_row, out=(x.view(torch.float8_e4m3fn).view(-1)[T * H:].view(T, H), scales)),
                 lambda: mb.quantize_fp8_block_out(x, out=(codes, raw.view(-1)[:4 * T].view(torch.float32).view(T, 1))),
                 lambda: mb.gemm_fp8_block_out(shared[:T * H].view(torch.float8_e4m3fn).view(T, H), scales, w, ws,
                                               out=shared.view(BF).view(T, H)),
                 lambda: mb.gemm_swiglu_fp8_block_out(codes, scales, w13, w13s, out=(codes, new(T, 1).float())),
                 lambda: mb.gemm_swiglu_fp8_block_out(codes, scales, w13, w13s, out=(torch.empty_like(codes), scales))):
        with pytest.raises(ValueError, match="overlap"):
            call()
    both = torch.empty(2 * T, H, dtype=BF, device="cuda")  # neighbours in one buffer are apart
    both[:T] = x
    assert torch.equal(mb.expert_gather_out(both[:T], row_slot, slot_row, out=both[T:]), mb.expert_gather(x, row_slot, slot_row))


def test_offsets_past_32_bits():
    """More than 2^31 elements on the experts' side: the last rows are right in every direction."""
    T, k, H, E = 66000, 4, 8192, 16
    ids = torch.randint(0, E, (T, k), generator=torch.Generator().manual_seed(1)).cuda()
    row_slot, slot_row, _ = mb.expert_sort(ids, E)
    assert T * k * H > 2 ** 31
    x = torch.randn(T, 1, generator=torch.Generator().manual_seed(2)).to(BF).cuda().expand(T, H).contiguous()
    xs = mb.expert_gather(x, row_slot, slot_row)
    assert torch.equal(xs[:, 0], x[row_slot.long() // k, 0]) and torch.equal(xs[:, -1], xs[:, 0])
    w = torch.full((T, k), 0.25, device="cuda")
    assert torch.equal(mb.expert_combine(xs, w, row_slot, slot_row), x)
    dy, dw = mb.expert_combine_backward(x, xs, w, row_slot, slot_row, True, True)
    assert torch.equal(dy[:, 0], (0.25 * xs[:, 0]).to(BF)) and torch.equal(dy[:, -1], dy[:, 0])
    want = (x[:, 0].double() ** 2 * H)[:, None].expand(T, k)
    assert ((dw.double() - want).abs() <= want * (H + 1) * 2.0 ** -24).all()
    del dy, dw, xs
    codes, scales = mb.expert_gather_fp8(x, row_slot, slot_row)
    full = mb.quantize_fp8_block(x)
    assert torch.equal(codes[:, -1].float(), full[0][row_slot.long() // k, -1].float())
    assert torch.equal(scales[:, -1], full[1][row_slot.long() // k, -1])
