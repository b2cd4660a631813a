"""Block-scaled fp8 products against the formula in 64 bits.

Tolerance of a sum.  The products of e4m3 codes are exact in fp32.  Let A = sum |terms|, scaled.  The tensor cores add the
128 products of a block in fp32 steps that may truncate (one unit, 2^-23, a step; at most 128 steps), the two scales'
product and the multiply-add round once each (2^-24), and the additions over the K blocks at most ceil(K/128) + 8 times:
|error| <= A * (128 + ceil(K/128) + 10) * 2^-23.  A bf16 result adds half a bf16 step of its own value, 2^-8.
SwiGLU: |d(silu(g) u)| <= 1.1 |u| dg + |silu(g)| du (|silu'| < 1.1) plus 2^-20 of the value for the exponential, the
reciprocal and the products.  A scale is 1/448 of the largest of 128 such values, a code is within half an e4m3 step
(2^-4 of the value, or 2^-10 of the scale below the smallest normal code) of value / scale."""
import contextlib

import pytest
import torch

import magicompiler_b200 as mb
from magicompiler_b200 import _loader

pytestmark = pytest.mark.gpu
F8, BF = torch.float8_e4m3fn, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes_of(shape, seed, spread=1.0):
    return (spread * torch.randn(*shape, generator=gen(seed), device="cuda")).clamp(-448, 448).to(F8)


def scales_of(shape, seed):
    return torch.exp2(4 * torch.rand(*shape, generator=gen(seed), device="cuda") - 6)


def wide(codes, scales, rows_per_scale):
    s = scales.double()
    s = s.repeat_interleave(rows_per_scale, -2)[..., :codes.shape[-2], :] if rows_per_scale > 1 else s
    return codes.double() * s.repeat_interleave(128, -1)[..., :codes.shape[-1]]


def case(M, N, K, E=0, halves=1, seed=0, counts=None):
    lead = (E,) if E else ()
    kb, nb = -(-K // 128), -(-N // 128)
    t = dict(a=codes_of((M, K), seed, 2.0), a_scale=scales_of((M, kb), seed + 1))
    t["b"], t["b_scale"] = codes_of((*lead, halves * N, K), seed + 2), scales_of((*lead, halves * nb, kb), seed + 3)
    t["offsets"] = None
    if E:
        t["offsets"] = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")
    return t


def sums(t, halves=1):
    """(sum, sum of magnitudes) [M, halves * N] in 64 bits; rows behind the last expert are zero."""
    a = wide(t["a"], t["a_scale"], 1)
    outs = []
    for x, mag in ((a, False), (a.abs(), True)):
        def product(rows, b, bs):
            n, nb = b.shape[0] // halves, bs.shape[0] // halves
            w = torch.cat([wide(b[h * n:(h + 1) * n], bs[h * nb:(h + 1) * nb], 128) for h in range(halves)])
            return rows @ (w.abs() if mag else w).t()
        if t["offsets"] is None:
            outs.append(product(x, t["b"], t["b_scale"]))
            continue
        out = torch.zeros(a.shape[0], t["b"].shape[1], dtype=torch.float64, device="cuda")
        off = t["offsets"].tolist()
        for e in range(len(off) - 1):
            out[off[e]:off[e + 1]] = product(x[off[e]:off[e + 1]], t["b"][e], t["b_scale"][e])
        outs.append(out)
    return outs


def slack(mag, K):
    return mag * (128 + -(-K // 128) + 10) * 2.0 ** -23


def check_plain(t, got):
    K = t["a"].shape[1]
    want, mag = sums(t)
    lim = want.abs() * 2.0 ** -8 + slack(mag, K) * (1 + 2.0 ** -8) + 2.0 ** -133
    err = (got.double() - want).abs()
    assert got.dtype == BF and got.shape == want.shape
    assert (err <= lim).all(), (err - lim).max().item()


def check_fused(t, codes, scales):
    K, N = t["a"].shape[1], codes.shape[1]
    h, mag = sums(t, 2)
    g, u, dg, du = h[:, :N], h[:, N:], slack(mag[:, :N], K), slack(mag[:, N:], K)
    silu = g * torch.sigmoid(g)
    y = silu * u
    dy = 1.1 * (u.abs() + du) * dg + silu.abs() * du + y.abs() * 2.0 ** -20
    nb = -(-N // 128)
    pad = lambda v: torch.nn.functional.pad(v, (0, nb * 128 - N)).view(-1, nb, 128)  # noqa: E731
    top, slop = pad(y.abs()).amax(2), pad(dy).amax(2)
    floor = torch.full_like(top, 2.0 ** -126)
    s = scales.double()
    assert codes.dtype == F8 and scales.dtype == torch.float32 and tuple(scales.shape) == tuple(top.shape)
    assert (s <= torch.maximum((top + slop) / 448, floor) * (1 + 2.0 ** -23)).all()
    assert (s >= torch.maximum((top - slop) / 448, floor) * (1 - 2.0 ** -23)).all()
    full = s.repeat_interleave(128, 1)[:, :N]
    err = (codes.double() * full - y).abs()
    lim = (y.abs() + dy) * 2.0 ** -4 + full * 2.0 ** -10 + dy * 1.001 + y.abs() * 2.0 ** -21
    assert (err <= lim).all(), (err - lim).max().item()


DENSE = [(1, 8, 16), (1, 128, 128), (1, 264, 144), (3, 136, 400), (16, 256, 512), (17, 384, 256), (31, 1000, 1040), (33, 128, 2048),
         (64, 520, 384), (65, 256, 640), (127, 136, 272), (128, 256, 256), (129, 264, 1152), (200, 2048, 512), (257, 776, 912),
         (300, 256, 4096), (513, 512, 384), (1000, 392, 1296), (2049, 1024, 256), (5, 4096, 8192),
         (300, 264, 2064), (260, 1032, 4112), (700, 136, 8192), (1030, 4096, 2048)]


@pytest.mark.parametrize("M,N,K", DENSE)
def test_dense(M, N, K):
    t = case(M, N, K, seed=M + N)
    check_plain(t, mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"]))


@pytest.mark.parametrize("M,N,K", [(m, -(-n // 16) * 16, k) for m, n, k in DENSE])
def test_dense_swiglu(M, N, K):
    t = case(M, N, K, halves=2, seed=M + N)
    check_fused(t, *mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"]))


GROUPED = [(1, [1], 0), (2, [0, 1], 0), (8, [0, 3, 0, 1, 17, 0, 2, 0], 5), (4, [130, 1, 64, 33], 0), (3, [0, 0, 0], 40),
           (2, [300, 257], 7), (5, [256, 512, 1, 255, 600], 300), (40, [i % 7 for i in range(40)], 1), (1, [700], 20),
           (70, [0] * 69 + [20], 0), (64, [9] * 64, 70)]


@pytest.mark.parametrize("E,counts,tail", GROUPED)
@pytest.mark.parametrize("N,K", [(136, 272), (256, 512)])
def test_experts(E, counts, tail, N, K):
    t = case(sum(counts) + tail, N, K, E=E, counts=counts, seed=E)
    got = mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    check_plain(t, got)
    assert (got[sum(counts):] == 0).all()


@pytest.mark.parametrize("E,counts,tail", GROUPED)
@pytest.mark.parametrize("N,K", [(144, 272), (256, 512)])
def test_experts_swiglu(E, counts, tail, N, K):
    t = case(sum(counts) + tail, N, K, E=E, counts=counts, halves=2, seed=E)
    codes, scales = mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    check_fused(t, codes, scales)
    assert (codes[sum(counts):].float() == 0).all() and (scales[sum(counts):] == 2.0 ** -126).all()


@pytest.mark.parametrize("halves,N,K", [(1, 2048, 256), (1, 1992, 640), (2, 1040, 256)])
def test_many_experts_with_a_few_rows_each(halves, N, K):
    counts, tail = [(0, 1, 2, 17, 0)[i % 5] for i in range(60)], 3
    t = case(sum(counts) + tail, N, K, E=60, counts=counts, halves=halves, seed=K)
    args = (t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    if halves == 1:
        check_plain(t, mb.gemm_fp8_block(*args))
    else:
        check_fused(t, *mb.gemm_swiglu_fp8_block(*args))


@pytest.mark.parametrize("halves,N,K", [(1, 2056, 128), (1, 2048, 400), (1, 2040, 256), (1, 4088, 1056), (2, 1040, 128),
                                        (2, 1024, 272), (2, 1008, 272), (2, 4080, 1056)])
def test_uneven_experts_with_half_empty_groups(halves, N, K):
    """Sizes at which tiles of 128 rows are expected to beat those of 256: an empty expert, one row over a group, a tail; the
    result does not depend on what the neighbouring experts' rows hold, guard rows stay."""
    counts, tail = [1003, 0, 129, 855], 13
    n = sum(counts)
    t = case(n + tail, N, K, E=4, counts=counts, halves=halves, seed=N)
    args = (t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    if halves == 1:
        got = mb.gemm_fp8_block(*args)
        check_plain(t, got)
        assert (got[n:] == 0).all()
        out = torch.full((n + tail + 2, N), 7.0, dtype=BF, device="cuda")
        mb.gemm_fp8_block_out(*args, out=out[1:-1])
        assert torch.equal(out[1:1 + n], got[:n]) and (out[0] == 7).all() and (out[1 + n:] == 7).all()
    else:
        codes, scales = mb.gemm_swiglu_fp8_block(*args)
        check_fused(t, codes, scales)
        assert (codes[n:].float() == 0).all() and (scales[n:] == 2.0 ** -126).all()
        got = codes
    t["a"].view(torch.uint8)[1003:1003 + 129] = 127  # NaN in e4m3: all of the third expert
    again = (mb.gemm_fp8_block if halves == 1 else lambda *x: mb.gemm_swiglu_fp8_block(*x)[0])(*args)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[1003:1003 + 129] = False
    assert torch.equal(again[:n][keep].view(torch.uint8), got[:n][keep].view(torch.uint8))
    assert again[:n][~keep].float().isnan().all()


@pytest.mark.parametrize("N,K", [(272, 2064), (144, 4112)])
def test_few_tiles_with_many_k_blocks(N, K):
    """Experts whose tiles share their K blocks among several CTA pairs, one of them empty, one with a partial group."""
    counts, tail = [300, 0, 257, 100], 9
    t = case(sum(counts) + tail, N, K, E=4, counts=counts)
    got = mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    check_plain(t, got)
    assert (got[sum(counts):] == 0).all()
    t = case(sum(counts) + tail, N, K, E=4, counts=counts, halves=2)
    codes, scales = mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    check_fused(t, codes, scales)
    assert (codes[sum(counts):].float() == 0).all() and (scales[sum(counts):] == 2.0 ** -126).all()


@pytest.mark.parametrize("M,E,counts", [(20, 3, [4, 0, 7]), (700, 3, [300, 0, 257])])
def test_rows_behind_the_last_expert_stay_with_out(M, E, counts):
    n = sum(counts)
    t = case(M, 256, 272, E=E, counts=counts)
    out = torch.full((M, 256), 7.0, dtype=BF, device="cuda")
    assert mb.gemm_fp8_block_out(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"], out=out) is out
    assert torch.equal(out[:n], mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])[:n])
    assert (out[n:] == 7).all()
    t = case(M, 256, 272, E=E, counts=counts, halves=2)
    codes, scales = torch.full((M, 256), 3.0, device="cuda").to(F8), torch.full((M, 2), 9.0, device="cuda")
    mb.gemm_swiglu_fp8_block_out(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"], out=(codes, scales))
    wc, ws = mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    assert torch.equal(codes[:n].float(), wc[:n].float()) and torch.equal(scales[:n], ws[:n])
    assert (codes[n:].float() == 3).all() and (scales[n:] == 9).all()


@pytest.mark.parametrize("M", [7, 300])
def test_guard_rows_and_strides(M):
    """Operands inside larger ones, the output between guard rows; what lies around A is NaN."""
    N, K = 264, 400
    t = case(M, N, K)
    want = mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"])
    big = torch.full((M + 2, 512), 127, dtype=torch.uint8, device="cuda")  # 127 is NaN in e4m3
    big[1:-1, 64:64 + K] = t["a"].view(torch.uint8)
    scales = torch.full((M + 2, 9), float("nan"), device="cuda")
    scales[1:-1, 3:7] = t["a_scale"]
    guard = torch.full((M + 2, N), 5.0, dtype=BF, device="cuda")
    mb.gemm_fp8_block_out(big.view(F8)[1:-1, 64:64 + K], scales[1:-1, 3:7], t["b"], t["b_scale"], out=guard[1:-1])
    assert torch.equal(guard[1:-1], want) and (guard[0] == 5).all() and (guard[-1] == 5).all()
    odd = torch.zeros(M, 512, dtype=torch.uint8, device="cuda")[:, 1:1 + K]  # unaligned: copied
    odd.copy_(t["a"].view(torch.uint8))
    assert torch.equal(mb.gemm_fp8_block(odd.view(F8), t["a_scale"].t().contiguous().t(), t["b"], t["b_scale"]), want)
    flat = torch.zeros(M * K + 8, dtype=torch.uint8, device="cuda")[8:].view(M, K)  # contiguous, 8-byte aligned
    flat.copy_(t["a"].view(torch.uint8))
    assert torch.equal(mb.gemm_fp8_block(flat.view(F8), t["a_scale"], t["b"], t["b_scale"]), want)


@pytest.mark.parametrize("M", [9, 260])
def test_nan_and_infinite_rows_stay_by_themselves(M):
    N, K, E, counts = 256, 272, 2, [M // 2, M - M // 2]
    t = case(M, N, K, E=E, counts=counts)
    clean = mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    t["a"].view(torch.uint8)[2, 100] = 127
    t["a_scale"][5, 1] = float("inf")
    got = mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    assert got[2].isnan().all() and not got[5].isfinite().any()
    keep = [i for i in range(M) if i not in (2, 5)]
    assert torch.equal(got[keep], clean[keep])
    t = case(M, N, K, E=E, counts=counts, halves=2)
    t["a"].view(torch.uint8)[2, 100] = 127
    codes, scales = mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"])
    assert scales[2].isnan().all() and codes[2].float().isnan().all()
    assert scales[keep].isfinite().all() and not codes[keep].float().isnan().any()


@pytest.mark.parametrize("bad", [[-9, 900, 2 ** 31 - 1], [0, 10 ** 6, 1000], [1000, 1000, 1000], [600, 200, 100]])
def test_bad_offsets_with_tiles_of_128_rows(bad):
    t = case(1000, 2048, 256, E=2, counts=[900, 100], halves=2)
    codes = torch.full((1002, 2048), 5.0, device="cuda").to(torch.float8_e4m3fn)
    scales = torch.full((1002, 16), 5.0, device="cuda")
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    mb.gemm_swiglu_fp8_block_out(t["a"], t["a_scale"], t["b"], t["b_scale"], off, out=(codes[1:-1], scales[1:-1]))
    for guarded in (codes.float(), scales):
        assert (guarded[0] == 5).all() and (guarded[-1] == 5).all()


@pytest.mark.parametrize("M,counts", [(12, [5, 7]), (600, [280, 320])])
def test_bad_offsets_touch_nothing_outside(M, counts):
    t = case(M, 256, 256, E=2, counts=counts)
    guard = torch.full((M + 2, 256), 5.0, dtype=BF, device="cuda")
    for bad in ([-9, counts[0], 2 ** 31 - 1], [0, 10 ** 6, M], [M, M, M]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        mb.gemm_fp8_block_out(t["a"], t["a_scale"], t["b"], t["b_scale"], off, out=guard[1:-1])
        torch.cuda.synchronize()
        assert (guard[0] == 5).all() and (guard[-1] == 5).all()
    assert mb.device_status(0)["code"] == 0


def fallen(offsets, M):
    """What the kernels make of an offsets array: clamped to [0, M], one below an earlier one counted as that one."""
    out = []
    for o in offsets:
        out.append(max(min(max(o, 0), M), out[-1] if out else 0))
    return out


FALLING = [(1100, [0, 1100, 0, 1100]), (600, [0, 600, 0, 600, 0, 600, 0, 600]), (1000, [0, 2 ** 31 - 1, -5, 700, 300, 900]),
           (40, [0] + [40, 0] * 20), (700, [0] * 20 + [650, 10] + [300] * 30 + [660, -2 ** 31]), (90, [90 - i for i in range(65)])]


@pytest.mark.parametrize("M,offsets", FALLING)
@pytest.mark.parametrize("halves,N,K", [(1, 272, 512), (1, 136, 8192), (2, 256, 8192), (2, 144, 272), (1, 2048, 256), (2, 1040, 272)])
def test_falling_offsets_count_as_the_largest_before(M, offsets, halves, N, K):
    """No row belongs to two experts, whichever kernel runs: the result is that of the array's running maximum, guard rows stay."""
    E, hull = len(offsets) - 1, fallen(offsets, M)
    t = case(M, N, K, E=E, counts=[0] * E, halves=halves, seed=M)
    bad, t["offsets"] = (torch.tensor(o, dtype=torch.int32, device="cuda") for o in (offsets, hull))
    args, lo, hi, nb = (t["a"], t["a_scale"], t["b"], t["b_scale"]), hull[0], hull[-1], -(-N // 128)
    if halves == 1:
        guarded = [torch.full((M + 8, N), 5.0, dtype=BF, device="cuda")]
        mb.gemm_fp8_block_out(*args, bad, out=guarded[0][4:-4])
        want = [mb.gemm_fp8_block(*args, t["offsets"])]
    else:
        guarded = [torch.full((M + 8, N), 5.0, device="cuda").to(F8), torch.full((M + 8, nb), 5.0, device="cuda")]
        mb.gemm_swiglu_fp8_block_out(*args, bad, out=(guarded[0][4:-4], guarded[1][4:-4]))
        want = mb.gemm_swiglu_fp8_block(*args, t["offsets"])
    for got, ref in zip(guarded, want):
        got, ref = got.float(), ref.float()
        assert torch.equal(got[4 + lo:4 + hi], ref[lo:hi]) and (got[4 + hi:] == 5).all() and (got[:4 + lo] == 5).all()
    if lo == 0:  # otherwise nothing has written the rows before the first expert's
        check_plain(t, *want) if halves == 1 else check_fused(t, *want)
    assert mb.device_status(0)["code"] == 0


@pytest.mark.parametrize("M,N,K,E", [(3, 512, 2048, 0), (40, 256, 512, 8), (700, 512, 384, 0), (900, 264, 512, 3),
                                     (300, 512, 4096, 0), (300, 512, 2048, 0)])
def test_the_same_bits_every_time(M, N, K, E):
    counts = [M // E] * E if E else None
    for halves, form in ((1, mb.gemm_fp8_block), (2, mb.gemm_swiglu_fp8_block)):
        t = case(M, -(-N // 16) * 16, K, E=E, counts=counts, halves=halves)
        runs = [form(t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"]) for _ in range(3)]
        for r in runs[1:]:
            for x, y in zip(r if halves == 2 else (r,), runs[0] if halves == 2 else (runs[0],)):
                assert torch.equal(x.float(), y.float())


def test_offsets_past_32_bits():
    """An output of more than 2^31 elements: its last rows equal those of a call on them alone (whole tiles either way)."""
    M, N, K = 262144 + 300, 8192, 128
    t = case(M, N, K)
    assert M * N > 2 ** 31
    c = mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"])
    tail = mb.gemm_fp8_block(t["a"][-812:], t["a_scale"][-812:], t["b"], t["b_scale"])
    assert torch.equal(c[-812:], tail)
    del c
    t = case(M, N, K, halves=2)
    codes, scales = mb.gemm_swiglu_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"])
    tail = mb.gemm_swiglu_fp8_block(t["a"][-812:], t["a_scale"][-812:], t["b"], t["b_scale"])
    assert torch.equal(codes[-812:].float(), tail[0].float()) and torch.equal(scales[-812:], tail[1])


def test_two_streams_at_once_and_beside_the_bf16_kernels():
    """Calls that overlap on the GPU share nothing: split and unsplit forms on two streams, the bf16 op between them."""
    small, large = case(24, 1024, 8192, seed=1), case(600, 1024, 8192, halves=2, seed=2)
    x = torch.randn(600, 1024, generator=gen(3), device="cuda").to(BF)
    w = (0.05 * torch.randn(2048, 1024, generator=gen(4), device="cuda")).to(BF)
    calls = [lambda: (mb.gemm_fp8_block(small["a"], small["a_scale"], small["b"], small["b_scale"]),),
             lambda: mb.gemm_swiglu_fp8_block(large["a"], large["a_scale"], large["b"], large["b_scale"]),
             lambda: (mb.gemm_swiglu(x, w),)]
    want = [[o.float() for o in call()] for call in calls]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for turn in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(((i + turn) % 3, calls[(i + turn) % 3]()))
    torch.cuda.synchronize()
    for i, outs in got:
        assert all(torch.equal(o.float(), ref) for o, ref in zip(outs, want[i]))
    assert mb.device_status(0)["code"] == 0


def test_both_watchdog_records_are_reported():
    """A wait of each kind runs out (on a barrier that nothing signals): neither record is lost."""
    lib, stream = _loader.load_library(), torch.cuda.current_stream().cuda_stream
    assert mb.device_status(0)["code"] == 0
    assert lib.magi_swiglu_fp8_block_watchdog_selftest(0, stream, 2_000_000) == 0, _loader.last_error()
    assert mb.device_status(0) == {"code": 7, "block": 0, "index": 43, "parity": 0}
    assert mb.device_status(0)["code"] == 0
    assert lib.magi_swiglu_watchdog_selftest(0, stream, 2_000_000) == 0
    assert lib.magi_swiglu_fp8_block_watchdog_selftest(0, stream, 2_000_000) == 0
    assert [mb.device_status(0)["index"] for _ in range(3)] == [42, 43, 0]
    t = case(17, 384, 256)
    check_plain(t, mb.gemm_fp8_block(t["a"], t["a_scale"], t["b"], t["b_scale"]))
    assert mb.device_status(0)["code"] == 0


# ------------------------------------------------------------------------------------------------ every form by itself
# The library chooses a kernel by the sizes; here each one is asked for: the stream kernel with 16, 32 or 64 rows a tile (+ 256 z:
# z CTAs share a tile's K blocks), single-CTA tiles (1), tiles of CTA pairs (2) and of 2 or 4 pairs that share K blocks (4, 8).
KINDS = [(h, f) for h in (1, 2) for f in (16, 32, 64, 256 + 16, 512 + 16, 1024 + 32, 2048 + 32, 2048 + 64, 1, 2, 4, 8)
         if not (h == 2 and f % 256 == 64)]


@contextlib.contextmanager
def form(value):
    prev = _loader.set_tuning("fp8_form", value)
    try:
        yield
    finally:
        _loader.set_tuning("fp8_form", prev)


def product(t, halves, offsets=None, out=None):
    args = (t["a"], t["a_scale"], t["b"], t["b_scale"], t["offsets"] if offsets is None else offsets)
    if halves == 1:
        return [mb.gemm_fp8_block(*args) if out is None else mb.gemm_fp8_block_out(*args, out=out[0])]
    return list(mb.gemm_swiglu_fp8_block(*args) if out is None else mb.gemm_swiglu_fp8_block_out(*args, out=tuple(out)))


def check(t, halves, got):
    check_plain(t, *got) if halves == 1 else check_fused(t, *got)


def same(x, y):
    return all(torch.equal(a.float(), b.float()) for a, b in zip(x, y))


def runs(value, M, N, K, halves, experts=0):
    """Whether the form serves this call, and that it is the one which runs."""
    with form(value):
        try:
            plan = _loader.fp8_block_plan(M, N, K, halves=halves, experts=experts)
        except ValueError:
            return False
    tok = value % 256 if value % 256 >= 16 else 0
    want = dict(tokens=tok, ctas=1, splits=max(value >> 8, 1)) if tok else dict(tokens=0, ctas=min(value, 2), splits=max(value // 2, 1))
    assert plan == want
    return True


@pytest.mark.parametrize("halves,value", KINDS)
@pytest.mark.parametrize("M,N,K", [(1, 16, 1040), (129, 144, 1040), (300, 272, 2064), (257, 128, 1024), (2100, 2576, 400), (1300, 2576, 1296)])
def test_every_form_dense(halves, value, M, N, K):
    many = M > 1000  # more tiles than a persistent grid has workers; too many and too short for shared K blocks
    assert runs(value, M, N, K, halves) or (many and value in (4, 8)) or value >> 8 > -(-K // 128)
    if not runs(value, M, N, K, halves):
        return
    t = case(M, N, K, halves=halves, seed=M)
    with form(value):
        got = product(t, halves)
        check(t, halves, got)
        assert same(product(t, halves), got)
    assert mb.device_status(0)["code"] == 0


UNEVEN = [([300, 0, 257, 100, 1], 9, 112, 1040), ([300, 0, 257, 100, 1], 9, 272, 2064), ([0, 0, 0], 40, 112, 1040),
          ([(i * 37) % 400 if i % 3 else 0 for i in range(40)], 300, 1040, 272)]


@pytest.mark.parametrize("halves,value", KINDS)
@pytest.mark.parametrize("counts,tail,N,K", UNEVEN)
def test_every_form_over_experts(halves, value, counts, tail, N, K):
    """Empty and partial groups, a tail without experts that comes out as zeros or stays, an expert full of NaN."""
    n, E = sum(counts), len(counts)
    assert runs(value, n + tail, N, K, halves, E) or value in (4, 8) and N > 112 or value >> 8 > -(-K // 128)
    if not runs(value, n + tail, N, K, halves, E):
        return
    t = case(n + tail, N, K, E=E, counts=counts, halves=halves, seed=N)
    with form(value):
        got = product(t, halves)
        check(t, halves, got)
        assert (got[0][n:].float() == 0).all() and (halves == 1 or (got[1][n:] == 2.0 ** -126).all())
        held = [torch.full((g.shape[0] + 8, g.shape[1]), 5.0, device="cuda").to(g.dtype) for g in got]
        product(t, halves, out=[h[4:-4] for h in held])
        for h, g in zip(held, got):
            assert torch.equal(h[4:4 + n].float(), g[:n].float()) and (h[:4].float() == 5).all() and (h[4 + n:].float() == 5).all()
        if n:
            lo, hi = int(t["offsets"][2]), int(t["offsets"][3])  # the third expert
            t["a"].view(torch.uint8)[lo:hi] = 127  # NaN in e4m3
            again = product(t, halves)
            keep = torch.ones(n + tail, dtype=torch.bool, device="cuda")
            keep[lo:hi] = False
            for x, g in zip(again, got):
                assert torch.equal(x[keep].float(), g[keep].float()) and x[lo:hi].float().isnan().all()
    assert mb.device_status(0)["code"] == 0


@pytest.mark.parametrize("halves,value", KINDS)
@pytest.mark.parametrize("M,offsets", FALLING)
def test_every_form_with_falling_offsets(halves, value, M, offsets):
    E, hull, K = len(offsets) - 1, fallen(offsets, M), 1040
    t = case(M, 112, K, E=E, counts=[0] * E, halves=halves, seed=M)
    bad, t["offsets"] = (torch.tensor(o, dtype=torch.int32, device="cuda") for o in (offsets, hull))
    assert runs(value, M, 112, K, halves, E) or value in (4, 8) and E > 7
    if not runs(value, M, 112, K, halves, E):
        return
    with form(value):
        want = product(t, halves)
        held = [torch.full((g.shape[0] + 8, g.shape[1]), 5.0, device="cuda").to(g.dtype) for g in want]
        product(t, halves, offsets=bad, out=[h[4:-4] for h in held])
        lo, hi = hull[0], hull[-1]
        for h, g in zip(held, want):
            assert torch.equal(h[4 + lo:4 + hi].float(), g[lo:hi].float())
            assert (h[:4 + lo].float() == 5).all() and (h[4 + hi:].float() == 5).all()
        if lo == 0:
            check(t, halves, want)
    assert mb.device_status(0)["code"] == 0


@pytest.mark.parametrize("halves", [1, 2])
def test_single_tiles_and_pairs_give_the_same_bits(halves):
    t = case(900, 528, 1296, E=3, counts=[257, 0, 600], halves=halves)
    with form(1):
        one = product(t, halves)
    with form(2):
        assert same(product(t, halves), one)


@pytest.mark.parametrize("halves,value", KINDS)
def test_every_form_captured_beside_other_kernels(halves, value):
    """Replayed with new rows between kernels that it overlaps; what it answers is what an eager call answers."""
    counts = [130, 0, 64, 6]
    t = case(200, 144, 1040, E=4, counts=counts, halves=halves, seed=3)
    x = torch.randn(200, 1040, generator=gen(5), device="cuda").to(BF)

    def step():
        t["a"], t["a_scale"] = mb.quantize_fp8_block_out(x)
        return product(t, halves)

    with form(value):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for seed in (6, 7):
            x.copy_(torch.randn(200, 1040, generator=gen(seed), device="cuda"))
            graph.replay()
            assert same(held, step())
    assert mb.device_status(0)["code"] == 0


@pytest.mark.parametrize("value", [16, 32, 512 + 16, 1, 2, 4])
@pytest.mark.parametrize("exponent", [0, -40, 40])
def test_fused_codes_are_the_quotients_rounded_once(value, exponent):
    """Values whose quotients lie at, or one fp32 step beside, the middle between two codes: a product with the reciprocal of the
    scale would put many on the wrong side.  Every gate is 64 or more, where silu(g) = g in fp32, and every sum has one or two
    terms of few bits, so the values to quantise are known bit for bit."""
    M, N, K = 300, 128, 2048
    grid = torch.arange(0, 127, dtype=torch.uint8, device="cuda").view(F8)  # 0 .. 448
    step = torch.cat([grid.float()[1:] - grid.float()[:-1], torch.zeros(1, device="cuda")])
    t = dict(offsets=None, a=torch.zeros(M, K, device="cuda"), b=torch.zeros(2 * N, K, device="cuda"))
    t["a"][:, :2] = 1
    t["b"][:N, 0] = 1  # gates: the row's scale
    up = torch.cat([grid.float(), torch.zeros(1, device="cuda")])
    t["b"][N:, 0], t["b"][N:N + 127, 1] = up, torch.where(step / 2 >= 2.0 ** -9, step / 2, 0.0)
    t["a"], t["b"] = t["a"].to(F8), t["b"].to(F8)
    t["a_scale"] = 64 + 64 * torch.rand(M, K // 128, generator=gen(1), device="cuda")  # 24 random bits
    t["b_scale"] = torch.ones(2, K // 128, device="cuda")
    t["b_scale"][1] = 2.0 ** exponent
    with form(value):
        codes, scales = product(t, 2)
    g = t["a_scale"][:, :1]
    u = (g * 2.0 ** exponent) * (up + t["b"][N:, 1].float())  # fp32: one rounding
    y = g * u
    s = y.amax(1, keepdim=True)
    s = s / torch.full_like(s, 448.0)
    assert torch.equal(scales, s)
    assert torch.equal(codes.float(), (y / s).to(F8).float())
    assert not torch.equal((y * (1 / s)).to(F8).float(), codes.float())  # the values do tell the two apart


@pytest.mark.parametrize("value", [16, 32, 1, 2])
@pytest.mark.parametrize("exponent", [-142, -140, -127, -120, -113, -111, -93, -91, 90, 103])
def test_fused_codes_of_extreme_scales(value, exponent):
    """The same quotients when the block's scale is near the ends of fp32 (K one block: the up half's scale carries it)."""
    M, N, K = 200, 128, 128
    t = dict(offsets=None, a=torch.zeros(M, K, device="cuda"), b=torch.zeros(2 * N, K, device="cuda"))
    t["a"][:, 0] = 1
    t["b"][:N, 0] = 1
    t["b"][N:, 0] = torch.cat([torch.arange(0, 127, dtype=torch.uint8, device="cuda").view(F8).float(), torch.zeros(1, device="cuda")])
    t["a"], t["b"] = t["a"].to(F8), t["b"].to(F8)
    t["a_scale"] = 64 + 64 * torch.rand(M, 1, generator=gen(2), device="cuda")
    t["b_scale"] = torch.tensor([[1.0], [2.0 ** exponent]], device="cuda")
    with form(value):
        codes, scales = product(t, 2)
    g = t["a_scale"]
    y = g * ((g * 2.0 ** exponent) * t["b"][N:, 0].float())
    s = y.amax(1, keepdim=True)
    s = (s / torch.full_like(s, 448.0)).clamp_min(2.0 ** -126)
    assert torch.equal(scales, s) and torch.equal(codes.float(), (y / s).to(F8).float())


@pytest.mark.parametrize("value", [16, 1, 2])
def test_silu_of_one_gate_a_row(value):
    """Gates from -80 to 80 against 64 bits: with one column a row's scale is its value over 448.  ex2 is off by 2^-22, its
    argument -g * log2(e) by |g| * 2^-23 after two roundings, the reciprocal by 2^-23, sum and products by 2^-24 each; the scale's
    division by 2^-24."""
    M, K, N = 4001, 128, 16
    g = torch.linspace(-80, 80, M, device="cuda")[:, None]
    t = dict(offsets=None, a=torch.zeros(M, K, device="cuda"), b=torch.zeros(2 * N, K, device="cuda"))
    t["a"][:, 0] = torch.where(g[:, 0] < 0, -1.0, 1.0)
    t["b"][0, 0], t["b"][N, 0] = 1, 1
    t["a"], t["b"] = t["a"].to(F8), t["b"].to(F8)
    t["a_scale"], t["b_scale"] = g.abs(), torch.ones(2, 1, device="cuda")
    with form(value):
        codes, scales = product(t, 2)
    g = g.double()
    y = g * torch.sigmoid(g) * g  # the up sum is the gate's
    err = (scales.double() * 448 - y.abs()).abs()
    assert (err <= y.abs() * (2.0 ** -21 + g.abs() * 2.0 ** -23 + 2.0 ** -24) * (1 + 2.0 ** -20) + 448 * 2.0 ** -126).all()
    assert (codes[:, 1:].float() == 0).all()


def routed_block(s):
    row_slot, slot_row, offsets = mb.expert_sort_out(s["ids"], s["w2"].shape[0])
    a, sc = mb.expert_gather_fp8_out(s["x"], row_slot, slot_row)
    h, hs = mb.gemm_swiglu_fp8_block_out(a, sc, s["w13"], s["w13_scale"], offsets)
    y = mb.gemm_fp8_block_out(h, hs, s["w2"], s["w2_scale"], offsets)
    return mb.expert_combine_out(y, s["w"], row_slot, slot_row)


def routed_state(T, k, E, H, N, seed, drop=0.0):
    g = gen(seed)
    w13 = (0.05 * torch.randn(E, 2 * N, H, generator=g, device="cuda")).to(BF)
    w2 = (0.05 * torch.randn(E, H, N, generator=g, device="cuda")).to(BF)
    s = dict(x=torch.randn(T, H, generator=g, device="cuda").to(BF), w13_bf16=w13, w2_bf16=w2)
    s["w13"], s["w13_scale"] = mb.quantize_fp8_gate_up(w13)
    s["w2"], s["w2_scale"] = mb.quantize_fp8_weight(w2)
    s["ids"] = torch.randint(0, E, (T, k), generator=g, device="cuda")
    s["ids"][torch.rand(T, k, generator=g, device="cuda") < drop] = -1
    s["w"] = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), 1)
    return s


@pytest.mark.parametrize("T,k,E,H,N,drop", [(1, 2, 8, 256, 272, 0), (37, 2, 4, 272, 256, 0.2), (500, 4, 6, 512, 384, 0.05)])
def test_the_operators_together(T, k, E, H, N, drop):
    """A routed block in 8 bits against the bf16 weights in 64 bits.  Each of the three quantisations (rows, weights, the
    activation) is a relative error of at most 2^-4 an element with random signs; over sums of hundreds of elements the
    result's 2-norm error stays under 3 * 2^-4 / sqrt(3) (uniform in a step) ~ 0.11 of its norm."""
    s = routed_state(T, k, E, H, N, seed=T, drop=drop)
    got = routed_block(s).double()
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for t in range(T):
        for j in range(k):
            e = int(s["ids"][t, j])
            if e >= 0:
                h = s["w13_bf16"][e].double() @ x[t]
                y = s["w2_bf16"][e].double() @ (h[:N] * torch.sigmoid(h[:N]) * h[N:])
                want[t] += s["w"][t, j].double() * y
    assert (got - want).norm() <= 0.11 * want.norm()


def test_the_operators_together_in_a_graph():
    """Captured once, replayed on new tokens and routings (decode and prompt sizes), two graphs in turn."""
    built = []
    for T in (3, 300):
        s = routed_state(T, 2, 4, 256, 256, seed=T)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            routed_block(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = routed_block(s)
        built.append((s, graph, out))
    for turn in range(3):
        for s, graph, _ in built:
            new = routed_state(s["x"].shape[0], 2, 4, 256, 256, seed=90 + turn, drop=0.3)
            for key in ("x", "ids", "w"):
                s[key].copy_(new[key])
            graph.replay()
        for s, _, out in built:
            assert torch.equal(out, routed_block(s))
    assert mb.device_status(0)["code"] == 0
