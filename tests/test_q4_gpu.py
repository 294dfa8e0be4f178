"""4-bit matrices on the GPU against the definition in 64 bits.

Tolerances. A result is rounded once (half a step: eps / 2 of the value). The
fp32 sum is a chain of at most 16 products, one addition for each 16 terms (8 a
group and one a 128-wide block, or 8 a block, up to 8 rows, 32 of 16-bit types
over k, 16 of fp32 over n), 8 warps and 8 CTAs; each of these loses at most a unit in the
last place (2^-23, the tensor cores truncate) of a partial sum that sum |x W|
bounds. More rows of fp32 are summed 256 terms at a time. Up to 8 rows the sum
over n keeps 2^-16 of each product of 16-bit types. Above, fp16 terms: a 16-bit
operand with bf16 scales loses only what lies below 2^-39 of its row's largest
value; two 8-bit terms of an fp32 scale leave 2^-18; fp32 rows in two terms
leave 2^-22, and the product of both seconds, left out, is 2^-20.
"""

from __future__ import annotations

import pytest
import torch

import trntensor_b200 as tt

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def make(n, k, group, scale_dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed + n + 7 * k)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = (torch.rand((n, -(-k // group)), generator=g) + 0.05).to(scale_dtype)
    wide = codes.double() * scales.double().repeat_interleave(group, 1)[:, :k]
    return codes, scales, wide


def rows(m, cols, dtype, seed=1):
    g = torch.Generator().manual_seed(seed + m + cols)
    x = torch.randn((m, cols), generator=g)
    x[:, :: max(1, cols // 5)] *= 10
    return x.to(dtype)


def check(got, x, wide, over_n=False):
    """wide is (cols of x, cols of the result)."""
    ref = x.double() @ wide
    mass = x.double().abs() @ wide.abs()
    wide_type = x.dtype == torch.float32
    if x.shape[0] <= ((16 if wide_type else 8) if over_n else (8 if wide_type else 32)):
        links = 48 + x.shape[1] / (16 if over_n else 128)
        if over_n and wide_type:
            # 12 in the tensor cores, 8 warps, 8 CTAs, and for every 64 of a
            # warp's rows (an eighth of all) an addition that rounds (half)
            links = 28 + x.shape[1] / 1024
        loss = links * 2.0**-23 + (2.0**-16 if over_n and x.dtype != torch.float32 else 0)
    elif x.dtype == torch.float32:
        # 16 in the tensor cores, 8 CTAs, and an addition (rounded: half of
        # 2^-23) for each 256 terms of up to four passes
        links = 24 + x.shape[1] / 128
        loss = links * 2.0**-23 + 2.0**-22 + 2.0**-20
    else:  # one or two passes over the sum
        links = 48 + x.shape[1] / 16 * 2
        loss = links * 2.0**-23 + 2.0**-18
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + 1.01 * loss * mass + torch.finfo(x.dtype).tiny
    assert got.dtype == x.dtype and got.shape == ref.shape
    worst = ((got.double().cpu() - ref).abs() / tol).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("m,n,k", [(20, 9600, 2000), (70, 300, 6000), (300, 500, 4100), (2, 14272, 2000), (16, 9600, 300)])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32])
def test_fp32_sums_of_one_sign(cuda_ok, m, n, k, scale_dtype):
    # what an accumulator loses at each addition then adds up
    codes, scales, _ = make(n, k, 64, scale_dtype)
    codes = codes.abs().clamp(1, 7)
    wide = codes.double() * scales.double().repeat_interleave(64, 1)[:, :k]
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=64)
    x = rows(m, k, torch.float32).abs()
    check(tt.q4_matmul(x.cuda(), w), x, wide.T)
    dy = rows(m, n, torch.float32).abs()
    check(tt.q4_matmul(dy.cuda(), w, over_n=True), dy, wide, over_n=True)


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 4096, 1024), (2, 17, 129), (3, 1001, 777), (7, 40, 4100),
          (8, 256, 256), (9, 130, 250), (16, 64, 2048), (17, 100, 384), (33, 272, 640),
          (70, 129, 1000), (130, 300, 260), (257, 513, 200), (32, 1000, 4100), (64, 128, 128), (128, 513, 2100),
          (256, 2000, 300), (300, 40, 5000), (1000, 5000, 640), (2049, 130, 131)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(cuda_ok, m, n, k, group, name):
    dtype = TYPES[name]
    codes, scales, wide = make(n, k, group, torch.float32 if (n + k) % 2 else torch.bfloat16)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=group)
    x = rows(m, k, dtype)
    check(tt.q4_matmul(x.cuda(), w), x, wide.T)
    dy = rows(m, n, dtype, seed=5)
    check(tt.q4_matmul(dy.cuda(), w, over_n=True), dy, wide, over_n=True)


@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (33, 300, 64), (128, 1024, 128)])
def test_pack_and_read_back(cuda_ok, n, k, group, scale_dtype):
    codes, scales, wide = make(n, k, group, scale_dtype)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=group)
    assert torch.equal(w.codes().cpu(), codes)
    assert torch.equal(w.group_scales().cpu().double(), scales.double())
    assert torch.equal(w.dequantize(torch.float64).cpu(), wide)
    for dtype in TYPES.values():  # one rounding of an exact product
        assert torch.equal(w.dequantize(dtype).cpu(), wide.float().to(dtype))
    again = tt.pack_q4(w.codes(), w.group_scales(), group=group)
    assert torch.equal(again.packed, w.packed) and torch.equal(again.scales, w.scales)


@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (16, 128, 128), (45, 333, 64), (64, 1000, 32)])
def test_quantize(cuda_ok, n, k, group, name, scale_dtype):
    wt = rows(n, k, TYPES[name], seed=3)
    wt[n // 2, : k // 2] = 0
    q = tt.quantize_q4(wt.cuda(), group=group, scale_dtype=scale_dtype)
    pad = torch.nn.functional.pad(wt.float(), (0, -k % group)).view(n, -1, group)
    s = (pad.abs().amax(-1) / 7).to(scale_dtype)
    assert torch.equal(q.group_scales().cpu(), s)
    c = torch.where(s[..., None] > 0, pad / s.float()[..., None], 0.0).round().clamp(-8, 7)
    assert torch.equal(q.codes().cpu(), c.view(n, -1)[:, :k].to(torch.int8))


def test_quantize_strided_and_not_finite(cuda_ok):
    wt = torch.randn(40, 200, device="cuda")
    a = tt.quantize_q4(wt[::2, 10:170], group=32)
    b = tt.quantize_q4(wt[::2, 10:170].contiguous(), group=32)
    assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)
    t = tt.quantize_q4(wt.t(), group=32)
    assert torch.equal(t.packed, tt.quantize_q4(wt.t().contiguous(), group=32).packed)
    wt[3, 40], wt[5, 70], wt[6, 0] = float("inf"), float("nan"), -float("inf")
    s = tt.quantize_q4(wt, group=32).group_scales().isnan().nonzero().tolist()
    assert s == [[3, 1], [5, 2], [6, 0]]


def test_einsum_forms(cuda_ok):
    codes, scales, wide = make(70, 90, 32)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=32)
    x = rows(6, 90, torch.float32)
    check(tt.einsum("mk,nk->mn", x.cuda(), w), x, wide.T)
    check(tt.einsum("nk,mk->nm", w, x.cuda()).T, x, wide.T)
    check(tt.einsum("km,nk->mn", x.T.contiguous().cuda(), w), x, wide.T)
    check(tt.einsum("mk,nk", x.cuda(), w), x, wide.T)
    check(tt.einsum("k,nk->n", x[0].cuda(), w)[None], x[:1], wide.T)
    check(tt.einsum("abk,nk->abn", x.view(2, 3, 90).cuda(), w).reshape(6, 70), x, wide.T)
    check(tt.einsum("abk,nk->bna", x.view(2, 3, 90).cuda(), w).permute(2, 0, 1).reshape(6, 70), x, wide.T)
    dy = rows(6, 70, torch.float32)
    check(tt.einsum("mn,nk->mk", dy.cuda(), w), dy, wide, over_n=True)
    base = torch.ones(6, 70, device="cuda")
    got = tt.einsum("mk,nk->mn", x.cuda(), w, alpha=2.0, beta=3.0, out=base)
    torch.testing.assert_close(got, 2 * tt.q4_matmul(x.cuda(), w) + 3, rtol=1e-6, atol=1e-5)
    assert tt.einsum("mk,nk->mn", x.cuda(), w, dtype="bf16").dtype == torch.bfloat16
    for precision in ("kahan", "dd"):  # in 64 bits or more, rounded once
        got = tt.einsum("mk,nk->mn", x.cuda(), w, precision=precision)
        torch.testing.assert_close(got.cpu(), (x.double() @ wide.T).float(), rtol=2.0**-22, atol=1e-12)
    a, b = tt.multi_einsum(("mk,nk->mn", x.cuda(), w), ("mn,nk->mk", dy.cuda(), w))
    check(a, x, wide.T)
    check(b, dy, wide, over_n=True)


def test_strides_and_host_operands(cuda_ok):
    codes, scales, wide = make(50, 96, 32)
    w = tt.pack_q4(codes, scales, group=32)  # host codes go to the current device
    for dtype in TYPES.values():
        big = rows(9, 200, dtype)
        for cut in (big[:, 5:101], big[::3, 8:104], big[:, ::2][:, :96], big[:1, 3:99], big[:1].expand(4, 200)[:, :96]):
            check(tt.q4_matmul(cut.cuda() if cut.is_contiguous() else big.cuda().as_strided(cut.shape, cut.stride(), cut.storage_offset()), w), cut, wide.T)
            y = tt.q4_matmul(cut, w)
            assert y.device.type == "cpu"
            check(y, cut, wide.T)


def test_empty(cuda_ok):
    w = tt.pack_q4(torch.zeros(5, 40, dtype=torch.int8).cuda(), torch.ones(5, 2).cuda(), group=32)
    assert tt.q4_matmul(torch.zeros(0, 40, device="cuda"), w).shape == (0, 5)
    none = tt.pack_q4(torch.zeros(0, 40, dtype=torch.int8).cuda(), torch.ones(0, 2).cuda(), group=32)
    assert tt.q4_matmul(torch.zeros(3, 40, device="cuda"), none).shape == (3, 0)
    assert torch.equal(tt.q4_matmul(torch.zeros(3, 0, device="cuda"), none, over_n=True),
                       torch.zeros(3, 40, device="cuda"))
    thin = tt.quantize_q4(torch.zeros(4, 0, device="cuda"))
    assert torch.equal(tt.q4_matmul(torch.zeros(2, 0, device="cuda"), thin), torch.zeros(2, 4, device="cuda"))


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("m", [3, 40, 300])
def test_not_finite(cuda_ok, name, m):
    """An infinity or NaN reaches the results that the definition puts it into, and no others."""
    dtype = TYPES[name]
    codes, scales, _ = make(300, 200, 64, torch.float32)
    codes[codes == 0] = 1
    scales[4, 1] = float("nan")
    wide = codes.double() * scales.double().repeat_interleave(64, 1)[:, :200]
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=64)
    for over_n, cols in ((False, 200), (True, 300)):
        x = rows(m, cols, dtype)
        x[0, 3], x[1, cols - 1], x[m - 1, 0] = float("inf"), float("nan"), -float("inf")
        got = tt.q4_matmul(x.cuda(), w, over_n=over_n).double().cpu()
        ref = x.double() @ (wide if over_n else wide.T)
        assert torch.equal(got.isnan(), ref.isnan())
        inf = ref.isinf()
        assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], ref[inf])


@pytest.mark.parametrize("m", [2, 40])
def test_wide_range(cuda_ok, m):
    """Rows and groups many decades apart: each result by its own mass."""
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(-8, 8, (80, 256), generator=g, dtype=torch.int8)
    scales = 10.0 ** torch.linspace(-12, 6, 80 * 4).view(80, 4)[torch.randperm(80, generator=g)]
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=64)
    wide = codes.double() * scales.double().repeat_interleave(64, 1)
    for dtype in (torch.float32, torch.bfloat16):
        x = rows(m, 256, dtype) * 10.0 ** torch.linspace(-8, 8, m)[:, None].to(dtype)
        check(tt.q4_matmul(x.cuda(), w), x, wide.T)
        dy = rows(m, 80, dtype)
        check(tt.q4_matmul(dy.cuda(), w, over_n=True), dy, wide, over_n=True)


@pytest.mark.parametrize("m", [4, 200])
def test_gradients(cuda_ok, m):
    codes, scales, wide = make(60, 100, 32)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=32)
    x = rows(m, 100, torch.float32)
    xc = x.cuda().requires_grad_()
    dy = rows(m, 60, torch.float32, seed=9)
    y = tt.einsum("mk,nk->mn", xc, w)
    (dx,) = torch.autograd.grad(y, xc, dy.cuda(), create_graph=True)
    check(dx.detach(), dy, wide, over_n=True)
    # differences: the map is linear, so a step of any size shows the slope up to rounding
    step = torch.zeros_like(x)
    step[1, 7] = 8.0
    slope = (tt.q4_matmul((x + step).cuda(), w) - tt.q4_matmul(x.cuda(), w)) / 8
    want = float((slope.cpu() * dy).sum())
    assert abs(want - float(dx[1, 7])) <= 1e-3 * float((wide[:, 7].abs() * dy[1].abs().double()).sum())
    # an expanded gradient (of a sum), and the gradient of a gradient for dy
    (ones,) = torch.autograd.grad(tt.q4_matmul(xc, w).sum(), xc)
    check(ones, torch.ones(m, 60), wide, over_n=True)
    d = dy.cuda().requires_grad_()
    (gx,) = torch.autograd.grad(tt.q4_matmul(xc, w), xc, d, create_graph=True)
    (gd,) = torch.autograd.grad(gx, d, x.cuda())
    check(gd, x, wide.T)
    xh = x.clone().requires_grad_()
    tt.q4_matmul(xh, w).backward(dy)
    check(xh.grad, dy, wide, over_n=True)


@pytest.mark.parametrize("m", [1, 12, 150])
def test_same_bits_and_graphs(cuda_ok, m):
    """Every call gives the same bits; two graphs and an eager call on another stream too."""
    codes, scales, _ = make(200, 3000, 128)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=128)
    x = rows(m, 3000, torch.bfloat16).cuda()
    dy = rows(m, 200, torch.bfloat16).cuda()
    want, back = tt.q4_matmul(x, w), tt.q4_matmul(dy, w, over_n=True)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = tt.q4_matmul(x, w), tt.q4_matmul(dy, w, over_n=True)
        graphs.append((gr, out))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for (gr, _), st in zip(graphs, side):
            with torch.cuda.stream(st):
                gr.replay()
        eager = tt.q4_matmul(x, w), tt.q4_matmul(dy, w, over_n=True)
        torch.cuda.synchronize()
        for out in (eager, graphs[0][1], graphs[1][1]):
            assert torch.equal(out[0], want) and torch.equal(out[1], back)


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("m", [7, 100])
def test_forward_and_backward_in_a_graph(cuda_ok, m, name):
    """A captured step replays with new inputs, and with another one in flight between."""
    codes, scales, _ = make(300, 2000, 64)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=64)

    def step(x, dy):
        leaf = x.detach().requires_grad_()
        y = tt.einsum("mk,nk->mn", leaf, w)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        return y.detach(), dx

    x, dy = rows(m, 2000, TYPES[name]).cuda(), rows(m, 300, TYPES[name]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, dy)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        got = step(x, dy)
    for seed in (3, 4):
        x.copy_(rows(m, 2000, TYPES[name], seed=seed))
        dy.copy_(rows(m, 300, TYPES[name], seed=seed + 9))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            gr.replay()
        want = step(x, dy)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w.check()
