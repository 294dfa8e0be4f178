"""4-bit matrices on the GPU: rows without a scale, forward-mode derivatives.

Tolerances are those of test_q4_gpu.check."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd
from test_q4_gpu import TYPES, check, make, rows

import trntensor_b200 as tt
from trntensor_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-9])
@pytest.mark.parametrize("m", [5, 40, 300])
def test_rows_of_zeros(cuda_ok, m, size, scale_dtype, name):
    """Pruned and padding rows of a matrix (scale 0) add nothing, and take
    nothing from the others."""
    codes, scales, _ = make(500, 300, 64, scale_dtype)
    scales = scales * size
    scales[::7] = 0
    wide = codes.double() * scales.double().repeat_interleave(64, 1)[:, :300]
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=64)
    # small results would drown in fp16's smallest step: the dense operand is large there
    up = 200.0 if name == "fp16" else 1.0
    dy = (rows(m, 500, torch.float32) * up).to(TYPES[name])
    check(tt.q4_matmul(dy.cuda(), w, over_n=True), dy, wide, over_n=True)
    x = (rows(m, 300, torch.float32) * up).to(TYPES[name])
    got = tt.q4_matmul(x.cuda(), w)
    check(got, x, wide.T)
    assert not got[:, ::7].any()


@pytest.mark.parametrize("m", [3, 40])
def test_zero_matrix_and_infinities(cuda_ok, m):
    """Nothing but zero rows gives zeros; an infinite operand on such a row is no number."""
    codes, _, _ = make(40, 130, 32)
    w = tt.pack_q4(codes.cuda(), torch.zeros(40, 5, device="cuda"), group=32)
    for dtype in TYPES.values():
        dy = rows(m, 40, dtype).cuda()
        assert not tt.q4_matmul(dy, w, over_n=True).any()
        dy[1, 7], dy[2, 39] = float("inf"), float("nan")
        got = tt.q4_matmul(dy, w, over_n=True)
        assert got[1:3].isnan().all() and not got[0].any() and not got[3:].any()


@pytest.mark.parametrize("over_n", [False, True])
@pytest.mark.parametrize("m", [4, 200])
def test_forward_mode(cuda_ok, m, over_n):
    """The map is linear: its derivative along t is the product of t."""
    codes, scales, _ = make(60, 100, 32)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=32)
    x, t = (rows(m, 60 if over_n else 100, torch.float32, seed=s).cuda() for s in (1, 2))
    sub = "mn,nk->mk" if over_n else "mk,nk->mn"
    want, slope = tt.q4_matmul(x, w, over_n=over_n), tt.q4_matmul(t, w, over_n=over_n)
    for leaf in (x, x.clone().requires_grad_()):
        with fwd.dual_level():
            dual = fwd.make_dual(leaf, t)
            for y in (tt.q4_matmul(dual, w, over_n=over_n), tt.einsum(sub, dual, w),
                      tt.q4_matmul(dual.view(2, m // 2, -1), w, over_n=over_n).flatten(0, 1)):
                primal, tangent = fwd.unpack_dual(y)
                assert tangent is not None and torch.equal(tangent, slope)
                assert torch.equal(primal, want)
            with torch.no_grad():
                assert torch.equal(fwd.unpack_dual(tt.q4_matmul(dual, w, over_n=over_n)).tangent, slope)
    # forward over backward: the gradient along a moving dy
    leaf = x.clone().requires_grad_()
    dy, dt = (rows(m, 100 if over_n else 60, torch.float32, seed=s).cuda() for s in (3, 4))
    with fwd.dual_level():
        (dx,) = torch.autograd.grad(tt.q4_matmul(leaf, w, over_n=over_n), leaf, fwd.make_dual(dy, dt))
        primal, tangent = fwd.unpack_dual(dx)
    assert torch.equal(primal, tt.q4_matmul(dy, w, over_n=not over_n))
    assert torch.equal(tangent, tt.q4_matmul(dt, w, over_n=not over_n))
    # a plain operand inside the level has no tangent
    with fwd.dual_level():
        assert fwd.unpack_dual(tt.q4_matmul(x, w, over_n=over_n)).tangent is None
    # functional transforms are refused, not answered wrongly
    for call in (lambda: torch.func.jvp(lambda a: tt.q4_matmul(a, w, over_n=over_n), (x,), (t,)),
                 lambda: torch.func.vmap(lambda a: tt.q4_matmul(a, w, over_n=over_n))(x.view(2, m // 2, -1)),
                 lambda: torch.func.grad(lambda a: tt.q4_matmul(a, w, over_n=over_n).sum())(x)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("m", [40, 300, 700])
def test_a_wait_that_ran_out_is_not_a_result(cuda_ok, m, name):
    """With a timeout noted, products of many rows are NaN until the word has been read."""
    codes, scales, _ = make(300, 2000, 64)
    w = tt.pack_q4(codes.cuda(), scales.cuda(), group=64)
    for over_n, cols in ((False, 2000), (True, 300)):
        x = rows(m, cols, TYPES[name]).cuda()
        want = tt.q4_matmul(x, w, over_n=over_n)
        w.status.fill_(0x101)
        for _ in range(2):
            assert tt.q4_matmul(x, w, over_n=over_n).isnan().all()
        with pytest.raises(_lib.DeviceError, match="0x101"):
            w.check()
        assert torch.equal(tt.q4_matmul(x, w, over_n=over_n), want)
        w.check()


@pytest.mark.parametrize("name,terms", [("fp16", 60_000), ("fp16", 300_000), ("bf16", 600_000)])
@pytest.mark.parametrize("over_n", [False, True])
def test_very_long_sums(cuda_ok, name, terms, over_n):
    """Terms of one sign, in so many tiles that no CTAs share a sum: what is cut off at each
    step of the tensor cores (up to 2^-23 of the sum) would come to as much as the result's
    rounding. Here 16 such steps make a part, and the parts' additions round: half of 2^-23 for
    each 256 terms."""
    other, m = 9600, 40
    n, k = (terms, other) if over_n else (other, terms)
    codes = torch.full((n, k), 7, dtype=torch.int8, device="cuda")
    w = tt.pack_q4(codes, torch.full((n, -(-k // 128)), 2.0**-6, dtype=torch.bfloat16, device="cuda"))
    del codes
    g = torch.Generator().manual_seed(3)
    x = (0.75 + 0.25 * torch.rand(m, terms, generator=g)).mul(2.0**-4).to(TYPES[name])
    got = tt.q4_matmul(x.cuda(), w, over_n=over_n).double().cpu()
    want = x.double().sum(1, keepdim=True) * (7 * 2.0**-6)
    bound = torch.finfo(x.dtype).eps / 2 + 1.01 * (16 * 2.0**-23 + (terms / 256 + 8) * 2.0**-24)
    worst = ((got - want).abs() / want).max().item()
    assert worst <= bound, (worst, bound)
