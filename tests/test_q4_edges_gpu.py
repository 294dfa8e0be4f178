"""4-bit matrices on the GPU: rows without a scale.

Tolerances are those of test_q4_gpu.check."""

from __future__ import annotations

import pytest
import torch
from test_q4_gpu import TYPES, check, make, rows

import trntensor_b200 as tt

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
