"""4-bit matrices without a GPU: the storage order, einsum's forms and the refusals."""

from __future__ import annotations

import pytest
import torch

import trntensor_b200 as tt
from trntensor_b200 import _lib


def blocked(codes: torch.Tensor, scales: torch.Tensor, group: int):
    """The stored bytes and scales, written from the description of the layout:
    16 x 128 blocks, lane 4 g + t with rows g and g + 8, word w with the codes
    k = 32 w + 8 t + i in nibble i / 2 (even i) or 4 + i / 2 (odd i)."""
    n, k = codes.shape
    rt, kb, gpb = -(-n // 16), -(-k // 128), 128 // group
    packed = torch.full((rt, kb, 2, 32, 4, 4), 0x88, dtype=torch.uint8)
    stored = torch.zeros((rt, kb, gpb, 16), dtype=scales.dtype)
    for row in range(n):
        for col in range(k):
            r, c = row % 16, col % 128
            w, t, i = c // 32, c % 32 // 8, c % 8
            nib = i // 2 + 4 * (i % 2)
            at = (row // 16, col // 128, r // 8, 4 * (r % 8) + t, w, nib // 2)
            byte = int(packed[at])
            byte = byte & ~(15 << 4 * (nib % 2)) | (int(codes[row, col]) + 8) << 4 * (nib % 2)
            packed[at] = byte
        for j in range(-(-k // group)):
            stored[row // 16, j // gpb, j % gpb, row % 16] = scales[row, j]
    return packed.reshape(-1), stored.reshape(-1)


def held(n, k, group, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = torch.rand((n, -(-k // group)), generator=g) + 0.1
    packed, stored = blocked(codes, scales, group)
    return codes, scales, tt.Q4Matrix(packed, stored, (n, k), group)


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (17, 130, 64), (16, 128, 128), (5, 300, 32)])
def test_storage_order(n, k, group):
    codes, scales, w = held(n, k, group)
    assert torch.equal(w.codes(), codes)
    assert torch.equal(w.group_scales(), scales)
    lib = _lib.load()
    assert lib.tt_q4_packed_bytes(n, k) == w.packed.numel()
    assert lib.tt_q4_scale_count(n, k, group) == w.scales.numel()
    assert tuple(w.shape) == (n, k) and w.dim() == w.ndim == 2


def test_refusals():
    _, _, w = held(6, 40, 32)
    x = torch.randn(3, 40)
    with pytest.raises(ValueError, match="end in 40"):
        tt.q4_matmul(torch.randn(3, 6), w)
    with pytest.raises(ValueError, match="end in 6"):
        tt.q4_matmul(x, w, over_n=True)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        tt.q4_matmul(x.double(), w)
    with pytest.raises(ValueError, match="must be a Q4Matrix"):
        tt.q4_matmul(x, torch.randn(6, 40))
    with pytest.raises(ValueError, match="group must be one of"):
        tt.quantize_q4(torch.randn(4, 4), group=48)
    with pytest.raises(ValueError, match="must be 2D"):
        tt.quantize_q4(torch.randn(4))
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        tt.quantize_q4(torch.ones(4, 4, dtype=torch.int8))
    with pytest.raises(ValueError, match="scale_dtype"):
        tt.quantize_q4(torch.randn(4, 4), scale_dtype=torch.float64)
    with pytest.raises(ValueError, match="2D int8"):
        tt.pack_q4(torch.randn(4, 4), torch.randn(4, 1))
    with pytest.raises(ValueError, match="scales must be"):
        tt.pack_q4(torch.zeros(4, 40, dtype=torch.int8), torch.randn(4, 1), group=32)
    with pytest.raises(ValueError, match="float type"):
        w.dequantize(torch.int32)


@pytest.mark.parametrize("sub", ["mk,nk->m", "mk,nk->mnk", "nk,nk->n", "nk,nk->nk", "kk,nk->kn",
                                 "mk,nn->mk"])
def test_einsum_refuses_other_forms(sub):
    _, _, w = held(6, 6, 32)
    with pytest.raises(ValueError):
        tt.einsum(sub, torch.randn(6, 6), w)


def test_einsum_refusals():
    _, _, w = held(6, 40, 32)
    x = torch.randn(3, 40)
    with pytest.raises(ValueError, match="index 'k'"):
        tt.einsum("mk,nk->mn", torch.randn(3, 41), w)
    with pytest.raises(ValueError, match="one dense operand"):
        tt.einsum("nk,mk->nm", w, w)
    with pytest.raises(ValueError, match="one dense operand"):
        tt.einsum("mk,nk,nj->mj", x, w, torch.randn(6, 2))
    with pytest.raises(ValueError, match="precision must be"):
        tt.einsum("mk,nk->mn", x, w, precision="bogus")


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU error path")
def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="CUDA"):
        tt.quantize_q4(torch.randn(4, 40))


def test_library_refuses_bad_arguments():
    """Argument checks of the C ABI come before any CUDA call."""
    lib = _lib.load()
    p = 16  # never dereferenced: a shape or NULL check answers first
    assert lib.tt_q4_matmul(None, 0, 8, p, p, 0, p, 1, 8, 8, 32, p, 8, None, 0, p, None) == _lib.TT_ERR_NULL
    # many rows need a workspace; how many are many depends on the type and the sum
    assert lib.tt_q4_matmul_workspace_bytes(1, 1, 0, 32, 8, 8) == 0
    assert lib.tt_q4_matmul_workspace_bytes(1, 1, 0, 33, 8, 8) >= 33 * (64 * 2 + 4)
    assert lib.tt_q4_matmul_workspace_bytes(1, 1, 1, 8, 8, 8) == 0
    assert lib.tt_q4_matmul_workspace_bytes(1, 1, 1, 9, 8, 8) >= 9 * (64 * 2 + 4)
    assert lib.tt_q4_matmul(p, 0, 8, p, p, 0, p, 17, 8, 8, 32, p, 8, None, 0, p, None) == _lib.TT_ERR_NULL
    assert lib.tt_q4_row_scale(p, 0, 8, 8, 33, p, None) == _lib.TT_ERR_SHAPE
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(group=16), dict(type=3), dict(st=2),
                dict(ldx=7), dict(ldy=7)):
        a = dict(m=1, n=8, k=8, group=32, type=0, st=0, ldx=8, ldy=8) | bad
        for fn in (lib.tt_q4_matmul, lib.tt_q4_matmul_t):
            assert fn(p, a["type"], a["ldx"], p, p, a["st"], p, a["m"], a["n"], a["k"], a["group"], p,
                      a["ldy"], p, 0, p, None) == _lib.TT_ERR_SHAPE, bad
    assert lib.tt_q4_matmul(p, 0, 8, 8, p, 0, p, 1, 8, 8, 32, p, 8, None, 0, p, None) == _lib.TT_ERR_ALIGN
    assert lib.tt_q4_quantize(p, 0, 7, 0, 8, 8, 32, p, p, None) == _lib.TT_ERR_SHAPE
    assert lib.tt_q4_pack(p, p, 2, 8, 8, 32, p, p, None) == _lib.TT_ERR_SHAPE
    assert lib.tt_q4_dequantize(p, p, 0, 8, 8, 33, p, 0, None) == _lib.TT_ERR_SHAPE
    assert lib.tt_q4_packed_bytes(0, 5) == 0 and lib.tt_q4_scale_count(5, 5, 31) == 0


def test_sizes_past_32_bits_are_refused():
    from trntensor_b200 import quantized

    for n, k in ((2**31, 1), (1, 2**31)):
        with pytest.raises(ValueError, match="at most"):
            quantized._empty_q4(n, k, 32, torch.float32, torch.device("cpu"))
