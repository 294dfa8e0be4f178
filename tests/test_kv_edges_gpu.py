"""The 8-bit cache on the GPU where it can go wrong: scales far apart, pages that
are not there, shared pages, subnormal values, rotation in every page size.

Tolerances of attention are those of test_kv_gpu, with what a case names."""

from __future__ import annotations

import pytest
import torch
from test_kv_gpu import filled, int32

import trntensor_b200 as tt

pytestmark = pytest.mark.gpu


def test_gradients_are_refused(cuda_ok):
    """What requires grad is refused where gradients are on, and served where they are off."""
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in filled(4, 2, 16, 32)))
    q, k = torch.randn(1, 2, 4, 32, device="cuda"), torch.randn(1, 2, 2, 32, device="cuda")
    table, lengths, freq = int32([[0, 1]]), int32([20]), torch.ones(4, device="cuda")
    want, turned_q = tt.kv_attention(q, cache, table, lengths), tt.kv_rotate(q, lengths, freq)
    q.requires_grad_()
    k.requires_grad_()
    for call in (lambda: tt.kv_attention(q, cache, table, lengths), lambda: tt.kv_rotate(q, lengths, freq),
                 lambda: tt.kv_append(cache, k, k.detach(), table, lengths),
                 lambda: tt.kv_append(cache, k.detach(), k, table, lengths)):
        with pytest.raises(ValueError, match="requires grad"):
            call()
    with torch.no_grad():
        assert torch.equal(tt.kv_attention(q, cache, table, lengths), want)
        assert torch.equal(tt.kv_rotate(q, lengths, freq), turned_q)
        tt.kv_append(cache, k, k, table, lengths)
    with torch.inference_mode():
        tt.kv_append(cache, k, k, table, lengths)
    cache.check()
