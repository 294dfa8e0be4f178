"""The 8-bit cache without a GPU: what is refused rather than answered in part."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd
from test_kv_cpu import append, attend, parts

from trntensor_b200 import kv_cache


def test_gradients_are_refused():
    """Nothing here is differentiable: an operand that asks for a gradient is not detached in silence."""
    p = parts()
    freq = torch.ones(4, requires_grad=True)
    for name, call in (("q", attend), ("k", append), ("v", append)):
        with pytest.raises(ValueError, match=f"^{name} requires grad.*detach"):
            call(p | {name: p[name].clone().requires_grad_()})
        with fwd.dual_level():
            dual = fwd.make_dual(p[name], torch.ones_like(p[name]))
            with pytest.raises(ValueError, match=f"^{name} has a tangent.*detach"):
                call(p | {name: dual})
    with pytest.raises(ValueError, match="inv_freq requires grad"):
        append(p, inv_freq=freq)


def test_a_failed_size_is_asked_for_again(monkeypatch):
    """One failure to get the workspace's size is an error then, and not for good."""
    class Lib:
        sizes = [0, 4096]

        def tt_kv8_attention_workspace_bytes(self, dim):
            return self.sizes.pop(0)

        def tt_last_cuda_error(self):
            return b"device busy"

    monkeypatch.setattr(kv_cache, "_WORKSPACE", {})
    lib, dev = Lib(), torch.device("cuda", 3)
    with pytest.raises(RuntimeError, match="device busy"):
        kv_cache._workspace_bytes(lib, dev, 64)
    assert kv_cache._workspace_bytes(lib, dev, 64) == 4096
    assert kv_cache._workspace_bytes(lib, dev, 64) == 4096 and not lib.sizes


def test_scale_beyond_fp32():
    """A scale that is finite in 64 bits alone would be infinite in the library."""
    for scale in (1e300, -1e39, 2.0**127, float("inf")):
        with pytest.raises(ValueError, match="scale must be finite"):
            attend(parts(), scale=scale)


def test_sizes_past_32_bits_are_refused():
    """Expanded operands can have more tokens, sequences or heads than the library counts."""
    p = parts(batch=1, new=1, heads=2, kv=2)
    big = 2**32 + 1
    far = p["k"].expand(1, big, 2, 32)
    with pytest.raises(ValueError, match="at most"):
        append(p, k=far, v=far)
    with pytest.raises(ValueError, match="at most"):
        attend(p, q=p["q"].expand(1, big, 2, 32))
    with pytest.raises(ValueError, match="at most"):
        attend(p, q=p["q"][:, :, :1].expand(1, 1, big + 1, 32))
    wide = p["table"][:, :1].expand(1, big)
    for call in (append, attend):
        with pytest.raises(ValueError, match="at most"):
            call(p, table=wide)
    many = dict(table=p["table"].expand(big, 2), lengths=p["lengths"].expand(big))
    with pytest.raises(ValueError, match="at most"):
        append(p, k=p["k"].expand(big, 1, 2, 32), v=p["k"].expand(big, 1, 2, 32), **many)
    with pytest.raises(ValueError, match="at most"):
        attend(p, q=p["q"].expand(big, 1, 2, 32), **many)
