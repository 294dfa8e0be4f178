"""The 8-bit cache without a GPU: storage order, refusals, the library's argument checks."""

from __future__ import annotations

import pytest
import torch

import trntensor_b200 as tt
from trntensor_b200 import _lib

CPU = torch.device("cpu")


def parts(batch=2, new=3, heads=4, kv=2, dim=32, page=16, pages=5, cols=2):
    cache = tt.KVCache8(pages, kv, dim, page_size=page, device="cpu")
    return dict(cache=cache, k=torch.randn(batch, new, kv, dim), v=torch.randn(batch, new, kv, dim),
                q=torch.randn(batch, new, heads, dim),
                table=torch.zeros(batch, cols, dtype=torch.int32),
                lengths=torch.zeros(batch, dtype=torch.int32))


def append(p, **kw):
    a = p | kw
    return tt.kv_append(a["cache"], a["k"], a["v"], a["table"], a["lengths"],
                        **{x: kw[x] for x in ("n_new", "inv_freq") if x in kw})


def attend(p, **kw):
    a = p | kw
    return tt.kv_attention(a["q"], a["cache"], a["table"], a["lengths"],
                           **{x: kw[x] for x in ("n_query", "scale") if x in kw})


def test_new_cache_is_zero():
    c = tt.KVCache8(3, 2, 32, page_size=32, device="cpu")
    k, v = c.codes()
    assert k.shape == v.shape == (3, 2, 32, 32) and not k.any() and not v.any()
    c.check()
    c.status.fill_(1 | 2)
    with pytest.raises(ValueError, match="page id outside.*length or count"):
        c.check()
    c.check()  # reading clears it
    c.status.fill_(8)
    with pytest.raises(_lib.DeviceError, match="never arrived"):
        c.check()


def test_geometry_refusals():
    for kw, word in ((dict(page_size=48), "page_size"), (dict(head_dim=40), "head_dim"),
                     (dict(head_dim=272), "head_dim"), (dict(num_pages=0), "positive"),
                     (dict(kv_heads=0), "positive")):
        a = dict(num_pages=2, kv_heads=2, head_dim=32, page_size=16) | kw
        with pytest.raises(ValueError, match=word):
            tt.KVCache8(a["num_pages"], a["kv_heads"], a["head_dim"], page_size=a["page_size"], device="cpu")
    codes, scales = torch.zeros(2, 1, 16, 32, dtype=torch.int8), torch.ones(2, 1)
    with pytest.raises(ValueError, match="codes must be int8"):
        tt.KVCache8.from_codes(codes.float(), scales, codes, scales)
    with pytest.raises(ValueError, match="scales must be"):
        tt.KVCache8.from_codes(codes, scales[0], codes, scales)
    with pytest.raises(ValueError, match="page_size"):
        tt.KVCache8.from_codes(codes[:, :, :15], scales, codes[:, :, :15], scales)


@pytest.mark.parametrize("kw,word", [
    (dict(k=torch.randn(2, 3, 2, 16)), "alike"),
    (dict(k=torch.randn(2, 3, 2, 32).double()), "k must be"),
    (dict(v=torch.randn(2, 3, 2, 32).half()), "alike"),
    (dict(k=torch.randn(2, 3, 64)), "k must be"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int64)), "block_table"),
    (dict(table=torch.zeros(3, 2, dtype=torch.int32)), "block_table"),
    (dict(table=torch.zeros(2, 0, dtype=torch.int32)), "block_table"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2)), "lengths"),
    (dict(n_new=torch.zeros(2, dtype=torch.int64)), "n_new"),
    (dict(inv_freq=torch.ones(17)), "inv_freq"),
    (dict(inv_freq=torch.ones(0)), "inv_freq"),
    (dict(inv_freq=torch.ones(4).double()), "inv_freq"),
])
def test_append_refusals(kw, word):
    with pytest.raises(ValueError, match=word):
        append(parts(), **kw)


@pytest.mark.parametrize("kw,word", [
    (dict(q=torch.randn(2, 3, 4, 16)), "q must end in"),
    (dict(q=torch.randn(2, 3, 3, 32)), "q must end in"),
    (dict(q=torch.randn(2, 3, 4, 32).double()), "q must be"),
    (dict(table=torch.zeros(2, 2)), "block_table"),
    (dict(lengths=torch.zeros(1, dtype=torch.int32)), "lengths"),
    (dict(n_query=torch.zeros(2)), "n_query"),
    (dict(scale=float("nan")), "scale must be finite"),
])
def test_attention_refusals(kw, word):
    with pytest.raises(ValueError, match=word):
        attend(parts(), **kw)


def test_rotate_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        tt.kv_rotate(torch.randn(1, 1, 1, 32), torch.zeros(1, dtype=torch.int32), torch.ones(4))
    with pytest.raises(ValueError, match="dtype must be"):
        parts()["cache"].dequantize(dtype=torch.float64)
    with pytest.raises(ValueError, match="pages must be"):
        parts()["cache"].dequantize(torch.zeros(2))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU error path")
def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="CUDA"):
        tt.KVCache8(2, 2, 32)


def test_library_refuses_bad_arguments():
    """Argument checks of the C ABI come before any CUDA call."""
    import ctypes

    lib = _lib.load()
    p = 16
    one = ctypes.byref(ctypes.c_float(1.0))

    def app(**kw):
        a = dict(k=p, type=0, pairs=0, freq=None, kc=p, batch=1, S=1, heads=1, dim=16, page=16, pages=1,
                 cols=1) | kw
        return lib.tt_kv8_append(a["k"], p, a["type"], 1, 1, 1, 1, 1, 1, p, 1, a["cols"], p, None,
                                 a["freq"], a["pairs"], 0, a["kc"], p, p, p, p, a["batch"], a["S"],
                                 a["heads"], a["dim"], a["page"], a["pages"], None)

    def att(**kw):
        a = dict(q=p, type=0, qs=16, cols=1, scale=one, batch=1, S=1, hq=2, heads=1, dim=16, page=16,
                 pages=1) | kw
        return lib.tt_kv8_attention(a["q"], a["type"], a["qs"], 16, 16, p, p, p, p, p, 1, a["cols"], p,
                                    None, a["scale"], 1, p, p, 0, p, a["batch"], a["S"], a["hq"],
                                    a["heads"], a["dim"], a["page"], a["pages"], None)

    assert app(k=None) == _lib.TT_ERR_NULL and app(pairs=4) == _lib.TT_ERR_NULL
    for bad in (dict(type=3), dict(batch=0), dict(batch=65536), dict(S=0), dict(heads=0), dict(dim=24),
                dict(dim=272), dict(page=17), dict(pages=0), dict(cols=0), dict(pairs=9, freq=p)):
        assert app(**bad) == _lib.TT_ERR_SHAPE, bad
    assert app(kc=8) == _lib.TT_ERR_ALIGN
    assert att(q=None) == _lib.TT_ERR_NULL and att(scale=None) == _lib.TT_ERR_NULL
    for bad in (dict(type=-1), dict(batch=0), dict(S=0), dict(hq=3, heads=2), dict(dim=8), dict(page=8),
                dict(pages=0), dict(cols=0), dict(S=2**31 - 1, hq=4), dict(cols=2**30)):
        assert att(**bad) == _lib.TT_ERR_SHAPE, bad
    assert att(q=8) == _lib.TT_ERR_ALIGN and att(qs=6) == _lib.TT_ERR_ALIGN
    assert lib.tt_kv8_rotate(p, 0, 1, 1, 1, p, p, 9, 0, p, 1, 1, 1, 16, None) == _lib.TT_ERR_SHAPE
    assert lib.tt_kv8_read(p, p, p, p, None, 2, p, p, 0, p, 1, 1, 16, 16, None) == _lib.TT_ERR_SHAPE
