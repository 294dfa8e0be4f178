"""Attention over a paged key-value cache that is held in 8 bits.

A fused chain of two contractions, like the DF-MP2 energy: scores
``q.K^T`` and their softmax never leave the chip, and the stored operands are
read as 8-bit codes with one scale for each page (block of tokens) and head.
:class:`KVCache8` owns the pages, :func:`kv_append` writes new tokens into them
(turning the keys to their positions on the way), :func:`kv_rotate` turns the
queries, and :func:`kv_attention` reads them. Nothing here has a counterpart in
the reference.

Sequences are given as a block table (batch, columns; int32 page ids in token
order) and lengths (batch; int32), both on the cache's device, so that a
program's step can be captured in a CUDA graph. What they say is checked on the
device: a page id, length or count out of range is left out and noted, and
:meth:`KVCache8.check` raises.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .dispatch import _device
from .quantized import _MOST, _TYPES, _on, _stream_of

_WORKSPACE: dict[tuple[int, int], int] = {}  # bytes by (device, head_dim)
_PAGES = (16, 32, 64, 128)
_WRONG = ((1, "a page id outside the cache"), (2, "a length or count out of range"),
          (4, "one append wrote a page for two places"), (8, "a device copy never arrived"))


def _at(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_geometry(num_pages: int, kv_heads: int, head_dim: int, page_size: int) -> None:
    if page_size not in _PAGES:
        raise ValueError(f"page_size must be one of {_PAGES}, got {page_size!r}")
    if head_dim < 16 or head_dim > 256 or head_dim % 16:
        raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {head_dim!r}")
    if num_pages < 1 or not 1 <= kv_heads <= 32767:
        raise ValueError(f"num_pages and kv_heads must be positive (kv_heads at most 32767), "
                         f"got {num_pages!r} and {kv_heads!r}")


class KVCache8:
    """Pages of keys and values as int8 codes with fp32 scales (page, head).

    All pages start as zeros. ``status`` is a device word that collects what the
    calls found wrong; :meth:`check` reads it. Where a device copy never arrived
    attention gives NaN, until the word has been read.
    """

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64,
                 device: torch.device | str | None = None):
        _check_geometry(num_pages, kv_heads, head_dim, page_size)
        dev = _device() if device is None else torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.num_pages, self.kv_heads, self.head_dim = num_pages, kv_heads, head_dim
        self.page_size = page_size
        self._k = torch.full((num_pages, kv_heads, page_size, head_dim), 128, dtype=torch.uint8,
                             device=dev)
        self._v = torch.full((num_pages, kv_heads, page_size // 16, head_dim, 16), 128,
                             dtype=torch.uint8, device=dev)
        self.k_scales = torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=dev)
        self.v_scales = torch.zeros_like(self.k_scales)
        self.status = torch.zeros((), dtype=torch.int32, device=dev)

    @property
    def device(self) -> torch.device:
        return self._k.device

    @classmethod
    def from_codes(cls, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                   v_scales: torch.Tensor) -> "KVCache8":
        """A cache from int8 codes (pages, kv_heads, page_size, head_dim) in
        -127..127 and scales (pages, kv_heads), as :meth:`codes` and the scales
        of another cache give them (a negative scale is kept as its magnitude,
        and its codes turn their signs)."""
        if k_codes.dim() != 4 or k_codes.dtype != torch.int8 or v_codes.dtype != torch.int8 \
                or k_codes.shape != v_codes.shape:
            raise ValueError("from_codes: codes must be int8 (pages, kv_heads, page_size, head_dim)")
        n, h, p, d = (int(s) for s in k_codes.shape)
        _check_geometry(n, h, d, p)
        if tuple(k_scales.shape) != (n, h) or tuple(v_scales.shape) != (n, h):
            raise ValueError(f"from_codes: scales must be {(n, h)}, got {tuple(k_scales.shape)} "
                             f"and {tuple(v_scales.shape)}")
        dev = k_codes.device if k_codes.device.type == "cuda" else _device()
        self = cls.__new__(cls)
        self.num_pages, self.kv_heads, self.head_dim, self.page_size = n, h, d, p
        # a negative scale's sign goes to its codes: the kernels compare scaled scores
        k_scales = k_scales.to(dev, torch.float32)
        v_scales = v_scales.to(dev, torch.float32)
        k_codes, v_codes = k_codes.to(dev), v_codes.to(dev)
        k_codes = torch.where((k_scales < 0)[..., None, None], -k_codes, k_codes)
        v_codes = torch.where((v_scales < 0)[..., None, None], -v_codes, v_codes)
        k_scales, v_scales = k_scales.abs(), v_scales.abs()
        # biased by 128: the sign bit turned over
        self._k = k_codes.contiguous().view(torch.uint8) ^ 128
        v = v_codes.reshape(n, h, p // 16, 16, d).transpose(-1, -2).contiguous()
        self._v = v.view(torch.uint8).bitwise_xor_(128)
        self.k_scales, self.v_scales = k_scales.contiguous(), v_scales.contiguous()
        self.status = torch.zeros((), dtype=torch.int32, device=dev)
        return self

    def codes(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The int8 codes of keys and values, (pages, kv_heads, page_size, head_dim)."""
        v = (self._v ^ 128).view(torch.int8).transpose(-1, -2)
        return (self._k ^ 128).view(torch.int8), v.reshape(self._k.shape)

    def dequantize(self, pages: torch.Tensor | None = None, *,
                   dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of the given pages (int32 or int64 ids; default all) as floats,
        each (n, kv_heads, page_size, head_dim)."""
        if dtype not in _TYPES:
            raise ValueError(f"dequantize: dtype must be fp32, bf16 or fp16, got {dtype}")
        if pages is not None:
            if pages.dim() != 1 or pages.dtype not in (torch.int32, torch.int64):
                raise ValueError("dequantize: pages must be a 1D tensor of int32 or int64 ids")
            if pages.dtype == torch.int64:  # what int32 cannot hold stays out of range
                pages = pages.clamp(-1, 2**31 - 1)
            pages = pages.to(self.device, torch.int32).contiguous()
        n = self.num_pages if pages is None else int(pages.shape[0])
        k = torch.empty((n, self.kv_heads, self.page_size, self.head_dim), dtype=dtype,
                        device=self.device)
        v = torch.empty_like(k)
        if n:
            with _on(self.device):
                _lib.check(_lib.load().tt_kv8_read(
                    _at(self._k), _at(self._v), _at(self.k_scales), _at(self.v_scales),
                    _at(pages), n, _at(k), _at(v), _TYPES[dtype], _at(self.status),
                    self.num_pages, self.kv_heads, self.page_size, self.head_dim,
                    _stream_of(self.device)), "tt_kv8_read")
        return k, v

    def check(self) -> None:
        """Raise if a call since the last check met a bad page, length or count
        (waits for the device)."""
        code = int(self.status.item())
        if code == 0:
            return
        self.status.zero_()
        what = "; ".join(text for bit, text in _WRONG if code & bit)
        raise (_lib.DeviceError if code & 8 else ValueError)(f"KVCache8: {what}")


def _int32(t: torch.Tensor | None, name: str, shape: tuple, dev: torch.device):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != shape or t.device != dev:
        raise ValueError(f"{name} must be int32 {shape} on {dev}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    return t.contiguous()


def _check_table(table: torch.Tensor, batch: int, dev: torch.device) -> torch.Tensor:
    if table.dim() != 2 or table.shape[0] != batch or table.dtype != torch.int32 or table.device != dev \
            or (batch and table.shape[1] < 1):
        raise ValueError(f"block_table must be int32 ({batch}, columns) on {dev}, got {table.dtype} "
                         f"{tuple(table.shape)} on {table.device}")
    if table.shape[1] > _MOST:
        raise ValueError(f"block_table may have at most {_MOST} columns, got {table.shape[1]}")
    return table if table.stride(1) == 1 else table.contiguous()


def _check_underived(x: torch.Tensor, name: str) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad, but no gradient is computed here: detach it, or call "
                         "under torch.no_grad()")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError(f"{name} has a tangent, but no derivative is computed here: detach it")


def _check_tokens(x: torch.Tensor, name: str, dev: torch.device) -> torch.Tensor:
    if x.dim() != 4 or x.dtype not in _TYPES:
        raise ValueError(f"{name} must be fp32, bf16 or fp16 (batch, tokens, heads, head_dim), "
                         f"got {x.dtype} {tuple(x.shape)}")
    if max(x.shape) > _MOST:
        raise ValueError(f"{name} may have at most {_MOST} of each, got {tuple(x.shape)}")
    if x.device != dev:
        raise ValueError(f"{name} must be on {dev}, got {x.device}")
    _check_underived(x, name)
    return x if x.stride(3) == 1 else x.contiguous()


def _check_freq(inv_freq: torch.Tensor, dim: int, dev: torch.device) -> torch.Tensor:
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or inv_freq.device != dev \
            or not 1 <= inv_freq.shape[0] <= dim // 2:
        raise ValueError(f"inv_freq must be fp32 of 1 to {dim // 2} values on {dev}, got "
                         f"{inv_freq.dtype} {tuple(inv_freq.shape)} on {inv_freq.device}")
    _check_underived(inv_freq, "inv_freq")
    return inv_freq.contiguous()


def kv_append(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
              lengths: torch.Tensor, *, n_new: torch.Tensor | None = None,
              inv_freq: torch.Tensor | None = None, interleaved: bool = False) -> None:
    """Write k, v (batch, S, kv_heads, head_dim) behind the ``lengths[b]`` tokens
    that each sequence has in the cache (rows from ``n_new[b]`` on are padding).

    With ``inv_freq`` (R / 2 frequencies) the first R values of each key are
    turned by ``position * inv_freq[j]``, in pairs (j, j + R / 2) or, where
    ``interleaved``, (2 j, 2 j + 1). A page's scale is its largest value / 127;
    it grows as tokens come in, and the earlier tokens' codes are then rounded
    onto it. A call that writes a page's first token starts that page anew.
    Rows of the same call may share a page for reading, but a page that is
    written belongs to one sequence. ``lengths`` is left as it is. Codes are
    integers and have no gradient: a k or v that requires grad is refused where
    gradients are on.
    """
    dev = cache.device
    k, v = _check_tokens(k, "k", dev), _check_tokens(v, "v", dev)
    if k.shape != v.shape or k.dtype != v.dtype or tuple(k.shape[2:]) != (cache.kv_heads, cache.head_dim):
        raise ValueError(f"k and v must be alike and end in {(cache.kv_heads, cache.head_dim)}, got "
                         f"{tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    batch, new = k.shape[:2]
    table = _check_table(block_table, batch, dev)
    lengths = _int32(lengths, "lengths", (batch,), dev)
    n_new = _int32(n_new, "n_new", (batch,), dev)
    if inv_freq is not None:
        inv_freq = _check_freq(inv_freq, cache.head_dim, dev)
    if batch == 0 or new == 0:
        return
    with _on(dev):
        _lib.check(_lib.load().tt_kv8_append(
            _at(k), _at(v), _TYPES[k.dtype], k.stride(0), k.stride(1), k.stride(2), v.stride(0),
            v.stride(1), v.stride(2), _at(table), table.stride(0), int(table.shape[1]),
            _at(lengths), _at(n_new), _at(inv_freq),
            0 if inv_freq is None else int(inv_freq.shape[0]), int(interleaved), _at(cache._k),
            _at(cache._v), _at(cache.k_scales), _at(cache.v_scales), _at(cache.status), batch,
            new, cache.kv_heads, cache.head_dim, cache.page_size, cache.num_pages,
            _stream_of(dev)), "tt_kv8_append")


def kv_rotate(x: torch.Tensor, lengths: torch.Tensor, inv_freq: torch.Tensor, *,
              interleaved: bool = False) -> torch.Tensor:
    """x (batch, S, heads, head_dim) turned to the positions ``lengths[b] + i``,
    as :func:`kv_append` turns keys; a new tensor. Not differentiated: an x that
    requires grad is refused where gradients are on."""
    dev = x.device
    if dev.type != "cuda":
        raise ValueError(f"kv_rotate: x must be on a CUDA device, got {dev}")
    x = _check_tokens(x, "x", dev)
    batch, new, heads, dim = x.shape
    lengths = _int32(lengths, "lengths", (batch,), dev)
    inv_freq = _check_freq(inv_freq, dim, dev)
    out = torch.empty((batch, new, heads, dim), dtype=x.dtype, device=dev)
    if out.numel():
        with _on(dev):
            _lib.check(_lib.load().tt_kv8_rotate(
                _at(x), _TYPES[x.dtype], x.stride(0), x.stride(1), x.stride(2), _at(lengths),
                _at(inv_freq), int(inv_freq.shape[0]), int(interleaved), _at(out), batch, new,
                heads, dim, _stream_of(dev)), "tt_kv8_rotate")
    return out


def _workspace_bytes(lib, dev: torch.device, dim: int) -> int:
    """Workspace of an attention on the current device ``dev``; a size is kept, a failure is not."""
    n = _WORKSPACE.get((dev.index, dim))
    if n is None:
        n = int(lib.tt_kv8_attention_workspace_bytes(dim))
        if n == 0:
            raise RuntimeError(f"tt_kv8_attention_workspace_bytes: no size for head_dim {dim} on {dev} "
                               f"({lib.tt_last_cuda_error().decode()})")
        _WORKSPACE[dev.index, dim] = n
    return n


def kv_attention(q: torch.Tensor, cache: KVCache8, block_table: torch.Tensor, lengths: torch.Tensor,
                 *, n_query: torch.Tensor | None = None, causal: bool = True,
                 scale: float | None = None) -> torch.Tensor:
    """Softmax attention of q (batch, S, heads, head_dim) over the first
    ``lengths[b]`` tokens of each sequence (after the append).

    Head h reads kv head ``h // (heads // kv_heads)``. Causal: query i of
    ``n_query[b]`` (default S) stands at position ``lengths[b] - n_query[b] + i``
    and sees the tokens up to its own. ``scale`` defaults to
    ``head_dim ** -0.5``. Rows that see no token, and padding rows, are zero.
    Scores, softmax sums and outputs are held in fp32; the result has q's type.
    Nothing here is differentiated: a q that requires grad (or has a tangent) is
    refused where gradients are on.
    """
    dev = cache.device
    q = _check_tokens(q, "q", dev)
    batch, new, heads, dim = q.shape
    if dim != cache.head_dim or heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"q must end in (a multiple of {cache.kv_heads} heads, {cache.head_dim}), "
                         f"got {tuple(q.shape)}")
    table = _check_table(block_table, batch, dev)
    lengths = _int32(lengths, "lengths", (batch,), dev)
    n_query = _int32(n_query, "n_query", (batch,), dev)
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) < 2.0**127:  # the library takes it as fp32, times log2(e)
        raise ValueError(f"scale must be finite, and below 2^127, got {scale}")
    out = torch.empty((batch, new, heads, dim), dtype=q.dtype, device=dev)
    if out.numel() == 0:
        return out
    per = 16 // q.element_size()
    sb, ss, sh, _ = q.stride()
    if q.data_ptr() % 16 or sb % per or ss % per or sh % per:
        q = q.clone(memory_format=torch.contiguous_format)
        sb, ss, sh, _ = q.stride()
    lib = _lib.load()
    with _on(dev):
        ws_bytes = _workspace_bytes(lib, dev, dim)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        _lib.check(lib.tt_kv8_attention(
            _at(q), _TYPES[q.dtype], sb, ss, sh, _at(cache._k),
            _at(cache._v), _at(cache.k_scales), _at(cache.v_scales), _at(table),
            table.stride(0), int(table.shape[1]), _at(lengths), _at(n_query),
            ctypes.byref(ctypes.c_float(scale)), int(causal), _at(out), _at(ws), ws_bytes, _at(cache.status),
            batch, new, heads, cache.kv_heads, dim, cache.page_size, cache.num_pages,
            _stream_of(dev)), "tt_kv8_attention")
    return out
