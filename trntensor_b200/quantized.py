"""Contractions with a matrix that is held in 4 bits.

``W^[n, k] = s[n, k // group] * c[n, k]`` with integer codes ``c`` in -8..7 and
one scale for each group of 32, 64 or 128 neighbouring k of a row. A
:class:`Q4Matrix` is laid out once (``quantize_q4`` from a float matrix,
``pack_q4`` from codes and scales) and stands as an operand of
:func:`trntensor_b200.einsum`, or of :func:`q4_matmul`, for any number of rows.
Both contractions exist: over k (``"mk,nk->mn"``) and over n (``"mn,nk->mk"``),
each the gradient of the other for the dense operand; the matrix itself gets no
gradient. Nothing here has a counterpart in the reference.
"""

from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from . import _lib
from .dispatch import _device, _ptr
from .plan import _check_precision, _parse_subscripts, _validate_subscripts

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_GROUPS = (32, 64, 128)
_FEW_ROWS = 8  # up to here no product needs a workspace
_MOST = 2**31 - 1024  # rows or columns: sizes are 32-bit in the library

_HERE = contextlib.nullcontext()


def _on(dev: torch.device):
    """Context in which ``dev`` is the current CUDA device."""
    return _HERE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _stream_of(dev: torch.device) -> int:
    """Handle of ``dev``'s current stream (the raw query: a Stream object costs
    more than a small launch)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


class Q4Matrix:
    """An (N, K) matrix of 4-bit codes with group scales, in kernel order.

    Made by :func:`quantize_q4` or :func:`pack_q4`; ``packed`` and ``scales``
    are the stored bytes and scales (bf16 or fp32), padded to 16 x 128 blocks,
    ``row_scale`` a power of two a row. ``status`` is a device word in which a
    product notes a device wait that ran out; its result is NaN, and so are those
    of later products of many rows until :meth:`check` has read the word.
    """

    ndim = 2

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int],
                 group: int):
        self.packed, self.scales, self.group = packed, scales, group
        self.shape = torch.Size(shape)
        self.status = torch.zeros((), dtype=torch.int32, device=packed.device)
        n, k = self.shape
        self.row_scale = torch.ones(n, dtype=torch.float32, device=packed.device)
        if n and k and packed.device.type == "cuda":
            with _on(packed.device):
                _lib.check(_lib.load().tt_q4_row_scale(
                    _ptr(scales), _TYPES[scales.dtype], n, k, group, _ptr(self.row_scale),
                    _stream_of(packed.device)), "tt_q4_row_scale")

    def check(self) -> None:
        """Raise if a device wait of a product ran out (waits for the device)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise _lib.DeviceError(f"Q4Matrix: device wait ran out (status 0x{code:x})")

    @property
    def device(self) -> torch.device:
        return self.packed.device

    def dim(self) -> int:
        return 2

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The (N, K) matrix as floats (each product rounded once to ``dtype``)."""
        kind = torch.float32 if dtype == torch.float64 else dtype
        if kind not in _TYPES:
            raise ValueError(f"dequantize: dtype must be a float type, got {dtype}")
        if dtype == torch.float64 and self.scales.dtype == torch.float32:
            # an fp32 scale times a code needs up to 27 bits
            codes = self.codes().double()
            wide = self.group_scales().double().repeat_interleave(self.group, dim=1)
            return codes * wide[:, : self.shape[1]]
        n, k = self.shape
        out = torch.empty((n, k), dtype=kind, device=self.device)
        if out.numel():
            lib = _lib.load()
            with _on(self.device):
                _lib.check(lib.tt_q4_dequantize(
                    _ptr(self.packed), _ptr(self.scales), _TYPES[self.scales.dtype], n, k,
                    self.group, _ptr(out), _TYPES[kind], _stream_of(self.device)),
                    "tt_q4_dequantize")
        return out.to(dtype)

    def codes(self) -> torch.Tensor:
        """The (N, K) int8 codes."""
        n, k = self.shape
        if n == 0 or k == 0:
            return torch.empty((n, k), dtype=torch.int8, device=self.device)
        # [row tile][k block][row half][g][t][word][byte], two codes a byte
        b = self.packed.view(-(-n // 16), -(-k // 128), 2, 8, 4, 4, 4)
        nib = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)  # nibble p of the word
        nib = nib.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-2)  # code i = 2 j + e
        full = nib.permute(0, 2, 3, 1, 5, 4, 6).reshape(16 * b.shape[0], 128 * b.shape[1])
        return (full[:n, :k].to(torch.int16) - 8).to(torch.int8)

    def group_scales(self) -> torch.Tensor:
        """The (N, ceil(K / group)) scales."""
        n, k = self.shape
        s = self.scales.view(-(-n // 16), -(-k // 128), 128 // self.group, 16)
        s = s.permute(0, 3, 1, 2).reshape(16 * s.shape[0], -1)
        return s[:n, : -(-k // self.group)].contiguous()

    def __repr__(self) -> str:
        return f"Q4Matrix(shape={tuple(self.shape)}, group={self.group}, device={self.device})"


def _check_group(group: int) -> None:
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS}, got {group!r}")


def _on_device(t: torch.Tensor) -> torch.Tensor:
    return t if t.device.type == "cuda" else t.to(_device())


def _empty_q4(n: int, k: int, group: int, scale_dtype: torch.dtype, dev: torch.device):
    if max(n, k) > _MOST:
        raise ValueError(f"a 4-bit matrix has at most {_MOST} rows and columns, got {(n, k)}")
    lib = _lib.load()
    packed = torch.empty(int(lib.tt_q4_packed_bytes(n, k)), dtype=torch.uint8, device=dev)
    scales = torch.empty(int(lib.tt_q4_scale_count(n, k, group)), dtype=scale_dtype, device=dev)
    return packed, scales


def quantize_q4(weight: torch.Tensor, *, group: int = 128,
                scale_dtype: torch.dtype = torch.bfloat16) -> Q4Matrix:
    """Quantise an (N, K) float matrix: ``s = amax / 7`` of each group, rounded to
    ``scale_dtype``, and ``c = round(w / s)`` clamped to -8..7.

    A group that holds an infinity or NaN gets the scale NaN. Host matrices are
    copied to the current CUDA device, where the result lives.
    """
    if weight.dim() != 2:
        raise ValueError(f"quantize_q4: weight must be 2D (N, K), got {tuple(weight.shape)}")
    if weight.dtype not in _TYPES:
        raise ValueError(f"quantize_q4: weight must be fp32, bf16 or fp16, got {weight.dtype}")
    _check_group(group)
    if scale_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"quantize_q4: scale_dtype must be bf16 or fp32, got {scale_dtype}")
    w = _on_device(weight.detach())
    if w.stride(1) != 1 or w.stride(0) < max(1, w.shape[1]):
        w = w.contiguous()
    n, k = (int(s) for s in w.shape)
    packed, scales = _empty_q4(n, k, group, scale_dtype, w.device)
    if n and k:
        with _on(w.device):
            _lib.check(_lib.load().tt_q4_quantize(
                _ptr(w), _TYPES[w.dtype], int(w.stride(0)) if n > 1 else k, _TYPES[scale_dtype],
                n, k, group, _ptr(packed), _ptr(scales), _stream_of(w.device)), "tt_q4_quantize")
    return Q4Matrix(packed, scales, (n, k), group)


def pack_q4(codes: torch.Tensor, scales: torch.Tensor, *, group: int = 128) -> Q4Matrix:
    """Lay out given codes (N, K; int8 in -8..7, of which the low four bits are
    kept) and scales (N, ceil(K / group); bf16, or fp32, or fp16, which is kept
    as fp32)."""
    _check_group(group)
    if codes.dim() != 2 or codes.dtype != torch.int8:
        raise ValueError(f"pack_q4: codes must be 2D int8, got {tuple(codes.shape)} {codes.dtype}")
    n, k = (int(s) for s in codes.shape)
    if scales.dtype not in _TYPES or tuple(scales.shape) != (n, -(-k // group)):
        raise ValueError(
            f"pack_q4: scales must be bf16, fp16 or fp32 of shape {(n, -(-k // group))}, "
            f"got {tuple(scales.shape)} {scales.dtype}")
    c = _on_device(codes).contiguous()
    s = scales.detach().to(c.device)
    s = (s.float() if s.dtype == torch.float16 else s).contiguous()
    packed, out = _empty_q4(n, k, group, s.dtype, c.device)
    if n and k:
        with _on(c.device):
            _lib.check(_lib.load().tt_q4_pack(
                _ptr(c), _ptr(s), _TYPES[s.dtype], n, k, group, _ptr(packed), _ptr(out),
                _stream_of(c.device)), "tt_q4_pack")
    return Q4Matrix(packed, out, (n, k), group)


def _product(x: torch.Tensor, w: Q4Matrix, over_n: bool) -> torch.Tensor:
    """(M, K) -> (M, N) or, over_n, (M, N) -> (M, K) on the matrix's device."""
    dev = x.device
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return _product(x, w, over_n)
    n, k = w.shape
    m, have = x.shape
    cols = k if over_n else n
    if m > _MOST:
        raise ValueError(f"q4_matmul: at most {_MOST} rows, got {m}")
    out = x.new_empty((m, cols))
    if m == 0 or cols == 0:
        return out
    if have == 0:
        return out.zero_()
    ldx, inner = x.stride()
    if inner != 1 or ldx < have:
        if m > 1 or inner != 1:
            x = x.contiguous()
        ldx = have
    lib = _lib.load()
    fn = lib.tt_q4_matmul_t if over_n else lib.tt_q4_matmul
    kind = _TYPES[x.dtype]
    ws, ws_bytes = None, 0
    if m > _FEW_ROWS:
        ws_bytes = lib.tt_q4_matmul_workspace_bytes(kind, _TYPES[w.scales.dtype], over_n, m, n, k)
        if ws_bytes:
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    st = fn(x.data_ptr(), kind, ldx, w.packed.data_ptr(), w.scales.data_ptr(),
            _TYPES[w.scales.dtype], w.row_scale.data_ptr(), m, n, k, w.group, out.data_ptr(),
            cols, None if ws is None else ws.data_ptr(), ws_bytes, w.status.data_ptr(),
            _stream_of(dev))
    if st:
        _lib.check(st, "tt_q4_matmul_t" if over_n else "tt_q4_matmul")
    return out


class _Q4Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, over_n):
        ctx.w, ctx.over_n = w, over_n
        return _product(x, w, over_n)

    @staticmethod
    def backward(ctx, dy):
        return _dispatch(dy, ctx.w, not ctx.over_n), None, None

    @staticmethod
    def jvp(ctx, t, *_):  # the map is linear
        return _dispatch(t, ctx.w, ctx.over_n)


def _dispatch(x: torch.Tensor, w: Q4Matrix, over_n: bool) -> torch.Tensor:
    # a tangent asks for no gradient, and stands without grad mode too
    if (x.requires_grad and torch.is_grad_enabled()) or (
            forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None):
        return _Q4Product.apply(x, w, over_n)
    return _product(x.detach() if x.requires_grad else x, w, over_n)


def q4_matmul(x: torch.Tensor, weight: Q4Matrix, *, over_n: bool = False) -> torch.Tensor:
    """``x @ W^T``: (..., K) -> (..., N); with ``over_n`` ``x @ W``: (..., N) -> (..., K).

    x is fp32, bf16 or fp16; sums are fp32 and the result is rounded once to
    x's type. Up to 8 rows (32 of 16-bit types over k, 16 of fp32 over n)
    products over k are exact, and over n they keep 2^-16 (fp32: all bits).
    With more both operands are brought to fp16's
    range by powers of two a row: products are exact where scales are bf16 and
    x is of 16 bits and no smaller than 2^-27 of its row's largest value, else
    they keep 2^-18 (fp32: 2^-20) of themselves and 2^-38 of the largest.
    Differentiable in x, any number of times and in forward mode. A host x is copied to the
    matrix's device and the result comes back.
    """
    if not isinstance(weight, Q4Matrix):
        raise ValueError(f"q4_matmul: weight must be a Q4Matrix, got {type(weight).__name__}")
    if x.dtype not in _TYPES:
        raise ValueError(f"q4_matmul: x must be fp32, bf16 or fp16, got {x.dtype}")
    want = weight.shape[0] if over_n else weight.shape[1]
    if x.dim() < 1 or x.shape[-1] != want:
        raise ValueError(f"q4_matmul: x must end in {want} for {weight!r}, got {tuple(x.shape)}")
    if x.device.type == "cuda" and x.device != weight.device:
        raise ValueError(f"q4_matmul: x is on {x.device}, the matrix on {weight.device}")
    if x.dim() == 2 and x.device == weight.device:
        return _dispatch(x, weight, over_n)
    lead = x.shape[:-1]
    rows = 1
    for s in lead:
        rows *= int(s)
    y = _dispatch(x.to(weight.device).reshape(rows, want), weight, over_n)
    return y.reshape(*lead, y.shape[-1]).to(x.device)


# (subscripts, place of the matrix, dimensions of the dense operand) -> how it runs
_FORMS: dict[tuple, tuple] = {}


def _form(subscripts: str, operands: tuple, held: int) -> tuple:
    """(axis of x that is contracted, its permutation or None, over_n, the
    result's permutation or None) of a contraction with one Q4Matrix."""
    _validate_subscripts(subscripts, operands)
    lhs, out = _parse_subscripts(subscripts)
    terms = lhs.split(",")
    tw, tx = terms[held], terms[1 - held]
    shared = [c for c in tw if c in tx]
    if (len(set(tw)) != 2 or len(set(tx)) != len(tx) or len(set(out)) != len(out)
            or len(shared) != 1 or shared[0] in out):
        raise ValueError(
            f"einsum {subscripts!r}: a Q4Matrix is contracted over exactly one of its indices, "
            "which the output drops; use dequantize() for other forms")
    c = shared[0]
    free = tw[1] if c == tw[0] else tw[0]
    rest = [ch for ch in tx if ch != c]
    if set(out) != set(rest) | {free}:
        raise ValueError(f"einsum {subscripts!r}: every uncontracted index must be in the output")
    into = [tx.index(ch) for ch in rest + [c]]
    order = [(rest + [free]).index(ch) for ch in out]
    plain = list(range(len(into)))
    return (tx.index(c), None if into == plain else into, c == tw[0],
            None if order == list(range(len(order))) else order)


def einsum_q4(subscripts: str, operands: tuple, precision: str) -> torch.Tensor:
    """Two-operand einsum with one :class:`Q4Matrix`: a product over k or over n
    with the dense operand's other indices kept."""
    if len(operands) != 2 or isinstance(operands[0], Q4Matrix) == isinstance(operands[1], Q4Matrix):
        _validate_subscripts(subscripts, operands)
        raise ValueError(
            f"einsum {subscripts!r}: a Q4Matrix contracts with one dense operand; "
            "use dequantize() for other forms")
    held = 0 if isinstance(operands[0], Q4Matrix) else 1
    w, x = operands[held], operands[1 - held]
    key = (subscripts, held, x.dim())
    form = _FORMS.get(key)
    if form is None:
        form = _FORMS[key] = _form(subscripts, operands, held)
    axis, into, over_n, order = form
    if x.shape[axis] != w.shape[0 if over_n else 1]:
        _validate_subscripts(subscripts, operands)
    if precision != "fast":
        from .einsum import einsum

        _check_precision(precision)
        ops = [x.double(), x.double()]
        ops[held] = w.dequantize(torch.float64).to(x.device)
        return einsum(subscripts, *ops, precision=precision).to(x.dtype)
    y = q4_matmul(x if into is None else x.permute(into), w, over_n=over_n)
    return y if order is None else y.permute(order).contiguous()
