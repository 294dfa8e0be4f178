"""The 8-bit cache on the GPU: appending against the definition, step by step in
the same fp32 operations, and attention against it in 64 bits.

Tolerances of attention. The scores' fp32 sums are chains of at most
dim / 16 + 16 additions, each off by at most 2^-23 of sum |q k|; two more
roundings bring a score's error to d = (dim / 16 + 20) 2^-23 max_t sum |q k|
scale, and ex2.approx adds 2^-21 of a weight. Weights are rounded to fp16,
whose 11 significant bits leave half a step of 2^-11 (two terms for fp32
operands: 2^-22), and q of fp32 likewise (2^-22 of its row's largest value).
Below fp16's normal range a weight is off by half of 2^-24, in units of which
the largest weight is at least 2^3. Numerator and denominator take the score's
error once each. The sums over tokens add at most L / 16 + 64 roundings of
2^-23. Everything is relative to a = sum p |v|; the result is rounded once.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import trntensor_b200 as tt
from trntensor_b200 import _lib

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Ref:
    """A cache in the definition's operations (fp32, one rounding each)."""

    def __init__(self, cache):
        k, v = cache.codes()
        self.codes = [k.cpu().numpy().astype(np.float32), v.cpu().numpy().astype(np.float32)]
        self.scales = [cache.k_scales.cpu().numpy().copy(), cache.v_scales.cpu().numpy().copy()]
        self.page = cache.page_size

    def append(self, x, which, table, lengths, counts):
        codes, scales, f = self.codes[which], self.scales[which], np.float32
        for b, (a, c) in enumerate(zip(lengths, counts)):
            at = a
            while at < a + c:
                end = min(a + c, (at // self.page + 1) * self.page)
                page, slot = table[b][at // self.page], at % self.page
                new = x[b, at - a:end - a]
                for h in range(new.shape[1]):
                    old = f(0) if slot == 0 else scales[page, h]
                    top = np.abs(new[:, h]).max()
                    need = f(top) / f(127) if np.isfinite(top) else f("nan")
                    now = f("nan") if np.isnan(old) or np.isnan(need) else max(old, need)
                    if now > old and slot:
                        codes[page, h, :slot] = np.rint(codes[page, h, :slot] * (old / now))
                    fresh = np.zeros_like(new[:, h])
                    if now > 0:
                        fresh = np.clip(np.rint(new[:, h] / now), -127, 127)
                    codes[page, h, slot:slot + end - at] = fresh
                    scales[page, h] = now
                at = end

    def same(self, cache):
        k, v = cache.codes()
        for got, want in ((k, self.codes[0]), (v, self.codes[1]),
                          (cache.k_scales, self.scales[0]), (cache.v_scales, self.scales[1])):
            np.testing.assert_array_equal(got.cpu().numpy().astype(np.float32), want)


def filled(pages, kv, page, dim, seed=0, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    kc = torch.randint(-127, 128, (pages, kv, page, dim), generator=g, dtype=torch.int8)
    vc = torch.randint(-127, 128, (pages, kv, page, dim), generator=g, dtype=torch.int8)
    ks = torch.exp(spread * torch.randn(pages, kv, generator=g)) / 60
    vs = torch.exp(spread * torch.randn(pages, kv, generator=g)) / 60
    return kc, ks, vc, vs


def test_codes_round_trip(cuda_ok):
    for page, dim in ((16, 16), (64, 128), (128, 80)):
        kc, ks, vc, vs = filled(4, 3, page, dim)
        c = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
        k, v = c.codes()
        assert torch.equal(k.cpu(), kc) and torch.equal(v.cpu(), vc)
        ids = [2, 0, 2]
        for dtype in TYPES.values():
            k, v = c.dequantize(int32(ids), dtype=dtype)
            assert torch.equal(k.cpu(), (kc[ids].float() * ks[ids][..., None, None]).to(dtype))
            assert torch.equal(v.cpu(), (vc[ids].float() * vs[ids][..., None, None]).to(dtype))
        assert torch.equal(c.dequantize()[1].cpu(), vc.float() * vs[..., None, None])
        c.check()
        k, _ = c.dequantize(int32([1, 4, -1]))
        assert torch.equal(k[0].cpu(), kc[1].float() * ks[1][..., None, None]) and not k[1:].any()
        with pytest.raises(ValueError, match="page id"):
            c.check()
        k, _ = c.dequantize(torch.tensor([1, 2**32, -2**32], device="cuda"))  # 64 bits
        assert torch.equal(k[0].cpu(), kc[1].float() * ks[1][..., None, None]) and not k[1:].any()
        with pytest.raises(ValueError, match="page id"):
            c.check()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("page,dim,kv", [(16, 16, 1), (32, 80, 3), (64, 128, 2), (128, 256, 1)])
def test_append_step_by_step(cuda_ok, page, dim, kv, name):
    """Prompts, single tokens, padding and a restarted page, in one cache."""
    dtype, batch, cols = TYPES[name], 3, 5
    cache = tt.KVCache8(batch * cols + 2, kv, dim, page_size=page)
    ref = Ref(cache)
    g = torch.Generator().manual_seed(page + dim)
    table = torch.randperm(batch * cols, generator=g).view(batch, cols).tolist()
    lengths = [0, 0, 0]
    steps = [[0, 1, 2 * page + 3], [page, 5, 1], [1, 1, 1], [1, 0, 1], [page + 1, page - 6, 2], [1, 1, 1]]
    for n, counts in enumerate(steps):
        new = max(counts)
        # values grow and shrink: some steps need larger scales, others do not
        k = (torch.randn(batch, new, kv, dim, generator=g) * (1 + n % 3)).to(dtype)
        v = (torch.randn(batch, new, kv, dim, generator=g) * (3 - n % 3)).to(dtype)
        tt.kv_append(cache, k.cuda(), v.cuda(), int32(table), int32(lengths), n_new=int32(counts))
        ref.append(k.float().numpy(), 0, table, lengths, counts)
        ref.append(v.float().numpy(), 1, table, lengths, counts)
        ref.same(cache)
        lengths = [a + c for a, c in zip(lengths, counts)]
    # the first sequence ends; its pages serve again, what is behind the new tokens stays
    k = torch.randn(1, 3, kv, dim, generator=g).to(dtype)
    tt.kv_append(cache, k.cuda(), k.cuda(), int32(table[:1]), int32([0]))
    ref.append(k.float().numpy(), 0, table[:1], [0], [3])
    ref.append(k.float().numpy(), 1, table[:1], [0], [3])
    ref.same(cache)
    cache.check()


def test_append_strides_and_zeros(cuda_ok):
    cache = tt.KVCache8(6, 2, 32, page_size=16)
    ref = Ref(cache)
    big = torch.randn(2, 7, 2, 3, 32, device="cuda")  # k, v and something else side by side
    k, v = big[:, :5, :, 0], big[:, :5, :, 2]
    table = torch.tensor([[9, 0, 9, 3], [9, 5, 9, 1]], dtype=torch.int32, device="cuda")[:, 1::2]
    tt.kv_append(cache, k, v, table, int32([14, 0]))
    ref.append(k.cpu().numpy(), 0, table.tolist(), [14, 0], [5, 5])
    ref.append(v.cpu().numpy(), 1, table.tolist(), [14, 0], [5, 5])
    ref.same(cache)
    zero = torch.zeros(1, 4, 2, 32, device="cuda")
    tt.kv_append(cache, zero, zero, int32([[2]]), int32([0]))
    assert not cache.k_scales[2].any() and not cache.codes()[0][2].any()
    tt.kv_append(cache, zero, zero, int32([[2]]), int32([4]))
    assert not cache.v_scales[2].any()
    tt.kv_append(cache, zero[:, :0], zero[:, :0], int32([[2]]), int32([4]))
    cache.check()


def test_append_not_finite(cuda_ok):
    cache = tt.KVCache8(4, 2, 32, page_size=16)
    ref = Ref(cache)
    k = torch.randn(1, 20, 2, 32)
    v = k.clone()
    k[0, 3, 1, 5], v[0, 18, 0, 0] = float("inf"), float("nan")
    for a, x in ((k, 0), (v, 1)):
        ref.append(a.numpy(), x, [[2, 1]], [0], [20])
    tt.kv_append(cache, k.cuda(), v.cuda(), int32([[2, 1]]), int32([0]))
    ref.same(cache)
    assert cache.k_scales.isnan().nonzero().tolist() == [[2, 1]]
    assert cache.v_scales.isnan().nonzero().tolist() == [[1, 0]]
    one = torch.randn(1, 1, 2, 32)  # a NaN page stays so until it starts anew
    tt.kv_append(cache, one.cuda(), one.cuda(), int32([[2, 1]]), int32([20]))
    assert cache.v_scales.isnan().nonzero().tolist() == [[1, 0]]
    tt.kv_append(cache, one.cuda(), one.cuda(), int32([[2, 1]]), int32([16]))
    assert not cache.v_scales.isnan().any()


def turned(x, pos, inv_freq, interleaved):
    """x (batch, S, heads, dim) float64 turned at pos (batch, S)."""
    half = len(inv_freq)
    a = pos[:, :, None, None] * inv_freq.double()
    c, s = torch.cos(a), torch.sin(a)
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out = x.clone()
    out[..., one] = x[..., one] * c - x[..., two] * s
    out[..., two] = x[..., two] * c + x[..., one] * s
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(16, 8), (64, 16), (128, 64), (80, 40), (96, 1)])
@pytest.mark.parametrize("start", [0, 1000003])
def test_rotation(cuda_ok, dim, half, interleaved, start):
    """Far positions too: angles of a million radians, exact to fp32."""
    g = torch.Generator().manual_seed(dim)
    page, new = 16, 19
    cols = (start + new) // page + 1
    freq = (10000.0 ** (-torch.arange(half) / half)).float()
    k = torch.randn(1, new, 2, dim, generator=g)
    cache = tt.KVCache8(4, 2, dim, page_size=page)
    table = torch.full((1, cols), 0, dtype=torch.int32)
    for n, col in enumerate(range(start // page, cols)):
        table[0, col] = n
    lengths = int32([start])
    tt.kv_append(cache, k.cuda(), k.cuda(), table.cuda(), lengths, inv_freq=freq.cuda(), interleaved=interleaved)
    cache.check()
    want = turned(k.double(), torch.arange(start, start + new)[None].double(), freq, interleaved)
    got = tt.kv_rotate(k.cuda(), lengths, freq.cuda(), interleaved=interleaved)
    # the angle to 2^-23 turns of a half circle, the sine and the sum to a few units
    assert (got.cpu().double() - want).abs().max() <= 2.0**-20 * k.abs().max()
    values, plain = cache.dequantize()
    for t in range(new):
        page_no, slot = int(table[0, (start + t) // page]), (start + t) % page
        step = cache.k_scales[page_no].cpu().double()[:, None]
        off = (values[page_no, :, slot].cpu().double() - want[0, t]).abs()
        assert (off <= 0.5001 * step + 2.0**-19 * k.abs().max()).all()
        off = (plain[page_no, :, slot].cpu().double() - k[0, t].double()).abs()
        assert (off <= 0.5001 * cache.v_scales[page_no].cpu().double()[:, None]).all()


def test_append_notes_what_is_wrong(cuda_ok):
    k = torch.randn(2, 3, 1, 16, device="cuda")

    def fresh():
        return tt.KVCache8(4, 1, 16, page_size=16)

    for table, lengths, counts, word in (
            ([[0], [4]], [0, 0], [3, 3], "page id"), ([[0], [-1]], [0, 0], [3, 3], "page id"),
            ([[0], [1]], [0, 14], [3, 3], "length"), ([[0], [1]], [0, -1], [3, 3], "length"),
            ([[0], [1]], [0, 0], [3, 4], "length"), ([[0], [1]], [0, 2**31 - 1], [3, 3], "length"),
            ([[2], [2]], [0, 5], [3, 3], "two places"), ([[0, 3, 3], [1, 2, 2]], [0, 30], [3, 3], "two places")):
        c = fresh()
        tt.kv_append(c, k, k, int32(table), int32(lengths), n_new=int32(counts))
        with pytest.raises(ValueError, match=word):
            c.check()
        if word != "two places":  # the sound sequence is written all the same
            want = fresh()
            tt.kv_append(want, k[:1], k[:1], int32([table[0]]), int32([0]))
            assert torch.equal(c.codes()[0][0], want.codes()[0][0])
    c = fresh()  # shared pages that are only read are nothing wrong
    tt.kv_append(c, k, k, int32([[0, 1], [0, 2]]), int32([16, 16]))
    c.check()


def reference(q, parts, table, lengths, counts, causal, scale):
    """(o, tolerance terms) in 64 bits: q (batch, S, heads, dim) on the CPU."""
    kc, ks, vc, vs = parts
    kk, vv = kc.double() * ks.double()[..., None, None], vc.double() * vs.double()[..., None, None]
    batch, new, heads, dim = q.shape
    kv = kc.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64)
    loss = torch.zeros(q.shape, dtype=torch.float64)
    two = q.dtype == torch.float32
    for b in range(batch):
        n, c = lengths[b], counts[b]
        ids = table[b][:-(-n // kc.shape[2])]
        k = kk[ids].transpose(0, 1).flatten(1, 2)[:, :n]
        v = vv[ids].transpose(0, 1).flatten(1, 2)[:, :n]
        for i in range(c):
            see = n - c + i + 1 if causal else n
            if see <= 0:
                continue
            for h in range(heads):
                kh, vh = k[h // (heads // kv), :see], v[h // (heads // kv), :see]
                x = q[b, i, h].double()
                p = torch.softmax(kh @ x * scale, 0)
                o[b, i, h] = p @ vh
                mass = p @ vh.abs()
                d = (dim / 16 + 20) * 2.0**-23 * float((kh.abs() @ x.abs()).max()) * abs(scale)
                if two:
                    d += 2.0**-22 * float(x.abs().max() * kh.abs().sum(1).max()) * abs(scale)
                e = (2.0**-22 if two else 2.0**-11) + 2 * d + 2.0**-20 + (n / 16 + 64) * 2.0**-22
                loss[b, i, h] = e * mass + n * 2.0**-28 * float(p.max() * vh.abs().max())
    return o, loss


def attend_case(name, batch, new, heads, kv, dim, page, lengths, counts=None, causal=True, scale=None,
                q_scale=2.0, spread=0.5, seed=0):
    dtype = TYPES[name]
    g = torch.Generator().manual_seed(seed + dim + page)
    cols = max(1, -(-max(lengths) // page))
    pages = batch * cols
    parts = filled(pages, kv, page, dim, seed, spread)
    table = torch.randperm(pages, generator=g).view(batch, cols)
    q = (torch.randn(batch, new, heads, dim, generator=g) * q_scale).to(dtype)
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    got = tt.kv_attention(q.cuda(), cache, table.int().cuda(), int32(lengths),
                          n_query=None if counts is None else int32(counts), causal=causal, scale=scale)
    cache.check()
    used = [new] * batch if counts is None else counts
    want, loss = reference(q, parts, table.tolist(), lengths, used, causal,
                           dim**-0.5 if scale is None else scale)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 1.01 * loss + torch.finfo(dtype).tiny
    off = (got.cpu().double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert not (off > tol).any() and not off.isnan().any(), (off / tol).max().item()
    for b in range(batch):
        assert not got[b, used[b]:].any()
    return got, want


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("dim,page,heads,kv", [
    (16, 16, 1, 1), (64, 16, 12, 12), (80, 32, 6, 2), (96, 64, 5, 1), (128, 64, 8, 1), (128, 16, 40, 2),
    (192, 128, 3, 3), (256, 32, 4, 2)])
def test_single_tokens(cuda_ok, dim, page, heads, kv, name):
    attend_case(name, 5, 1, heads, kv, dim, page, [1, 16, 65, 300, 0])


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,page,heads,kv,new,lengths,counts", [
    (64, 16, 4, 2, 5, [5, 40, 130], None), (128, 64, 8, 2, 9, [9, 64, 200], [9, 1, 0]),
    (32, 32, 3, 1, 33, [33, 90, 20], [33, 7, 33]), (128, 16, 6, 6, 70, [70, 300, 129], [70, 64, 65]),
    (256, 64, 2, 1, 20, [100, 20, 64], None), (80, 128, 4, 1, 130, [130, 257, 260], [130, 1, 129]),
    (128, 64, 12, 6, 150, [700, 150, 20], [150, 149, 150]), (64, 32, 16, 16, 60, [60, 128, 513], [60, 1, 59]),
    (96, 16, 24, 3, 40, [300, 40, 41], None), (16, 16, 8, 8, 300, [300, 1, 129], [300, 1, 128])])
def test_several_tokens(cuda_ok, dim, page, heads, kv, new, lengths, counts, causal, name):
    """Tokens that enter with a prompt or a draft; more queries than tokens leave rows that see nothing."""
    attend_case(name, 3, new, heads, kv, dim, page, lengths, counts, causal)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,page,heads,kv,new,lengths,counts", [
    (64, 32, 16, 16, 210, [210, 128, 513], [210, 1, 209]), (96, 16, 24, 3, 140, [300, 40, 41], None),
    (16, 16, 8, 8, 400, [400, 1, 129], [400, 1, 128]), (80, 128, 4, 1, 800, [830, 257, 260], [800, 1, 129]),
    (128, 64, 12, 6, 270, [700, 150, 20], [270, 149, 270]), (128, 16, 40, 40, 64, [64, 65, 1000], [64, 63, 64])])
def test_tiles_of_many_rows(cuda_ok, dim, page, heads, kv, new, lengths, counts, causal, name):
    """Enough rows for the tensor cores' tiles on any GPU of up to 148 SMs."""
    attend_case(name, 3, new, heads, kv, dim, page, lengths, counts, causal)


@pytest.mark.parametrize("length", [1000, 20011])
def test_long_and_ragged(cuda_ok, length):
    attend_case("bf16", 1, 1, 8, 2, 128, 64, [length])
    attend_case("fp32", 4, 2, 2, 1, 64, 16, [length, 3, length // 2, 17])
    got, _ = attend_case("fp16", 7, 1, 4, 4, 128, 128, [length // (b + 1) for b in range(7)])


def test_long_sums_of_fp32(cuda_ok):
    """So many sequences that a warp has a hundred blocks of 64 tokens of each:
    what the tensor cores cut off may add up inside a block (8 additions, and the
    score's own), then rounded ones follow (half of 2^-23 a block, and a rounding
    of each block's own sum of weights). All sequences read the same pages; all
    values are positive, so that every cut goes the same way."""
    pages, dim, batch = 128, 64, 1000
    kc, ks, vc, vs = filled(pages, 1, 64, dim, seed=9, spread=0.1)
    vc = vc.abs().clamp(min=1)
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    q = torch.randn(batch, 1, 1, dim, generator=torch.Generator().manual_seed(3)) * 0.1
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, -1)
    got = tt.kv_attention(q.cuda(), cache, table, int32([64 * pages] * batch)).double().cpu()
    k = (kc.double() * ks.double()[..., None, None]).reshape(-1, dim)
    v = (vc.double() * vs.double()[..., None, None]).reshape(-1, dim)
    s = q[:, 0, 0].double() @ k.T * dim ** -0.5
    want = torch.softmax(s, -1) @ v
    d = (dim / 16 * 2 + 20) * 2.0**-23 * (q[:, 0, 0].double().abs() @ k.abs().T).max().item() * dim ** -0.5
    tol = 2 * d + 2 * 2.0**-22 + 2.0**-21 + (8 + pages / 2 + 8) * 2.0**-23
    worst = ((got[:, 0, 0] - want).abs() / want).max().item()
    assert worst <= tol, (worst, tol)


@pytest.mark.parametrize("name", list(TYPES))
def test_extremes(cuda_ok, name):
    attend_case(name, 2, 1, 4, 2, 64, 16, [100, 50], q_scale=0.0)       # all scores alike
    attend_case(name, 2, 1, 4, 2, 64, 16, [100, 50], q_scale=60.0)      # one token has all the weight
    attend_case(name, 2, 1, 4, 2, 64, 16, [100, 50], scale=-0.3)
    attend_case(name, 2, 1, 4, 2, 64, 16, [100, 50], scale=0.0)
    attend_case(name, 2, 3, 4, 2, 64, 16, [500, 60], spread=6.0)        # scales decades apart


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("more", [
    {"q_scale": 0.0}, {"q_scale": 60.0}, {"scale": -0.3}, {"scale": 0.0}, {"spread": 6.0}])
def test_extremes_of_many_rows(cuda_ok, name, more):
    attend_case(name, 3, 800, 4, 1, 64, 16, [830, 257, 900], **more)
    attend_case(name, 3, 800, 4, 1, 64, 16, [0, 1, 900], counts=[800, 0, 800], **more)


def test_negative_scales(cuda_ok):
    """A sign in a scale means the same as in its codes."""
    kc, ks, vc, vs = filled(8, 2, 16, 32)
    ks[::2], vs[1::3] = -ks[::2], -vs[1::3]
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    k, v = cache.dequantize()
    assert torch.equal(k.cpu(), kc.float() * ks[..., None, None])
    assert torch.equal(v.cpu(), vc.float() * vs[..., None, None])
    q = torch.randn(1, 3, 4, 32)
    got = tt.kv_attention(q.cuda(), cache, int32([list(range(8))]), int32([125]))
    want, loss = reference(q, (kc, ks, vc, vs), [list(range(8))], [125], [3], True, 32**-0.5)
    assert ((got.cpu().double() - want).abs() <= 2.0**-24 * want.abs() + loss).all()


def test_zero_pages_and_rows(cuda_ok):
    kc, ks, vc, vs = filled(8, 1, 16, 32)
    vs[::2] = 0
    ks[1::3] = 0
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    q = torch.randn(1, 1, 2, 32)
    got = tt.kv_attention(q.cuda(), cache, int32([list(range(8))]), int32([120]))
    want, loss = reference(q, (kc, ks, vc, vs), [list(range(8))], [120], [1], True, 32**-0.5)
    assert ((got.cpu().double() - want).abs() <= 2.0**-24 * want.abs() + loss).all()
    none = tt.kv_attention(q.cuda(), cache, int32([list(range(8))]), int32([0]))
    assert not none.any()
    assert tt.kv_attention(q.cuda()[:, :0], cache, int32([[0]]), int32([4])).shape == (1, 0, 2, 32)
    assert tt.kv_attention(q.cuda()[:0], cache, int32([[0]])[:0], int32([4])[:0]).shape == (0, 1, 2, 32)


@pytest.mark.parametrize("new", [1, 40, 140, 900, 1300])
def test_not_finite_stays_where_it_belongs(cuda_ok, new):
    """A NaN scale, or an infinite query, reaches the rows that see it and no others."""
    kc, ks, vc, vs = filled(24, 2, 16, 64)
    table = [list(range(12)), list(range(12, 24))]
    vs[9, 0] = float("nan")   # tokens 144 .. 159 of sequence 0, kv head 0
    ks[8, 1] = float("nan")   # tokens 128 .. 143, kv head 1
    vs[3 + 12, 0] = ks[3 + 12, 1] = float("nan")  # sequence 1 does not reach it
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    q = torch.randn(2, new, 4, 64)
    lengths = [150, 48]
    counts = [new, min(new, 48)]
    for dtype in TYPES.values():
        got = tt.kv_attention(q.to(dtype).cuda(), cache, int32(table), int32(lengths), n_query=int32(counts))
        first = 150 - new  # position of query 0
        for i in range(new):
            assert bool(got[0, i, :2].isnan().all()) == (first + i >= 144), i
            assert bool(got[0, i, 2:].isnan().all()) == (first + i >= 128), i
        assert got[0].isnan().any(-1).equal(got[0].isnan().all(-1))
        assert not got[1].isnan().any() and not got[1, counts[1]:].any()
    q[0, 0, 0, 3], q[1, 0, 1, 0] = float("inf"), float("nan")
    got = tt.kv_attention(q.cuda(), cache, int32([table[1], table[1]]), int32([40, 40]), n_query=int32([1, 1]))
    bad = got.isnan().any(-1).nonzero().tolist()
    assert bad == [[0, 0, 0], [1, 0, 1]]


@pytest.mark.parametrize("new", [1, 40, 1300])
def test_infinite_scales_stay_where_they_belong(cuda_ok, new):
    """Rows that do not see a page are as they were; those that do are not finite."""
    kc, ks, vc, vs = filled(12, 2, 16, 64, seed=4)
    q = torch.randn(2, new, 8, 64, device="cuda")
    table, lengths = int32([list(range(12)), list(range(12))]), int32([192, 150])
    for dtype in TYPES.values():
        want = tt.kv_attention(q.to(dtype), tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda()),
                               table, lengths)
        wild = vs.clone()
        wild[11] = float("inf")  # tokens 176 .. 191: rows from position 176 of sequence 0
        got = tt.kv_attention(q.to(dtype), tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), wild.cuda()),
                              table, lengths)
        first = max(0, 176 - (192 - new))
        assert not got[0, first:].isfinite().any()
        # (weights are relative to the largest scale in sight, and round by it)
        tol = {torch.float32: 1e-5, torch.float16: 2.0**-9, torch.bfloat16: 2.0**-7}[dtype]
        assert ((got - want)[0, :first].abs() <= tol * want[0, :first].abs().amax(-1, keepdim=True)).all()
        assert ((got - want)[1].abs() <= tol * want[1].abs().amax(-1, keepdim=True)).all()


def test_stale_slots_do_not_matter(cuda_ok):
    """Codes and pages behind a sequence's end, and NaN scales of pages that it does not use."""
    kc, ks, vc, vs = filled(6, 2, 64, 128)
    q = torch.randn(2, 2, 4, 128, device="cuda")
    table, lengths = int32([[0, 1, 5], [2, 3, 4]]), int32([70, 100])
    want = tt.kv_attention(q, tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda()), table, lengths)
    kc[1, :, 6:], vc[1, :, 6:], kc[3, :, 36:], vc[3, :, 36:] = 127, -127, -127, 127
    for s in (ks, vs):
        s[5], s[4] = float("nan"), float("inf")
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    assert torch.equal(tt.kv_attention(q, cache, table, lengths), want)
    wild = int32([[0, 1, 2**31 - 1], [2, 3, -7]])  # columns behind the end are not looked at
    assert torch.equal(tt.kv_attention(q, cache, wild, lengths), want)
    cache.check()


def test_attention_notes_what_is_wrong(cuda_ok):
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in filled(4, 1, 16, 32)))
    q = torch.randn(1, 2, 1, 32, device="cuda")
    for table, lengths, counts, word in (([[0, 4]], [20], [2], "page id"), ([[0, -1]], [32], [2], "page id"),
                                         ([[0, 1]], [33], [2], "length"), ([[0, 1]], [-1], [2], "length"),
                                         ([[0, 1]], [20], [3], "length"), ([[0, 1]], [0], [-2], "length")):
        out = tt.kv_attention(q, cache, int32(table), int32(lengths), n_query=int32(counts))
        assert out.isfinite().all()
        with pytest.raises(ValueError, match=word):
            cache.check()
    want = tt.kv_attention(q, cache, int32([[0, 1]]), int32([20]))  # and the cache still serves
    assert want.abs().max() > 0
    cache.check()


def test_query_strides(cuda_ok):
    parts = filled(8, 2, 32, 64)
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    table, lengths = int32([[0, 1, 2, 3], [4, 5, 6, 7]]), int32([100, 128])
    for dtype in TYPES.values():
        big = torch.randn(2, 5, 8, 64, device="cuda").to(dtype)
        for q in (big[:, 1:4], big[:, :, 2:6], big.transpose(1, 2)[:, 2:6, :4], big[:, :, :, :64].flip(1),
                  torch.randn(2, 3, 4, 65, device="cuda").to(dtype)[..., 1:]):
            want = tt.kv_attention(q.contiguous(), cache, table, lengths)
            assert torch.equal(tt.kv_attention(q, cache, table, lengths), want)


@pytest.mark.parametrize("new,heads", [(1, 8), (6, 4), (200, 4), (1200, 8)])
def test_same_bits_graphs_and_streams(cuda_ok, new, heads):
    """Eager calls, two graphs and two streams at a time give the same bits."""
    parts = filled(64, 2, 32, 128)
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    lengths = int32([1000, 700])
    q = torch.randn(2, new, heads, 128, device="cuda", dtype=torch.bfloat16)
    want = tt.kv_attention(q, cache, table, lengths)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = tt.kv_attention(q, cache, table, lengths)
        graphs.append((gr, out))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for (gr, _), st in zip(graphs, side):
            with torch.cuda.stream(st):
                gr.replay()
        eager = tt.kv_attention(q, cache, table, lengths)
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)


def test_decode_step_in_a_graph(cuda_ok):
    """Append, rotate and attend as a serving step does, eagerly and replayed: lengths
    move on the device, and each step equals the definition on the cache's own values."""
    batch, kv, heads, dim, page, cols = 3, 2, 6, 64, 16, 6
    freq = (10000.0 ** (-torch.arange(dim // 2) / (dim // 2))).float().cuda()
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(batch * cols, generator=g).view(batch, cols).int().cuda()

    def setup():
        cache = tt.KVCache8(batch * cols, kv, dim, page_size=page)
        k = torch.randn(batch, 40, kv, dim, generator=torch.Generator().manual_seed(4)).cuda()
        tt.kv_append(cache, k, k * 2, table, int32([0, 0, 0]), n_new=int32([40, 15, 1]), inv_freq=freq)
        return cache, int32([40, 15, 1])

    def step(cache, lengths, q, k, v):
        tt.kv_append(cache, k, v, table, lengths, inv_freq=freq)
        turned_q = tt.kv_rotate(q, lengths, freq)
        lengths += 1
        return turned_q, tt.kv_attention(turned_q, cache, table, lengths)

    tokens = [[torch.randn(batch, 1, n, dim, generator=g).to(torch.bfloat16).cuda() for n in (heads, kv, kv)]
              for _ in range(20)]
    cache, lengths = setup()
    eager = []
    for q, k, v in tokens:
        tq, o = step(cache, lengths, q, k, v)
        eager.append(o)
        kc, vc = cache.codes()
        parts = (kc.cpu(), cache.k_scales.cpu(), vc.cpu(), cache.v_scales.cpu())
        want, loss = reference(tq.cpu(), parts, table.tolist(), lengths.tolist(), [1] * batch, True, dim**-0.5)
        assert ((o.cpu().double() - want).abs() <= 2.0**-8 * want.abs() + 1.01 * loss).all()
    cache.check()
    again, moving = setup()
    held = [torch.empty_like(x) for x in tokens[0]]
    warm = torch.cuda.Stream()
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr, stream=warm):
        _, out = step(again, moving, *held)
    for (q, k, v), want in zip(tokens, eager):
        for a, b in zip(held, (q, k, v)):
            a.copy_(b)
        gr.replay()
        assert torch.equal(out, want)
    assert torch.equal(moving, lengths) and torch.equal(again.codes()[1], cache.codes()[1])
    again.check()


def test_offsets_past_32_bits(cuda_ok):
    """Pages whose codes lie more than 2^31 bytes into the cache."""
    page, kv, dim = 128, 8, 256
    pages = 2**31 // (page * kv * dim) + 6
    cache = tt.KVCache8(pages, kv, dim, page_size=page)
    small = tt.KVCache8(4, kv, dim, page_size=page)
    k = torch.randn(1, 300, kv, dim, device="cuda", dtype=torch.bfloat16)
    far, near = int32([[pages - 1, 0, pages - 2]]), int32([[3, 0, 1]])
    q = torch.randn(1, 2, kv, dim, device="cuda", dtype=torch.bfloat16)
    for c, t in ((cache, far), (small, near)):
        tt.kv_append(c, k, -k, t, int32([0]))
        c.check()
    a = tt.kv_attention(q, cache, far, int32([300]))
    assert torch.equal(a, tt.kv_attention(q, small, near, int32([300])))
    x, y = cache.dequantize(int32([pages - 1]))
    p, r = small.dequantize(int32([3]))
    assert torch.equal(x, p) and torch.equal(y, r)


def test_workspace_is_checked(cuda_ok):
    import ctypes

    lib = _lib.load()
    cache = tt.KVCache8(1, 1, 32, page_size=16)
    q = torch.zeros(1, 1, 1, 32, device="cuda")
    need = lib.tt_kv8_attention_workspace_bytes(32)
    assert need > 0 and lib.tt_kv8_attention_workspace_bytes(33) == 0
    t, n = int32([[0]]), int32([1])
    p = [x.data_ptr() for x in (q, cache._k, cache._v, cache.k_scales, cache.v_scales, t, n, cache.status)]
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    rc = lib.tt_kv8_attention(p[0], 0, 32, 32, 32, p[1], p[2], p[3], p[4], p[5], 1, 1, p[6], None,
                              ctypes.byref(ctypes.c_float(1.0)), 1, p[0], ws.data_ptr(), need - 1, p[7], 1, 1, 1,
                              1, 32, 16, 1, None)
    assert rc == _lib.TT_ERR_WORKSPACE
