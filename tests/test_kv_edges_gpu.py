"""The 8-bit cache on the GPU where it can go wrong: scales far apart, pages that
are not there, shared pages, subnormal values, rotation in every page size.

Tolerances of attention are those of test_kv_gpu, with what a case names."""

from __future__ import annotations

import pytest
import torch
from test_kv_gpu import TYPES, Ref, attend_case, filled, int32, reference, turned

import trntensor_b200 as tt
from trntensor_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("new", [1, 20, 1300])
@pytest.mark.parametrize("factor", [1e6, 1e10])
def test_large_scales_out_of_sight(cuda_ok, factor, new, name):
    """A page with finite value scales far above the others', which most rows do not see:
    those rows come out as the definition has them."""
    kc, ks, vc, vs = filled(12, 2, 16, 64, seed=4)
    vs[11] *= factor  # tokens 176 .. 191
    parts = (kc, ks, vc, vs)
    q = torch.randn(2, new, 8, 64, generator=torch.Generator().manual_seed(new)).to(TYPES[name])
    table, lengths = [list(range(12))] * 2, [192, 150]
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    got = tt.kv_attention(q.cuda(), cache, int32(table), int32(lengths)).cpu()
    cache.check()
    want, loss = reference(q, parts, table, lengths, [new] * 2, True, 64**-0.5)
    tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 1.01 * loss + torch.finfo(q.dtype).tiny
    first = max(0, 176 - (192 - new))  # the first row of sequence 0 that sees it
    for g, w, t in ((got[0, :first], want[0, :first], tol[0, :first]), (got[1], want[1], tol[1])):
        assert not ((g.double() - w).abs() > t).any() and g.isfinite().all()
    if name != "fp16":  # whose range the others leave
        # a scale's logarithm is up to 2^5 and off by 2^-22 of itself; the exponent it
        # enters is up to 2^6 and rounded to 2^-18: 2^-16 of a weight in all
        off = (got.double() - want).abs()
        assert not (off > tol + 2.0**-16 * want.abs().amax(-1, keepdim=True)).any()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("new", [1, 6, 1300])
@pytest.mark.parametrize("ratio", [-24, -34, -44, -70])
def test_small_scales_with_all_the_weight(cuda_ok, ratio, new, name):
    """Pages whose value scales are 2^ratio of the largest in sight, and which the
    attention goes to all the same: what counts is weight times scale."""
    dim, kv = 64, 1
    kc, ks, vc, vs = filled(12, kv, 16, dim, seed=6, spread=0.1)
    small = torch.arange(12) % 2 == 0
    vs[small] *= 2.0**ratio
    # scores of the small pages: q.k = 16 x 8 x 127 x ks; of the others 0
    kc[:, :, :, :16], ks[:] = 127, 0.02
    kc[:, :, :, 16:] = 0
    ks[~small] = 0
    scale = 1.0
    # e^(-gap) x 2^-ratio is below 2^-24 of the small pages' own sum
    gap = (30 - ratio) * 0.6931
    q = torch.zeros(1, new, 4, dim)
    q[..., :16] = gap / (16 * 127 * 0.02)
    q = q.to(TYPES[name])
    parts, table, lengths = (kc, ks, vc, vs), [list(range(12))], [192]
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    got = tt.kv_attention(q.cuda(), cache, int32(table), int32(lengths), scale=scale, causal=False).cpu().double()
    s = q[0, 0, 0].double() @ (kc[:, 0].double() * ks[:, 0].double()[:, None, None]).flatten(0, 1).T
    p = torch.softmax(s, 0)
    v = (vc[:, 0].double() * vs[:, 0].double()[:, None, None]).flatten(0, 1)
    want, mass = p @ v, p @ v.abs()
    # test_kv_gpu's terms; the slack of small weights goes by weight times scale
    two = name == "fp32"
    d = (dim / 16 + 20) * 2.0**-23 * float(s.abs().max()) + (2.0**-22 * float(s.abs().max()) if two else 0)
    loss = ((2.0**-22 if two else 2.0**-11) + 2 * d + 2.0**-20 + (192 / 16 + 64) * 2.0**-22 + 2.0**-16) * mass
    loss = loss + 192 * 2.0**-28 * float((p[:, None] * v.abs()).max())
    tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 1.01 * loss + torch.finfo(q.dtype).tiny
    assert not ((got[0] - want).abs() > tol).any(), ((got[0] - want).abs() / tol).max()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("new,causal", [(1, True), (20, True), (1300, True), (7, False), (1300, False)])
def test_pages_outside_are_left_out(cuda_ok, new, causal, name):
    """Tokens of a page that the cache does not have are not there: no weight, wherever
    they stand, and a row that has no others is zero."""
    pages, page, kv, dim = 12, 16, 2, 64
    parts = filled(pages, kv, page, dim, seed=8)
    parts[0].abs_()  # all scores are well below 0: a token of score 0 would have all the weight
    q = -torch.rand(3, new, 8, dim, generator=torch.Generator().manual_seed(new)).to(TYPES[name]) - 0.5
    wrong = {1: pages, 4: -1, 5: 2**31 - 1, 9: -2**31}
    table = [[wrong.get(i, i) for i in range(12)], [wrong.get(i, i) for i in range(12)], [-1] * 12]
    lengths = [12 * page - 3, 5 * page, 40]
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    got = tt.kv_attention(q.cuda(), cache, int32(table), int32(lengths), causal=causal)
    with pytest.raises(ValueError, match="page id"):
        cache.check()
    # the definition over the tokens that are there: rows by the last of those that they see
    there = [[t for t in range(n) if 0 <= table[b][t // page] < pages] for b, n in enumerate(lengths)]
    ids = [i for i in range(12) if i not in wrong]
    for b in range(3):
        first = lengths[b] - new
        by_seen = {}
        for i in range(new):
            by_seen.setdefault(sum(t <= first + i for t in there[b]) if causal else len(there[b]), []).append(i)
        for seen, rows in by_seen.items():
            if seen == 0:
                assert not got[b, rows].any()
                continue
            # sequence b's own tokens stand side by side in the pages `ids`
            want, loss = reference(q[b:b + 1, rows], parts, [ids], [seen], [len(rows)], False, dim**-0.5)
            tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 1.01 * loss + torch.finfo(q.dtype).tiny
            off = (got[b:b + 1, rows].cpu().double() - want).abs()
            assert not (off > tol).any() and not off.isnan().any(), (b, seen, (off / tol).max())


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("dim,page,heads,kv,new,lengths", [
    (64, 16, 12, 12, 1, [1, 16, 65, 300, 3]), (128, 64, 8, 1, 1, [1000, 64, 9]), (192, 32, 4, 2, 1, [300, 5]),
    (256, 32, 4, 2, 3, [200, 64]), (80, 32, 6, 2, 5, [40, 5, 130])])
def test_few_rows_closely(cuda_ok, dim, page, heads, kv, new, lengths, name):
    """Few rows have their weights held up by 2^14: what is lost of small ones is half of
    2^-24 of that, 2^-39 of the largest."""
    got, want = attend_case(name, len(lengths), new, heads, kv, dim, page, lengths, seed=2)
    g = torch.Generator().manual_seed(2 + dim + page)  # attend_case's inputs
    pages = len(lengths) * max(1, -(-max(lengths) // page))
    parts = filled(pages, kv, page, dim, 2)
    table = torch.randperm(pages, generator=g).view(len(lengths), -1).tolist()
    q = (torch.randn(len(lengths), new, heads, dim, generator=g) * 2.0).to(TYPES[name])
    kk, vv = parts[0].double() * parts[1].double()[..., None, None], parts[2].double() * parts[3].double()[..., None, None]
    two = name == "fp32"
    for b, n in enumerate(lengths):
        k, v = (x[table[b]].transpose(0, 1).flatten(1, 2) for x in (kk, vv))
        for i in range(new):
            see = n - new + i + 1
            for h in range(heads if see > 0 else 0):
                kh, vh, x = k[h // (heads // kv), :see], v[h // (heads // kv), :see], q[b, i, h].double()
                p = torch.softmax(kh @ x * dim**-0.5, 0)
                d = (dim / 16 + 20) * 2.0**-23 * float((kh.abs() @ x.abs()).max()) * dim**-0.5
                if two:
                    d += 2.0**-22 * float(x.abs().max() * kh.abs().sum(1).max()) * dim**-0.5
                e = (2.0**-22 if two else 2.0**-11) + 2 * d + 2.0**-20 + (n / 16 + 64) * 2.0**-22
                tol = (torch.finfo(q.dtype).eps / 2 * want[b, i, h].abs() + 1.01 * e * (p @ vh.abs())
                       + n * 2.0**-38 * float(p.max() * vh.abs().max()))
                assert ((got[b, i, h].cpu().double() - want[b, i, h]).abs() <= tol).all()


@pytest.mark.parametrize("top", [1, 63, 64, 100, 190, 191, 500, 127 * 127])
def test_append_of_subnormals(cuda_ok, top):
    """Values of a few times 2^-149: the page's scale is so coarse that a value can be more
    than 127 of it, and codes stop at 127."""
    step = 2.0**-149
    cache = tt.KVCache8(2, 1, 32, page_size=16)
    ref = Ref(cache)
    at = 0
    for factor in (1, 2, 1):
        x = torch.linspace(-top * factor, top * factor, 5 * 32).round().view(1, 5, 1, 32).double().mul(step).float()
        assert float(x.abs().max()) > 0
        tt.kv_append(cache, x.cuda(), -x.cuda(), int32([[1]]), int32([at]))
        ref.append(x.numpy(), 0, [[1]], [at], [5])
        ref.append(-x.numpy(), 1, [[1]], [at], [5])
        ref.same(cache)
        at += 5
    assert min(c.min().item() for c in cache.codes()) >= -127
    cache.check()


def test_sequences_that_add_nothing_share_pages(cuda_ok):
    """A sequence without new tokens writes nothing: the page of its last token may be
    another's to write."""
    k = torch.randn(3, 4, 1, 16, device="cuda")
    for counts, wrong in (([4, 0, 0], False), ([4, 0, 4], True), ([0, 0, 0], False), ([4, -1, 0], False)):
        cache = tt.KVCache8(4, 1, 16, page_size=16)
        tt.kv_append(cache, k, k, int32([[2, 0], [2, 1], [2, 3]]), int32([5, 5, 5]), n_new=int32(counts))
        code = int(cache.status.item())
        assert bool(code & 4) == wrong and bool(code & 2) == (min(counts) < 0), (counts, code)


@pytest.mark.parametrize("batch,new,page", [(3, 40, 16), (64, 600, 16), (5, 12000, 16), (2, 8191, 128)])
def test_shared_pages_are_found(cuda_ok, batch, new, page):
    """One page twice among few and among thousands, anywhere; and none where there is none."""
    cols = -(-(new + 7) // page)
    pages = batch * cols + 5
    k = torch.zeros(batch, new, 1, 16, device="cuda", dtype=torch.bfloat16)
    cache = tt.KVCache8(pages, 1, 16, page_size=page)
    good = torch.randperm(pages, generator=torch.Generator().manual_seed(batch))[:batch * cols].view(batch, cols).int()
    start = int32([7 * (b % 2) for b in range(batch)])
    tt.kv_append(cache, k, k, good.cuda(), start)
    cache.check()
    last = (new - 1) // page
    for (b, c), (o, d) in (((0, 0), (batch - 1, last)), ((1, last), (1, 0)), ((0, last // 2), (1, last // 2))):
        table = good.clone()
        table[b, c] = table[o, d]
        tt.kv_append(cache, k, k, table.cuda(), start)
        with pytest.raises(ValueError, match="two places"):
            cache.check()
    # a page that stands twice behind what is written, and ids that are not there, are no sharing
    table = torch.cat((good, good[:1, :1].expand(batch, 2)), 1)
    tt.kv_append(cache, k, k, table.cuda(), start)
    cache.check()
    table = good.clone()
    table[:2, 0] = pages
    tt.kv_append(cache, k, k, table.cuda(), start)
    with pytest.raises(ValueError, match="page id") as wrong:
        cache.check()
    assert "two places" not in str(wrong.value)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("page,dim,half", [(32, 128, 64), (64, 192, 96), (128, 256, 128), (128, 256, 100),
                                           (64, 192, 33), (128, 80, 18), (16, 256, 128)])
def test_rotation_in_every_page(cuda_ok, page, dim, half, aligned, interleaved, name):
    """Rotation beyond a page's first sixteen tokens and a head's first 128 values, with
    tokens that cannot be read sixteen bytes at a time."""
    g = torch.Generator().manual_seed(dim + page)
    new, start, kv = 2 * page + 21, [page - 3, 5], 2
    freq = (10000.0 ** (-torch.arange(half) / half)).float()
    wide = torch.randn(2, new, kv, dim + 1, generator=g).to(TYPES[name]).cuda()
    k = wide[..., 1:]
    if aligned:
        k = k.contiguous()
    v = -k
    cols = (page + new) // page + 1
    cache = tt.KVCache8(2 * cols, kv, dim, page_size=page)
    table = torch.randperm(2 * cols, generator=g).view(2, cols)
    lengths = int32(start)
    tt.kv_append(cache, k, v if aligned else (-wide)[..., 1:], table.int().cuda(), lengths, inv_freq=freq.cuda(),
                 interleaved=interleaved)
    cache.check()
    pos = torch.tensor(start)[:, None] + torch.arange(new)
    x = k.cpu().double()
    want = turned(x, pos.double(), freq, interleaved)
    got = tt.kv_rotate(k, lengths, freq.cuda(), interleaved=interleaved).cpu().double()
    # the angle to 2^-23 turns of a half circle, the sine and the sum to a few units, a rounding
    eps = 2.0**-20 * x.abs().max()
    assert ((got - want).abs() <= eps + torch.finfo(TYPES[name]).eps / 2 * want.abs()).all()
    keys, values = (y.cpu().double() for y in cache.dequantize())
    ks, vs = cache.k_scales.cpu().double(), cache.v_scales.cpu().double()
    for b in range(2):
        home, slot = table[b][pos[b] // page], pos[b] % page
        off = (keys[home, :, slot] - want[b]).abs()
        assert (off <= 0.5001 * ks[home][..., None] + 2 * eps).all()
        # a page's scale is its largest value / 127
        for p in home.unique():
            top = want[b][home == p].abs().amax((0, 2))
            assert ((ks[p] * 127 - top).abs() <= 2 * eps).all()
        off = (values[home, :, slot] + x[b]).abs()
        assert (off <= 0.5001 * vs[home][..., None]).all()


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


def test_shared_pages_of_a_large_cache(cuda_ok):
    """More page ids than one search has bits for."""
    pages, batch, new = 600_000, 2, 4096
    cols = new // 16
    cache = tt.KVCache8(pages, 1, 16, page_size=16)
    k = torch.zeros(batch, new, 1, 16, device="cuda", dtype=torch.bfloat16)
    good = torch.arange(batch * cols).mul(1171).view(batch, cols).int()  # 0 .. 598381, all parts
    assert int(good.max()) < pages
    tt.kv_append(cache, k, k, good.cuda(), int32([0, 0]))
    cache.check()
    for a, b in ((0, batch * cols - 1), (100, 101), (batch * cols - 1, batch * cols - 2), (230, 5)):
        table = good.flatten().clone()
        table[a] = table[b]
        tt.kv_append(cache, k, k, table.view(batch, cols).cuda(), int32([0, 0]))
        with pytest.raises(ValueError, match="two places"):
            cache.check()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("new", [1, 6, 1300])
def test_a_copy_that_never_arrived_is_not_a_result(cuda_ok, new, name):
    """With the timeout noted, what sees a token is NaN until the word has been read; other
    notes leave results alone."""
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in filled(24, 2, 16, 64)))
    table, lengths = int32([list(range(12)), list(range(12, 24))]), int32([180, 0])
    q = torch.randn(2, new, 8, 64, device="cuda").to(TYPES[name])
    want = tt.kv_attention(q, cache, table, lengths)
    sees = max(0, new - 180)  # the first row that sees a token
    cache.status.fill_(8)
    for _ in range(2):
        got = tt.kv_attention(q, cache, table, lengths)
        assert got[0, sees:].isnan().all() and not got[0, :sees].any() and not got[1].any()
    with pytest.raises(_lib.DeviceError, match="never arrived"):
        cache.check()
    assert torch.equal(tt.kv_attention(q, cache, table, lengths), want)
    cache.status.fill_(7)
    assert torch.equal(tt.kv_attention(q, cache, table, lengths), want)
    with pytest.raises(ValueError, match="page id.*length.*two places"):
        cache.check()


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,batch", [(1, 1200), (12, 1190)])
def test_long_runs_of_one_warp(cuda_ok, heads, batch, name):
    """So many long sequences that a warp has whole ones, of values of one sign. Tensor cores
    cut off up to 2^-23 of a sum at every 16 tokens: 1024 times in a run of 256 blocks, where
    262144 tokens in one would lose 1.6e-3. Then there are roundings, half of 2^-23 for each of
    the 16 runs, and for each of the 4096 blocks in the sum of the weights. The weights' own
    roundings (2^-11, of N weights of about 1 / N and of either sign) come to 6 of their standard
    deviations; scores are below 1 and good to 2^-19."""
    pages, dim, page = 2048, 16, 128
    g = torch.Generator().manual_seed(1)
    kc = torch.randint(-127, 128, (pages, 1, page, dim), generator=g, dtype=torch.int8)
    vc = torch.randint(64, 128, (pages, 1, page, dim), generator=g, dtype=torch.int8)
    ks, vs = torch.full((pages, 1), 1 / 500), (1 + 0.2 * torch.rand(pages, 1, generator=g)) / 128
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    q = (torch.randn(1, 1, heads, dim, generator=g) * 0.3).to(TYPES[name])
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, -1)
    n = pages * page
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    lengths[1::2] -= 1001
    got = tt.kv_attention(q.cuda().expand(batch, -1, -1, -1), cache, table, lengths)[:, 0].double().cpu()
    k = (kc.double() * ks.double()[..., None, None]).reshape(-1, dim)
    v = (vc.double() * vs.double()[..., None, None]).reshape(-1, dim)
    bound = (torch.finfo(TYPES[name]).eps / 2 + 1024 * 2.0**-23 + (16 + 4096) * 2.0**-24
             + 6 * 2.0**-11 / (n / 2) ** 0.5 + 2 * 2.0**-19)
    for b in (0, 1):
        end = n - 1001 * b
        want = torch.softmax(q[0, 0].double() @ k[:end].T * dim**-0.5, -1) @ v[:end]
        worst = ((got[b::2] - want).abs() / want).max().item()
        assert worst <= bound, (worst, bound)


@pytest.mark.parametrize("name,most", [("fp16", 2**15), ("bf16", 2**18)])
def test_prompts_in_a_wide_table(cuda_ok, name, most):
    """Many rows of sequences on both sides of the length up to which the tensor cores keep a
    row's sum: each as the definition has it, the short ones as with a narrow table."""
    page, kv, dim, new, heads = 128, 2, 64, 900, 8
    pages = most // page + 3
    parts = filled(pages, kv, page, dim, seed=5)
    cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(pages, generator=g)[None].repeat(4, 1)
    lengths = [most + 300, most, 1000, 0]
    q = torch.randn(4, new, heads, dim, generator=g).to(TYPES[name])
    got = tt.kv_attention(q.cuda(), cache, table.int().cuda(), int32(lengths))
    cache.check()
    assert not got[3].any() and got.isfinite().all()
    narrow = tt.kv_attention(q[1:3].cuda(), cache, table[1:3, :most // page].int().cuda().contiguous(), int32(lengths[1:3]))
    assert torch.equal(got[1:3], narrow)
    ks, vs = (parts[i].double() * parts[i + 1].double()[..., None, None] for i in (0, 2))
    for b in range(3):
        n = lengths[b]
        k, v = (x[table[b]].transpose(0, 1).flatten(1, 2)[:, :n].cuda() for x in (ks, vs))
        for i in (0, 1, 450, 899):
            see = n - new + i + 1
            for h in (0, 3, 4, 7):
                kh, vh, x = k[h // 4, :see], v[h // 4, :see], q[b, i, h].double().cuda()
                p = torch.softmax(kh @ x * dim**-0.5, 0)
                want = p @ vh
                d = (dim / 16 + 20) * 2.0**-23 * float((kh.abs() @ x.abs()).max()) * dim**-0.5
                e = 2.0**-11 + 2 * d + 2.0**-20 + (n / 16 + 64) * 2.0**-23
                tol = (torch.finfo(q.dtype).eps / 2 * want.abs() + 1.01 * e * (p @ vh.abs())
                       + n * 2.0**-28 * float(p.max() * vh.abs().max()))
                assert ((got[b, i, h].double() - want).abs() <= tol).all(), (b, i, h)


@pytest.mark.parametrize("name,bits", [("fp16", 11), ("bf16", 8)])
def test_prompts_over_long_runs(cuda_ok, name, bits):
    """Values of one sign over more tokens than a tile's sums may stay in the tensor cores for.
    The bound is test_long_runs_of_one_warp's."""
    page, dim, new = 128, 16, 1000
    n = 2**19 if name == "bf16" else 2**17
    pages = n // page
    g = torch.Generator().manual_seed(1)
    kc = torch.randint(-127, 128, (pages, 1, page, dim), generator=g, dtype=torch.int8)
    vc = torch.randint(64, 128, (pages, 1, page, dim), generator=g, dtype=torch.int8)
    ks, vs = torch.full((pages, 1), 1 / 500), (1 + 0.2 * torch.rand(pages, 1, generator=g)) / 128
    cache = tt.KVCache8.from_codes(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda())
    q = (torch.randn(1, 1, 12, dim, generator=g) * 0.3).to(TYPES[name])
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    got = tt.kv_attention(q.cuda().expand(1, new, -1, -1), cache, table, int32([n]), causal=False)[0].double().cpu()
    k = (kc.double() * ks.double()[..., None, None]).reshape(-1, dim)
    v = (vc.double() * vs.double()[..., None, None]).reshape(-1, dim)
    want = torch.softmax(q[0, 0].double() @ k.T * dim**-0.5, -1) @ v
    bound = (2.0**-bits + 1024 * 2.0**-23 + n / 64 * 2.0**-24 + 6 * 2.0**-11 / (n / 2) ** 0.5 + 2 * 2.0**-19)
    worst = ((got - want).abs() / want).max().item()
    assert worst <= bound, (worst, bound)


@pytest.mark.parametrize("name", ["fp32", "bf16"])
@pytest.mark.parametrize("new", [1, 6, 1300])
@pytest.mark.parametrize("size", [2.0**81, 2.0**100, 2.0**120])
def test_huge_scales(cuda_ok, size, new, name):
    """Values near the end of fp32's range, in all pages or in one of them. (Scales in a row's
    sight may be 2^100 apart: a weight is 2^14 times 2^-100 then, and as many scores' bits below
    the largest as are left down to fp32's 2^-126. The others here are about 2^-6.)"""
    for mixed in (False, True) if size <= 2.0**100 else (False,):
        kc, ks, vc, vs = filled(12, 2, 16, 64, seed=11)
        vs[3 if mixed else slice(None)] *= size * (1 / 8 if mixed else 15)
        parts = (kc, ks, vc, vs)
        q = torch.randn(1, new, 4, 64, generator=torch.Generator().manual_seed(new)).to(TYPES[name])
        cache = tt.KVCache8.from_codes(*(x.cuda() for x in parts))
        got = tt.kv_attention(q.cuda(), cache, int32([list(range(12))]), int32([190])).cpu().double()
        want, loss = reference(q, parts, [list(range(12))], [190], [new], True, 64**-0.5)
        # a scale's logarithm is up to 2^7 and off by 2^-22 of itself, and the exponent it enters
        # is rounded to 2^-17: 2^-14 of a weight in all
        tol = torch.finfo(q.dtype).eps / 2 * want.abs() + 1.01 * loss + 2.0**-14 * want.abs().amax(-1, keepdim=True)
        assert not ((got - want).abs() > tol).any() and not got.isnan().any()
