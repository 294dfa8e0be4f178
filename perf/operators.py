"""Cases of the contractions whose stored operand is held in 4 or 8 bits.

Four kinds of case, by ``case["op"]``:

* ``product``: y = x W^T with W held as 4-bit codes and a scale for each group of a row;
* ``train``: the same product and its gradient for x;
* ``append``: new keys and values rotated to their positions, quantised and written into
  a paged 8-bit cache with one scale for each page and head; the written pages are read back;
* ``attend``: softmax attention of queries over such a cache.

``run`` computes the plain form in elementary fp32 torch operations, or calls
trntensor_b200 where ``own`` is true.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token through a square projection: the latency of a decode step's smallest layer
        {"name": "product 1 x 4096 x 4096", "op": "product", "rows": 1, "n": 4096, "k": 4096,
         "group": 128, "dtype": "bf16", "scales": "bf16"},
        # a decode batch through a wide layer
        {"name": "product 32 x 16384 x 8192", "op": "product", "rows": 32, "n": 16384, "k": 8192,
         "group": 128, "dtype": "bf16", "scales": "bf16"},
        # a prompt's tokens through a large square layer
        {"name": "product 2048 x 8192 x 8192", "op": "product", "rows": 2048, "n": 8192, "k": 8192,
         "group": 64, "dtype": "bf16", "scales": "bf16"},
        # odd sizes in 32 bits: a last group that is cut short, rows off every alignment
        {"name": "product 5 x 1001 x 777", "op": "product", "rows": 5, "n": 1001, "k": 777,
         "group": 32, "dtype": "fp32", "scales": "fp32"},
        # a short sequence trained through a frozen 4-bit layer (adapters beside it)
        {"name": "train 7 x 4096 x 11000", "op": "train", "rows": 7, "n": 4096, "k": 11000,
         "group": 128, "dtype": "bf16", "scales": "bf16"},
        # a training batch through the same kind of layer
        {"name": "train 2000 x 8192 x 4096", "op": "train", "rows": 2000, "n": 8192, "k": 4096,
         "group": 128, "dtype": "fp16", "scales": "bf16"},
        # every sequence of a decode batch adds one token
        {"name": "append 64 x 1", "op": "append", "batch": 64, "new": 1, "have": 4100, "kv_heads": 8,
         "dim": 128, "rot": 128, "interleaved": False, "page": 64, "dtype": "bf16"},
        # two long prompts enter the cache
        {"name": "append 2 x 8191", "op": "append", "batch": 2, "new": 8191, "have": 70, "kv_heads": 8,
         "dim": 128, "rot": 64, "interleaved": True, "page": 16, "dtype": "fp16"},
        # a few short sequences with a head for each query, in 32 bits
        {"name": "attend 3 x 1 over 100", "op": "attend", "batch": 3, "new": 1, "length": 100,
         "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "dtype": "fp32"},
        # a decode batch of ordinary lengths
        {"name": "attend 64 x 1 over 8192", "op": "attend", "batch": 64, "new": 1, "length": 8192,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one user far into a long context
        {"name": "attend 1 x 1 over 131000", "op": "attend", "batch": 1, "new": 1, "length": 131000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a piece of a prompt against what is cached already
        {"name": "attend 2 x 1000 over 8000", "op": "attend", "batch": 2, "new": 1000, "length": 8000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["product", "train", "append", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("product", "train"):
        n, k = _spread(rng, 64, 16384), _spread(rng, 32, 16384)
        rows = _spread(rng, 1, 2048)
        most = 2048 * 8192 * 8192 // (2 if op == "train" else 1)
        rows = max(1, min(rows, most // (n * k)))
        return {"op": op, "rows": rows, "n": n, "k": k, "group": rng.choice([32, 64, 128]),
                "dtype": dtype, "scales": rng.choice(["bf16", "bf16", "fp32"])}
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "append":
        batch = _spread(rng, 1, 64)
        new = _spread(rng, 1, 8191)
        new = max(1, min(new, 2 * 8191 * 8 * 128 // (batch * kv * dim)))
        have = _spread(rng, 1, max(2, min(8192, (1 << 28) // (batch * kv * dim))))
        return {"op": op, "batch": batch, "new": new, "have": have, "kv_heads": kv, "dim": dim,
                "rot": dim // rng.choice([1, 1, 2]) // 4 * 4, "interleaved": rng.random() < 0.5,
                "page": page, "dtype": rng.choice(["bf16", "fp16"])}
    batch = _spread(rng, 1, 64)
    new = 1 if rng.random() < 0.5 else _spread(rng, 2, 1000)
    heads = kv * rng.choice([1, 2, 4, 5, 8])
    length = _spread(rng, 1, 131000)
    length = max(1, min(length, (1 << 29) // (batch * kv * dim)))
    length = max(1, min(length, 2 * 32 * 1000 * 8000 // (batch * heads * new)))
    return {"op": op, "batch": batch, "new": min(new, length), "length": length, "heads": heads,
            "kv_heads": kv, "dim": dim, "page": page, "dtype": dtype}


def _ragged(most, batch):
    """Lengths between a half of `most` and `most`, the first the longest."""
    return [most - most * ((11 * b) % 16) // 32 for b in range(batch)]


def _new_counts(case):
    new = case["new"]
    return [new - new * ((5 * b) % 8) // 16 for b in range(case["batch"])]


def _table(gen, batch, per, dev):
    """Pages in no order: `per` for each sequence."""
    return torch.randperm(batch * per, generator=gen, device=dev).view(batch, per).to(torch.int32)


def _codes(gen, shape, dev):
    c = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16).mul_(40)
    return c.round_().clamp_(-127, 127).to(torch.int8)


def _page_scales(gen, shape, dev):
    return torch.randn(shape, generator=gen, device=dev).mul_(0.3).exp_().div_(40)


def _matrix(case, gen, dev):
    n, k, g = case["n"], case["k"], case["group"]
    codes = torch.randn((n, k), generator=gen, device=dev, dtype=torch.float16).mul_(3)
    codes = codes.round_().clamp_(-8, 7).to(torch.int8)
    groups = -(-k // g)
    scales = torch.randn((n, groups), generator=gen, device=dev).mul_(0.5).exp_().mul_(0.01)
    return codes, scales.to(_TYPES[case["scales"]])


def _rows(gen, rows, cols, dtype, dev):
    """Activations: normal values, with a few columns that are much larger than the rest."""
    x = torch.randn((rows, cols), generator=gen, device=dev)
    x[:, :: max(1, cols // 8)] *= 8
    return x.to(dtype)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("product", "train"):
        codes, scales = _matrix(case, gen, dev)
        s["x"] = _rows(gen, case["rows"], case["k"], dtype, dev)
        if case["op"] == "train":
            s["x"].requires_grad_()
            s["dy"] = _rows(gen, case["rows"], case["n"], dtype, dev)
        if own:
            import trntensor_b200 as tt

            s["weight"] = tt.pack_q4(codes, scales, group=case["group"])
        else:
            s["codes"], s["scales"] = codes, scales
        return s
    batch, kv, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        start, count = _ragged(case["have"], batch), _new_counts(case)
        per = -(-(case["have"] + case["new"]) // page)
    else:
        start, count = _ragged(case["length"], batch), _new_counts(case)
        per = -(-case["length"] // page)
    pages = batch * per
    s["table"] = _table(gen, batch, per, dev)
    s["lengths"] = torch.tensor(start, dtype=torch.int32, device=dev)
    s["count"] = torch.tensor(count, dtype=torch.int32, device=dev)
    # one page at the end stands in no table
    kc, vc = (_codes(gen, (pages + 1, kv, page, dim), dev) for _ in range(2))
    ks, vs = (_page_scales(gen, (pages + 1, kv), dev) for _ in range(2))
    if own:
        import trntensor_b200 as tt

        s["cache"] = tt.KVCache8.from_codes(kc, ks, vc, vs)
    else:
        s["kc"], s["vc"], s["ks"], s["vs"] = kc, vc, ks, vs
    if case["op"] == "append":
        shape = (batch, case["new"], kv, dim)
        s["k"] = torch.randn(shape, generator=gen, device=dev).to(dtype)
        s["v"] = torch.randn(shape, generator=gen, device=dev).to(dtype)
        half = case["rot"] // 2
        s["inv_freq"] = (10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64)
                                     / half)).float()
        host = s["table"].cpu()
        s["pages"] = torch.cat([host[b, start[b] // page: (start[b] + count[b] - 1) // page + 1]
                                for b in range(batch)]).to(dev)
    else:
        q = torch.randn((batch, case["new"], case["heads"], dim), generator=gen, device=dev)
        s["q"] = (q * 3).to(dtype)
    return s


def _weights(s):
    g = s["case"]["group"]
    n, k = s["codes"].shape
    wide = s["scales"].float().repeat_interleave(g, dim=1)[:, :k]
    return s["codes"].float() * wide


def _turn(x, pos, inv_freq, interleaved):
    """x (batch, new, heads, dim) in 32 bits, turned by pos (batch, new) times inv_freq; the
    angles in 64 bits."""
    half = inv_freq.numel()
    a = pos.double()[:, :, None, None] * inv_freq.double()
    cos, sin = a.cos().float(), a.sin().float()
    if interleaved:
        u, w = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((u * cos - w * sin, w * cos + u * sin), dim=-1).flatten(-2)
    else:
        u, w = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((u * cos - w * sin, w * cos + u * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _put(codes, scales, x, s):
    """Quantises x (batch, new, heads, dim; 32 bits) into the pages of `codes`, in place."""
    page = s["case"]["page"]
    pages, heads = scales.shape
    batch, new = x.shape[:2]
    dev = x.device
    start, count = s["lengths"].long(), s["count"].long()
    i = torch.arange(new, device=dev)
    pos = start[:, None] + i
    ok = i < count[:, None]
    cols = s["table"].shape[1]
    home = s["table"].long().gather(1, (pos // page).clamp(max=cols - 1))
    home = torch.where(ok, home, pages - 1)  # the spare page takes what is not to be written
    # what the new tokens need, for each page
    need = torch.zeros((pages, heads), device=dev)
    need.index_reduce_(0, home.flatten(), x.abs().amax(-1).flatten(0, 1) / 127, "amax")
    # the first slot that is written in each page: `page` where none is
    first = torch.full((pages,), page, device=dev, dtype=torch.long)
    first.scatter_reduce_(0, home.flatten(), (pos % page).flatten(), "amin")
    old = torch.where(first[:, None] == 0, torch.zeros_like(scales), scales)
    now = torch.where(first[:, None] < page, torch.maximum(old, need), scales)
    # the earlier tokens of the pages that this call touches
    span = torch.arange(-(-(new - 1) // page) + 1, device=dev) + start[:, None] // page
    there = span * page < (start + count)[:, None]
    touched = s["table"].long().gather(1, span.clamp(max=cols - 1))
    touched = torch.where(there, touched, touched[:, :1]).flatten()
    ratio = torch.where(now > old, old / now, torch.ones_like(now))[touched]
    before = torch.arange(page, device=dev) < first[touched][:, None]
    kept = codes[touched]
    again = (kept.float() * ratio[:, :, None, None]).round().to(torch.int8)
    codes[touched] = torch.where(before[:, None, :, None], again, kept)
    # the new tokens
    scale = now[home][..., None]
    fresh = torch.where(scale > 0, x / scale, torch.zeros_like(x)).round().clamp(-127, 127)
    codes[home, :, pos % page] = fresh.to(torch.int8)
    scales.copy_(now)


def _read(codes, scales, pages, dtype):
    pages = pages.long()
    return (codes[pages].float() * scales[pages][:, :, None, None]).to(dtype)


def _plain_append(s):
    case, dtype = s["case"], _TYPES[s["case"]["dtype"]]
    pos = s["lengths"].long()[:, None] + torch.arange(case["new"], device=s["k"].device)
    _put(s["kc"], s["ks"], _turn(s["k"].float(), pos, s["inv_freq"], case["interleaved"]), s)
    _put(s["vc"], s["vs"], s["v"].float(), s)
    return {"k": _read(s["kc"], s["ks"], s["pages"], dtype),
            "v": _read(s["vc"], s["vs"], s["pages"], dtype)}


def _plain_attend(s):
    case, q, page = s["case"], s["q"], s["case"]["page"]
    batch, new, heads, dim = q.shape
    kv = case["kv_heads"]
    table = s["table"].long()
    length = table.shape[1] * page

    def whole(codes, scales):  # (batch, kv, length, dim)
        x = codes[table].float() * scales[table][..., None, None]
        return x.transpose(1, 2).reshape(batch, kv, length, dim)

    k, v = whole(s["kc"], s["ks"]), whole(s["vc"], s["vs"])
    qg = q.float().view(batch, new, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(qg.reshape(batch, kv, -1, dim), k.transpose(2, 3)) / math.sqrt(dim)
    score = score.view(batch, kv, heads // kv, new, length)
    i = torch.arange(new, device=q.device)
    pos = (s["lengths"] - s["count"]).long()[:, None] + i
    pos = torch.where(i < s["count"][:, None], pos, torch.full_like(pos, -1))
    seen = torch.arange(length, device=q.device) <= pos[:, :, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, kv, -1, length), v).view(batch, kv, heads // kv, new, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(batch, new, heads, dim).to(q.dtype)


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        import trntensor_b200 as tt

        if op == "product":
            return tt.einsum("mk,nk->mn", s["x"], s["weight"])
        if op == "train":
            y = tt.einsum("mk,nk->mn", s["x"], s["weight"])
            return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
        if op == "append":
            tt.kv_append(s["cache"], s["k"], s["v"], s["table"], s["lengths"], n_new=s["count"],
                         inv_freq=s["inv_freq"], interleaved=s["case"]["interleaved"])
            k, v = s["cache"].dequantize(s["pages"], dtype=s["k"].dtype)
            return {"k": k, "v": v}
        return tt.kv_attention(s["q"], s["cache"], s["table"], s["lengths"], n_query=s["count"])
    if op == "append":
        return _plain_append(s)
    if op == "attend":
        return _plain_attend(s)
    w, x = _weights(s), s["x"].detach()
    y = torch.matmul(x.float(), w.t()).to(x.dtype)
    if op == "product":
        return y
    return {"y": y, "dx": torch.matmul(s["dy"].float(), w).to(x.dtype)}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("product", "train"):
        m, n, k = case["rows"], case["n"], case["k"]
        held = n * k // 2 + n * -(-k // case["group"]) * (4 if case["scales"] == "fp32" else 2)
        if case["op"] == "product":
            return {"bytes": held + size * (m * k + m * n), "flops": 2.0 * m * n * k}
        return {"bytes": held + size * 2 * (m * k + m * n), "flops": 4.0 * m * n * k}
    batch, kv, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    count = _new_counts(case)
    if case["op"] == "append":
        start = _ragged(case["have"], batch)
        tokens = sum(count)
        touched = sum((a + c - 1) // page + 1 - a // page for a, c in zip(start, count))
        once = 2 * kv * dim
        return {"bytes": once * (tokens * (size + 1) + touched * page * (1 + size)),
                "flops": 6.0 * once * tokens}
    lengths = _ragged(case["length"], batch)
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lengths, count))
    held = sum(2 * kv * dim * n + 8 * kv * -(-n // page) for n in lengths)
    moved = size * case["heads"] * dim * (sum(count) + batch * case["new"])
    return {"bytes": held + moved, "flops": 4.0 * dim * case["heads"] * pairs}


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _plain_state(case, seed):
    """The inputs of `prepare`, in the plain layout."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _exact_page(x, codes, scale, slot):
    """Tokens x (t, heads, dim) enter a page's codes (heads, page, dim) at `slot`: the page's values."""
    held = torch.zeros_like(scale) if slot == 0 else scale
    new = torch.maximum(held, x.abs().amax(dim=(0, 2)) / 127)
    c = codes.double()
    if slot:
        grown = (new > held)[:, None, None]
        c[:, :slot] = torch.where(grown, torch.round(c[:, :slot] * (held / new)[:, None, None]), c[:, :slot])
    put = torch.round(x / new.clamp(min=1e-300)[None, :, None])
    c[:, slot:slot + x.shape[0]] = put.transpose(0, 1)
    return c * new[:, None, None]


def exact(case, seed):
    s = _plain_state(case, seed)
    if case["op"] in ("product", "train"):
        n, k, g = case["n"], case["k"], case["group"]
        w = torch.empty((n, k), dtype=torch.float64, device=s["codes"].device)
        for j in range(0, k, g):
            w[:, j:j + g] = s["codes"][:, j:j + g].double() * s["scales"][:, j // g].double()[:, None]
        y = torch.einsum("mk,nk->mn", s["x"].detach().double(), w)
        return y if case["op"] == "product" else {
            "y": y, "dx": torch.einsum("mn,nk->mk", s["dy"].double(), w)}
    page = case["page"]
    starts, counts = s["lengths"].tolist(), s["count"].tolist()
    table = s["table"].tolist()
    if case["op"] == "append":
        half = s["inv_freq"].numel()
        ks, vs = [], []
        for b, (a, c) in enumerate(zip(starts, counts)):
            t = torch.arange(a, a + c, device=s["k"].device, dtype=torch.float64)
            angle = torch.outer(t, s["inv_freq"].double())[:, None, :]
            pairs = torch.arange(half, device=s["k"].device)
            one = 2 * pairs if case["interleaved"] else pairs
            two = one + 1 if case["interleaved"] else one + half
            k, v = s["k"][b, :c].double(), s["v"][b, :c].double()
            turned = k.clone()
            turned[..., one] = k[..., one] * torch.cos(angle) - k[..., two] * torch.sin(angle)
            turned[..., two] = k[..., one] * torch.sin(angle) + k[..., two] * torch.cos(angle)
            at = a
            while at < a + c:
                end = min(a + c, (at // page + 1) * page)
                home = table[b][at // page]
                ks.append(_exact_page(turned[at - a:end - a], s["kc"][home], s["ks"][home].double(), at % page))
                vs.append(_exact_page(v[at - a:end - a], s["vc"][home], s["vs"][home].double(), at % page))
                at = end
        return {"k": torch.stack(ks), "v": torch.stack(vs)}
    q = s["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    rep = case["heads"] // case["kv_heads"]
    for b, (n, c) in enumerate(zip(starts, counts)):
        held = s["table"][b, :-(-n // page)].long()
        k = (s["kc"][held].double() * s["ks"][held].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
        v = (s["vc"][held].double() * s["vs"][held].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
        ahead = torch.ones((c, n), dtype=torch.bool, device=q.device).triu(n - c + 1)
        for h in range(case["kv_heads"]):
            z = torch.einsum("chd,td->hct", q[b, :c, h * rep:(h + 1) * rep].double(), k[h]) * case["dim"] ** -0.5
            p = torch.softmax(z.masked_fill(ahead, -math.inf), dim=-1)
            out[b, :c, h * rep:(h + 1) * rep] = torch.einsum("hct,td->chd", p, v[h])
    return out
