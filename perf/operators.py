"""The serving operators and what they are compared with.

Five operators of one decode step: the residual's addition with the RMS norm and its e4m3 output (``norm``),
the e4m3 paged key/value cache's append (``append``) and attention (``attention``), the selection of a beam
search (``beam``) and the reordering of its states (``reorder``).  With ``own`` false, ``run`` computes them in
elementary torch operations; with ``own`` true it calls ``tilelang.ops``.

Shapes: 7168-wide rows, 129280 tokens and the 512 + 64 + 128 wide caches are the DeepSeek-V3.2 configuration's,
3200-wide rows, 32 heads of 100 and 32002 tokens BitNet 3B's, 32 query heads on 8 key/value heads of 128 and
8192 cached tokens the decode examples'.
"""
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
EOS = 2


# ------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # one token's row in front of the fp8 projections: latency
        dict(name="norm one token", op="norm", rows=1, width=7168, type="bf16", group=128, pow2=False, residual=True,
             norm=True),
        # a prefill chunk: bandwidth
        dict(name="norm prefill", op="norm", rows=8192, width=7168, type="bf16", group=128, pow2=False, residual=True,
             norm=False),
        # one new token for each of a decode batch's sequences: latency
        dict(name="append one token", op="append", batch=32, new=1, past=1000, kv_heads=8, dim=128, page=64,
             type="bf16"),
        # prompts of uneven ends written into the cache: bandwidth
        dict(name="append prompts", op="append", batch=8, new=4001, past=37, kv_heads=8, dim=128, page=64,
             type="bf16"),
        # one user, a short context: latency
        dict(name="attention one user", op="attention", batch=1, new=1, longest=777, heads=32, kv_heads=8, dim=128,
             page=64, type="bf16"),
        # the decode examples' heads and context, ragged: the cache's bytes
        dict(name="attention batch", op="attention", batch=32, new=1, longest=8192, heads=32, kv_heads=8, dim=128,
             page=64, type="bf16"),
        # BitNet 3B's heads at its longest context: every head its own keys, 100 wide
        dict(name="attention 100 wide", op="attention", batch=16, new=1, longest=2048, heads=32, kv_heads=32, dim=100,
             page=16, type="fp16"),
        # a chunk of a long prompt against the cache: the matrix cores
        dict(name="attention chunk", op="attention", batch=2, new=509, longest=4096, heads=32, kv_heads=8, dim=128,
             page=64, type="bf16"),
        # one user's beams over BitNet's vocabulary: latency
        dict(name="beam one user", op="beam", batch=1, beams=4, vocab=32002, take=8, type="fp16"),
        # a batch of beams over 129280 tokens: bandwidth
        dict(name="beam batch", op="beam", batch=8, beams=8, vocab=129280, take=16, type="fp32"),
        # the states of a small model
        dict(name="reorder small", op="reorder", batch=1, beams=4, layers=2, slots=256, used=97, latent=128, rope=32,
             index=128),
        # long latent and indexer caches of several layers
        dict(name="reorder long", op="reorder", batch=8, beams=8, layers=4, slots=4096, used=3001, latent=512,
             rope=64, index=128),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attention", "attention", "beam", "reorder"])
    if op == "norm":
        group = rng.choice([0, 64, 128, 128, 256])
        width = _log(rng, 65, 8192) if group == 0 else group * _log(rng, 2, 8192 // group)
        rows = _log(rng, 1, min(16384, 8192 * 7168 // width))
        # a power-of-two scale turns the last bit of a sum into a factor of two where a maximum meets a border:
        # few enough groups that none does
        pow2 = rng.random() < 0.5 and group > 0 and rows * (width // group) <= 20000
        return dict(op=op, rows=rows, width=width, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), group=group,
                    pow2=pow2, residual=rng.random() < 0.7, norm=rng.random() < 0.5)
    kv_heads, dim = rng.choice([1, 2, 4, 8, 32]), rng.choice([64, 80, 100, 128, 128, 192, 256])
    page, kind = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "fp16"])
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, 4096)])
        batch = max(1, min(_log(rng, 1, 64), 32 * 1024 * 1024 // (new * kv_heads * dim)))
        return dict(op=op, batch=batch, new=new, past=rng.randrange(0, 600), kv_heads=kv_heads, dim=dim, page=page,
                    type=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "attention":
        heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8, 16])
        new = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 512)])
        longest = max(new, _log(rng, 16, 16384))
        new = min(new, max(1, 60_000_000 // (heads * longest)))  # a chunk's products
        most = 250_000_000 // (longest * kv_heads * dim * (1 + new // 8))
        batch = max(1, min(_log(rng, 1, 64), most, 60_000_000 // (heads * new * longest)))
        return dict(op=op, batch=batch, new=new, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    type=kind)
    if op == "beam":
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 16]), _log(rng, 500, 150_000)
        batch = max(1, min(_log(rng, 1, 32), 8_000_000 // (beams * vocab)))
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, take=rng.choice([beams, 2 * beams]),
                    type=rng.choice(["bf16", "fp16", "fp32"]))
    slots = _log(rng, 64, 4096)
    beams = rng.choice([2, 3, 4, 5, 8, 16])
    latent, rope, index = rng.choice([128, 512]), rng.choice([32, 64]), rng.choice([64, 128])
    batch, layers = _log(rng, 1, 8), rng.choice([1, 2, 4])
    layers = max(1, min(layers, 900_000_000 // (batch * beams * slots * (2 * latent + 2 * rope + index + 4))))
    return dict(op=op, batch=batch, beams=beams, layers=layers, slots=slots, used=rng.randrange(1, slots + 1),
                latent=latent, rope=rope, index=index)


def _lengths(case):
    """The cached tokens of each sequence, the new ones among them: known from the case alone."""
    b, new = case["batch"], case["new"]
    if case["op"] == "append":  # every sequence ends at another place in its page
        return [new + max(0, case["past"] - 13 * i) for i in range(b)]
    low = max(new, case["longest"] // 2)  # between half the longest and it
    return [case["longest"] - (case["longest"] - low) * i // max(1, b) for i in range(b)]


def work(case):
    op = case["op"]
    if op == "norm":
        n, e = case["rows"] * case["width"], SIZE[case["type"]]
        groups = case["rows"] * (case["width"] // case["group"] if case["group"] else 1)
        per = e + 1 + (2 * e if case["residual"] else 0) + (e if case["norm"] else 0)
        return {"bytes": n * per + 4 * groups + e * case["width"], "flops": 8 * n}
    if op == "append":
        n = 2 * case["batch"] * case["new"] * case["kv_heads"] * case["dim"]
        pages = sum((t - 1) // case["page"] - max(0, t - case["new"]) // case["page"] + 1 for t in _lengths(case))
        return {"bytes": n * (SIZE[case["type"]] + 1) + 2 * 4 * pages * case["kv_heads"], "flops": 3 * n}
    if op == "attention":
        lens, d, new = _lengths(case), case["dim"], case["new"]
        keys = sum(lens) * case["kv_heads"]
        rows = case["batch"] * new * case["heads"]
        seen = case["heads"] * sum(new * t - new * (new - 1) // 2 for t in lens)
        return {"bytes": 2 * d * keys + 8 * keys // case["page"] + 2 * rows * d * SIZE[case["type"]] + 4 * rows,
                "flops": 4 * d * seen}
    if op == "beam":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * SIZE[case["type"]] + 20 * case["batch"] * case["take"], "flops": 3 * n}
    k, rows = case["beams"], case["batch"]
    row = case["layers"] * case["used"] * (2 * case["latent"] + 2 * case["rope"] + case["index"] + 4)
    moved, read = k - 1, (k - 1) * (1 - (1 - 1 / k) ** k)  # parents drawn evenly: one of k stays on average
    return {"bytes": row * rows * (moved + read), "flops": 0}


# ------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cache(g, pages, kv_heads, dim, page):
    """A pool in use: every slot holds codes, a scale for each page and head; one spare page at the end."""
    wide = -(-dim // 64) * 64
    out = []
    for tokens_last in (False, True):
        size = 0.5 + 2 * torch.rand(kv_heads, 1, 1, generator=g, device="cuda")
        x = _randn(g, pages + 1, kv_heads, page, wide) * size
        x[..., dim:] = 0
        scale = _pow2_scale(x.abs().amax(dim=(2, 3)))
        codes = (x / scale[:, :, None, None]).to(FP8)
        out += [codes.view(torch.uint8).transpose(2, 3).contiguous().view(FP8) if tokens_last else codes, scale]
    return dict(k=out[0], k_scale=out[1], v=out[2], v_scale=out[3])


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "norm":
        t = TYPES[case["type"]]
        x = _randn(g, case["rows"], case["width"]).mul_(0.5).to(t)
        residual = _randn(g, case["rows"], case["width"]).mul_(2).to(t) if case["residual"] else None
        weight = (1 + 0.2 * _randn(g, case["width"])).to(t)
        return dict(case=case, x=x, residual=residual, weight=weight)
    if op in ("append", "attention"):
        lens, b, new = _lengths(case), case["batch"], case["new"]
        page, d = case["page"], case["dim"]
        per = -(-max(lens) // page)
        pages = sum(-(-t // page) for t in lens)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).tolist()
        table, at = [], 0
        for t in lens:  # each sequence has the pages that it needs, in no order
            n = -(-t // page)
            table.append(order[at:at + n] + [0] * (per - n))
            at += n
        state = dict(case=case, table=torch.tensor(table, dtype=torch.int32, device="cuda"),
                     lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"), pages=pages,
                     **_cache(g, pages, case["kv_heads"], d, page))
        t = TYPES[case["type"]]
        if op == "append":
            state["new_k"] = (_randn(g, b, new, case["kv_heads"], d) * 2).to(t)
            state["new_v"] = _randn(g, b, new, case["kv_heads"], d).to(t)
        else:
            state["q"] = (_randn(g, b, new, case["heads"], d) * 1.5).to(t)
        return state
    b, k = case["batch"], case["beams"]
    if op == "beam":
        logits = torch.empty(b * k, case["vocab"], dtype=TYPES[case["type"]], device="cuda")
        for i in range(b * k):
            logits[i] = _randn(g, case["vocab"]) * 3
        scores = -5 * _randn(g, b, k).abs()
        finished = torch.rand(b, k, generator=g, device="cuda") < 0.15
        return dict(case=case, logits=logits.view(b, k, case["vocab"]), scores=scores, finished=finished)
    states = []
    for _ in range(case["layers"]):
        for width, t in ((case["latent"], torch.bfloat16), (case["rope"], torch.bfloat16), (case["index"], FP8)):
            x = torch.randint(0, 256, (b * k, case["slots"], width * (1 if t is FP8 else 2)), generator=g,
                              device="cuda", dtype=torch.uint8)
            if t is FP8:
                x.bitwise_and_(0xF7)  # no not-a-number among the codes
            else:
                x[..., 1::2].bitwise_and_(0xBF)
            states.append(x.view(t))
        states.append(_randn(g, b * k, case["slots"]))
    parents = torch.randint(0, k, (b, k), generator=g, device="cuda")
    return dict(case=case, states=states, parents=parents)


# ------------------------------------------------------------------------------------------- plain forms


def _pow2_scale(amax):
    """The smallest power of two that is no smaller than amax / 448, and at least 2^-22."""
    m, e = torch.frexp(amax.float() / 448)
    return torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)).clamp_min(2.0 ** -22)


def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    g = y.view(y.shape[0], -1, case["group"] or y.shape[1])
    amax = g.abs().amax(-1).clamp_min(1e-4)
    if case["pow2"]:
        m, e = torch.frexp(amax / 448)
        scale = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e))
    else:
        scale = amax / 448
    q = (g / scale[..., None]).clamp(-448, 448).to(FP8).view(y.shape)
    return dict(q=q, scale=scale, h=h.to(t) if s["residual"] is not None else None,
                y=y.to(t) if case["norm"] else None)


def _touched(s):
    """For every page that new tokens may reach: its id, and for its slots the new token there and who is old."""
    page, new = s["case"]["page"], s["case"]["new"]
    lens = s["lengths"].long()
    past = lens - new
    nth = past[:, None] // page + torch.arange((new - 1) // page + 2, device="cuda")
    at = nth[..., None] * page + torch.arange(page, device="cuda")  # the slots' positions
    is_new = (at >= past[:, None, None]) & (at < lens[:, None, None])
    ids = s["table"].long().gather(1, nth.clamp_max(s["table"].shape[1] - 1))
    ids = torch.where(is_new.any(-1), ids, s["pages"])  # the spare page takes what nobody wants
    return ids, (at - past[:, None, None]).clamp(0, new - 1), is_new, at < past[:, None, None]


def _plain_append(s):
    dim = s["case"]["dim"]
    ids, token, is_new, is_old = _touched(s)
    which = torch.arange(ids.shape[0], device="cuda")[:, None, None]

    def one(pool, scales, x, tokens_last):
        new = x.float()[which, token].transpose(2, 3)  # [batch, page, head, slot, dim]
        new = torch.where(is_new[:, :, None, :, None], new, 0.0)
        fresh = is_new[:, :, :1]
        before = torch.where(fresh, 0.0, scales[ids])
        after = torch.maximum(before, _pow2_scale(new.abs().amax(dim=(3, 4))))
        codes = pool.view(torch.uint8)[ids].view(FP8)
        codes = codes.transpose(3, 4) if tokens_last else codes
        old = (codes.float() * (before / after)[..., None, None]).to(FP8).view(torch.uint8)
        keep = torch.where((is_old & ~fresh)[:, :, None, :, None], old, codes.view(torch.uint8))
        new = torch.nn.functional.pad(new / after[..., None, None], (0, codes.shape[4] - dim)).to(FP8)
        codes = torch.where(is_new[:, :, None, :, None], new.view(torch.uint8), keep)
        pool.view(torch.uint8)[ids] = codes.transpose(3, 4) if tokens_last else codes
        scales[ids] = after

    one(s["k"], s["k_scale"], s["new_k"], False)
    one(s["v"], s["v_scale"], s["new_v"], True)
    return dict(k=s["k"][:-1], v=s["v"][:-1], k_scale=s["k_scale"][:-1], v_scale=s["v_scale"][:-1])


def _read(pool, scales, table, tokens_last, kind):
    """The values of each sequence's tokens: [batch, head, token, width]."""
    x = pool.view(torch.uint8)[table.long()].view(FP8).to(kind) * scales[table.long()][..., None, None].to(kind)
    x = x.transpose(3, 4) if tokens_last else x
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    case, q = s["case"], s["q"]
    b, new, heads, d = q.shape
    kv = case["kv_heads"]
    k = _read(s["k"], s["k_scale"], s["table"], False, torch.float32)[..., :d]
    v = _read(s["v"], s["v_scale"], s["table"], True, torch.float32)[..., :d]
    x = q.float().view(b, new, kv, heads // kv, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = (x @ k.transpose(2, 3).contiguous()) * d ** -0.5  # [batch, kv head, (query, head), token]
    at = s["lengths"].long()[:, None] - new + torch.arange(new, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") <= at.repeat_interleave(heads // kv, 1)[..., None]
    x = x.masked_fill(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = (p / total) @ v.contiguous()
    o = o.view(b, kv, new, heads // kv, d).permute(0, 2, 1, 3, 4).reshape(b, new, heads, d)
    lse = (top + torch.log(total)).view(b, kv, new, heads // kv).permute(0, 2, 1, 3).reshape(b, new, heads)
    return dict(out=o.to(q.dtype), lse=lse)


def _plain_beam(s):
    case, x = s["case"], s["logits"].double()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    scores = s["scores"].double()[..., None]
    value = scores + (x - lse)
    token = torch.arange(case["vocab"], device="cuda")
    value = torch.where(s["finished"][..., None], torch.where(token == EOS, scores, -math.inf), value)
    value, at = torch.sort(value.flatten(1), dim=-1, descending=True, stable=True)
    value, at = value[:, :case["take"]], at[:, :case["take"]]
    return dict(scores=value.float(), parents=at // case["vocab"], tokens=at % case["vocab"])


def _plain_reorder(s):
    b, k = s["parents"].shape
    rows = (s["parents"] + k * torch.arange(b, device="cuda")[:, None]).flatten()
    used = [t.view(torch.uint8)[:, :s["case"]["used"]] if t.dtype is FP8 else t[:, :s["case"]["used"]]
            for t in s["states"]]
    return [t.copy_(t[rows]) for t in used]


# ------------------------------------------------------------------------------------------- one pass


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        return _own(op, s)
    if op == "norm":
        return _plain_norm(s)
    if op == "append":
        return _plain_append(s)
    if op == "attention":
        return _plain_attention(s)
    if op == "beam":
        return _plain_beam(s)
    _plain_reorder(s)
    return _reordered(s)


def _reordered(s):
    return [t[:, :s["case"]["used"]] for t in s["states"]]


def _own(op, s):
    case = s["case"]
    if op == "norm":
        from tilelang.ops.norm import add_rms_norm_quant
        r = add_rms_norm_quant(s["x"], s["weight"], s["residual"], eps=EPS, group=case["group"],
                               pow2_scale=case["pow2"], return_norm=case["norm"])
        return dict(q=r.q, scale=r.scale, h=r.h, y=r.y)
    if op in ("append", "attention"):
        from tilelang.ops.kv_cache import KVCache, kv_cache_append, kv_cache_attention
        cache = KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"], case["dim"])
        if op == "append":
            kv_cache_append(cache, s["new_k"], s["new_v"], s["table"], s["lengths"])
            return dict(k=cache.k[:-1], v=cache.v[:-1], k_scale=cache.k_scale[:-1], v_scale=cache.v_scale[:-1])
        out, lse = kv_cache_attention(s["q"], cache, s["table"], s["lengths"], return_lse=True)
        return dict(out=out, lse=lse)
    if op == "beam":
        from tilelang.ops.beam import beam_select
        scores, parents, tokens = beam_select(s["logits"], s["scores"], case["take"], finished=s["finished"],
                                              eos_id=EOS)
        return dict(scores=scores, parents=parents, tokens=tokens)
    from tilelang.ops.beam import reorder_states
    reorder_states(s["states"], s["parents"], case["used"])
    return _reordered(s)


# ------------------------------------------------------------------------------------------- 64 bits


def _smallest_pow2(v):
    """The smallest power of two that is no smaller than v."""
    m, e = math.frexp(v)
    return math.ldexp(1.0, e - 1 if m == 0.5 else e)


def _exact_norm(s):
    case = s["case"]
    h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    y = s["weight"].double() * h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["width"] + EPS)
    parts = y.unflatten(1, (-1, case["group"] or case["width"]))
    scale = parts.abs().max(-1).values.clamp(min=1e-4) / 448
    if case["pow2"]:
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    q = (parts / scale.unsqueeze(-1)).flatten(1)
    return dict(q=q, scale=scale, h=h if s["residual"] is not None else None, y=y if case["norm"] else None)


def _exact_append(s):
    case = s["case"]
    page, new, d = case["page"], case["new"], case["dim"]
    table, lens = s["table"].tolist(), s["lengths"].tolist()
    out = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale")}
    for pool, x in (("k", s["new_k"].double()), ("v", s["new_v"].double())):
        for b, end in enumerate(lens):
            begin = end - new
            for nth in range(begin // page, (end - 1) // page + 1):
                lo, hi = max(begin, nth * page), min(end, (nth + 1) * page)
                a, z, i = lo - nth * page, hi - nth * page, table[b][nth]
                part = x[b, lo - begin:hi - begin].transpose(0, 1)  # [head, slot, dim]
                need = [_smallest_pow2(max(m / 448, 2.0 ** -22)) for m in part.abs().amax(dim=(1, 2)).tolist()]
                scale = torch.tensor(need, dtype=torch.float64, device="cuda")
                codes = out[pool][i] if pool == "k" else out[pool][i].transpose(1, 2)
                if a:
                    before = out[pool + "_scale"][i]
                    scale = torch.maximum(scale, before)
                    codes[:, :a] *= (before / scale)[:, None, None]
                codes[:, a:z, :d] = part / scale[:, None, None]
                codes[:, a:z, d:] = 0
                out[pool + "_scale"][i] = scale
    return {n: t[:-1] for n, t in out.items()}


def _exact_attention(s):
    q = s["q"].double()
    b, new, heads, d = q.shape
    kv = s["case"]["kv_heads"]
    out, lse = torch.empty_like(q), torch.empty(b, new, heads, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(s["lengths"][i])
        ids = s["table"][i].tolist()[:-(-n // s["case"]["page"])]
        k = torch.stack([s["k"][j].double() * s["k_scale"][j].double()[:, None, None] for j in ids], 1)
        v = torch.stack([s["v"][j].double() * s["v_scale"][j].double()[:, None, None] for j in ids], 1)
        k, v = k.flatten(1, 2)[:, :n, :d], v.transpose(2, 3).flatten(1, 2)[:, :n, :d]
        for g in range(kv):
            mine = slice(g * (heads // kv), (g + 1) * (heads // kv))
            x = torch.matmul(q[i, :, mine], k[g].t().contiguous()) / math.sqrt(d)
            hidden = torch.ones(new, n, dtype=torch.bool, device="cuda").triu(n - new + 1)
            x = x.masked_fill(hidden[:, None], -math.inf)
            lse[i, :, mine] = torch.logsumexp(x, -1)
            out[i, :, mine] = torch.matmul(torch.softmax(x, -1), v[g])
    return dict(out=out, lse=lse)


def _exact_beam(s):
    case = s["case"]
    found = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[:, :, None]
    found[s["finished"]] = -math.inf
    found[:, :, EOS] = torch.where(s["finished"], s["scores"].double(), found[:, :, EOS])
    return dict(scores=found.flatten(1).topk(case["take"], -1).values, parents=None, tokens=None)


def exact(case, seed):
    op = case["op"]
    if op == "reorder":  # bytes are moved, nothing is computed
        return None
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attention": _exact_attention, "beam": _exact_beam}[op](s)
