"""The attention side of a block between its packed linears: cases, plain forms and values in 64 bits.

A case is a dict of plain values; `op` is one of
  plan    block tables and slot maps for a step of `requests` requests (contexts from `shortest` to `longest`, new tokens from
          1 to `new` each) over pages of `page` tokens;
  rope    rotation of q and k by positions on several axes;
  norm    per-head norms of q and k with the rotation, k and v written into the paged cache;
  train   per-head norms of q and k with the rotation, forward and backward;
  attend  attention of one new token a row over the paged cache, `rows` rows of `shortest` to `longest` tokens.
Lengths are spread evenly over their logarithm and dealt to the rows by the seed, so that the work of a case is fixed.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # a decode step of a server: 32 requests with one new token each
        {"name": "plan_decode", "op": "plan", "requests": 32, "shortest": 77, "longest": 4096, "new": 1, "page": 16},
        # a mixed step: new prompts, chunks of long ones and single tokens together
        {"name": "plan_prompts", "op": "plan", "requests": 256, "shortest": 0, "longest": 32768, "new": 512, "page": 64},
        # image tokens of a diffusion transformer, positions on three axes
        {"name": "rope_image", "op": "rope", "tokens": 4608, "heads": 48, "kv_heads": 48, "dim": 128, "axes": "16,56,56",
         "interleaved": True, "dtype": "bf16"},
        # video tokens
        {"name": "rope_video", "op": "rope", "tokens": 9504, "heads": 40, "kv_heads": 40, "dim": 128, "axes": "44,42,42",
         "interleaved": True, "dtype": "fp16"},
        # one token of one request: the decode step where latency counts
        {"name": "norm_token", "op": "norm", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "axes": "128",
         "interleaved": False, "dtype": "bf16", "page": 16, "layout": "token"},
        # a prompt that goes into the cache, an odd number of tokens
        {"name": "norm_prompt", "op": "norm", "tokens": 4095, "heads": 40, "kv_heads": 8, "dim": 128, "axes": "128",
         "interleaved": False, "dtype": "fp16", "page": 64, "layout": "head"},
        # one block in LoRA training, 1056 tokens
        {"name": "train_image", "op": "train", "tokens": 1056, "heads": 48, "kv_heads": 48, "dim": 128, "axes": "16,56,56",
         "interleaved": True, "dtype": "bf16"},
        # the same for video
        {"name": "train_video", "op": "train", "tokens": 9504, "heads": 40, "kv_heads": 40, "dim": 128, "axes": "44,42,42",
         "interleaved": True, "dtype": "bf16"},
        # the first answer token after a short prompt
        {"name": "attend_short", "op": "attend", "rows": 1, "shortest": 77, "longest": 77, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "dtype": "fp16", "layout": "token"},
        # a decode batch of middling contexts
        {"name": "attend_batch", "op": "attend", "rows": 8, "shortest": 3000, "longest": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "layout": "token"},
        # one long document
        {"name": "attend_long", "op": "attend", "rows": 1, "shortest": 131071, "longest": 131071, "heads": 40, "kv_heads": 8,
         "dim": 128, "page": 64, "window": 0, "dtype": "fp16", "layout": "head"},
        # a server's batch: very unequal contexts
        {"name": "attend_ragged", "op": "attend", "rows": 64, "shortest": 100, "longest": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "layout": "head"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One call of the ranges above: from one token to the largest listed ones, odd sizes, the usual head layouts."""
    op = rng.choice(("plan", "rope", "norm", "norm", "train", "attend", "attend", "attend"))
    if op == "plan":
        requests = _log(rng, 1, 512)
        new = rng.choice((1, 1, _log(rng, 2, 512)))
        return {"op": op, "requests": requests, "shortest": rng.choice((0, 1, 100)), "longest": _log(rng, 101, 65536), "new": new,
                "page": rng.choice((8, 16, 32, 64, 100, 256))}
    dtype, layout = rng.choice(("fp16", "bf16")), rng.choice(("token", "head"))
    if op == "attend":
        kv_heads, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 4, 5, 8, 16))
        dim = rng.choice((64, 96, 128, 128, 128, 256))
        rows, longest = _log(rng, 1, 256), _log(rng, 1, 131072)
        window = rng.choice((0, 0, 0, _log(rng, 16, 4096)))
        while rows * longest * kv_heads * dim > 2.6e8:  # the plain form gathers all rows at the longest one's length
            rows, longest = max(1, rows // 2), max(1, longest * 3 // 4)
        return {"op": op, "rows": rows, "shortest": rng.randint(1, longest), "longest": longest, "heads": kv_heads * group,
                "kv_heads": kv_heads, "dim": dim, "page": rng.choice((16, 16, 32, 64, 100, 256)), "window": window, "dtype": dtype,
                "layout": layout}
    dim = rng.choice((64, 80, 96, 128, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 16, 24))
    heads = kv_heads * rng.choice((1, 1, 2, 4, 5))
    tokens = _log(rng, 1, 9504)
    while tokens * (heads + kv_heads) * dim > 9e7:
        tokens //= 2
    case = {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if op == "norm":
        # whole heads or the first half of them rotate
        case.update(axes=str(rng.choice((dim, dim, dim // 2))), interleaved=rng.random() < 0.25,
                    page=rng.choice((16, 32, 64, 100)), layout=layout)
    else:
        quarter = dim // 16 * 2
        case.update(axes=rng.choice(("%d,%d,%d" % (dim - 6 * quarter, 3 * quarter, 3 * quarter), "%d,%d" % (dim // 2, dim // 2),
                                     str(dim))), interleaved=rng.random() < 0.7)
    return case


# ------------------------------------------------------------------------------------------ inputs

def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly over their logarithm; the last is hi."""
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1) if n > 1 else 1.0))) - 1 for i in range(n)]


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(case):
    return _spread(case["requests" if case["op"] == "plan" else "rows"], case["shortest"], case["longest"])


def _dealt(values, seed):
    values = list(values)
    random.Random(seed).shuffle(values)
    return values


def _table(gen, blocks, lengths, page):
    """A block table of shuffled pages for `lengths` tokens a row; -1 where a row has no page."""
    need = torch.tensor([_pages(n, page) for n in lengths], device=DEV)
    width = max(1, int(need.max()))
    first = torch.cumsum(need, 0) - need
    at = torch.arange(width, device=DEV)
    order = torch.randperm(blocks, generator=gen, device=DEV).to(torch.int32)
    entry = order[(first[:, None] + at).clamp(max=blocks - 1)]
    return torch.where(at < need[:, None], entry, -1).contiguous(), order[int(need.sum()):].contiguous()


def _cache(gen, blocks, page, heads, dim, layout, dtype):
    """A cache [blocks, page, heads, dim], in memory by token or by head, with earlier tokens' values in it."""
    shape = (blocks, page, heads, dim) if layout == "token" else (blocks, heads, page, dim)
    c = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)
    return c if layout == "token" else c.transpose(1, 2)


def _frequencies(axes):
    """(inv_freq, axis) of the rotated pairs: each axis has its own ladder of frequencies."""
    sizes = [int(a) for a in axes.split(",")]
    freq = torch.cat([10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n in sizes])
    axis = torch.cat([torch.full((n // 2,), i, dtype=torch.int32) for i, n in enumerate(sizes)])
    return freq.float().to(DEV), axis.to(DEV)


def _positions(case, seed):
    """[axes, tokens]: a grid of frames, rows and columns, or the tokens' places in their request."""
    n, t = len(case["axes"].split(",")), torch.arange(case["tokens"], device=DEV)
    start = random.Random(seed).randrange(4096)
    if n == 1:
        return (t + start)[None].to(torch.int32)
    side = max(1, int(math.sqrt(case["tokens"] / 4)))
    grid = torch.stack([t // (side * side) + start % 7, t // side % side, t % side])
    return grid[-n:].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    op, s = case["op"], {"case": dict(case)}
    if op == "plan":
        context, new, page = _dealt(_lengths(case), seed), _dealt(_spread(case["requests"], 1, case["new"]), seed + 1), case["page"]
        every = [a + b for a, b in zip(context, new)]
        used = sum(_pages(e, page) - _pages(c, page) for c, e in zip(context, every))
        blocks = sum(_pages(e, page) for e in every) + 8
        table, free = _table(gen, blocks, context, page)
        width = max(_pages(e, page) for e in every)
        s["table"] = torch.nn.functional.pad(table[:, :width], (0, max(0, width - table.shape[1])), value=-1).contiguous()
        s["free"], s["tokens"] = free[: used + 8].contiguous(), sum(new)
        s["context"], s["new"] = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (context, new))
        return s
    dtype, dim, heads, kv_heads = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    if op == "attend":
        lengths = _dealt(_lengths(case), seed)
        blocks = sum(_pages(n, case["page"]) for n in lengths) + 3
        s["table"], _ = _table(gen, blocks, lengths, case["page"])
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        s["k_cache"], s["v_cache"] = (_cache(gen, blocks, case["page"], kv_heads, dim, case["layout"], dtype) for _ in range(2))
        # longer queries than keys: some tokens stand out, as in trained heads
        s["q"] = (2 * torch.randn(case["rows"], heads, dim, generator=gen, device=DEV)).to(dtype)
        return s
    tokens = case["tokens"]
    # q, k and v as the fused projection leaves them: one row a token, channels of unequal size
    gain = torch.exp(0.3 * torch.randn(heads + 2 * kv_heads, dim, generator=gen, device=DEV))
    qkv = (torch.randn(tokens, heads + 2 * kv_heads, dim, generator=gen, device=DEV) * gain).to(dtype)
    s["q"], s["k"], s["v"] = qkv.split((heads, kv_heads, kv_heads), 1)
    s["positions"] = _positions(case, seed)
    s["freq"], s["axis"] = _frequencies(case["axes"])
    if op != "rope":
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(dim, generator=gen, device=DEV)).to(dtype) for _ in range(2))
    if op == "norm":
        blocks = _pages(tokens, case["page"]) + 2
        s["k_cache"], s["v_cache"] = (_cache(gen, blocks, case["page"], kv_heads, dim, case["layout"], dtype) for _ in range(2))
        t, page = torch.arange(tokens, device=DEV), case["page"]
        s["slots"] = torch.randperm(blocks, generator=gen, device=DEV)[t // page] * page + t % page
    if op == "train":
        s["gq"], s["gk"] = (torch.randn(tokens, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads))
    return s


# ------------------------------------------------------------------------------------- plain forms

def _plain_plan(s):
    context, new, page, tokens = s["context"].long(), s["new"].long(), s["case"]["page"], s["tokens"]
    lengths = context + new
    old, every = (context + page - 1) // page, (lengths + page - 1) // page
    need = every - old
    first = torch.cumsum(need, 0) - need
    ends = torch.cumsum(new, 0)
    starts = ends - new
    at = torch.arange(s["table"].shape[1], device=DEV)
    fresh = s["free"][(first[:, None] + at - old[:, None]).clamp(0, s["free"].numel() - 1)]
    table = torch.where((at >= old[:, None]) & (at < every[:, None]), fresh, s["table"])
    token = torch.arange(tokens, device=DEV)
    row = (token[:, None] >= ends).sum(1)
    position = context[row] + token - starts[row]
    slots = table[row, position // page].long() * page + position % page
    s["table"].copy_(table)
    return [slots, position.int(), row.int(), torch.cat([starts, ends[-1:]]).int(), lengths.int(), need.sum().int().reshape(1),
            s["table"]]


def _plain_angles(s):
    a = s["positions"].float()[s["axis"].long()].T * s["freq"]
    return a.cos()[:, None], a.sin()[:, None]


def _plain_rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    a, rest = x[..., : 2 * half], x[..., 2 * half:]
    u, v = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., :half], a[..., half:])
    p, q = u * cos - v * sin, u * sin + v * cos
    a = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([a, rest], -1)


def _plain_norm(x):
    rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return x * rstd, rstd


def _plain_norm_rope(s, x, w, cos, sin):
    return _plain_rotate(w.float() * _plain_norm(x.float())[0], cos, sin, s["case"]["interleaved"])


def _plain_store(cache, values, slots, page):
    cache[slots // page, slots % page] = values.to(cache.dtype)
    return cache


def _plain_gradient(s, g, x, w, cos, sin):
    g = _plain_rotate(g.float(), cos, -sin, s["case"]["interleaved"])
    unit, rstd = _plain_norm(x.float())
    wg = w.float() * g
    dx = rstd * (wg - unit * (wg * unit).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * unit).sum((0, 1)).to(w.dtype)


def _plain_attend(s):
    case, table, lengths = s["case"], s["table"], s["lengths"]
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    at = torch.arange(case["longest"], device=DEV)
    block = table[:, at // page].long().clamp(min=0)
    k, v = (c[block, at % page].float() for c in (s["k_cache"], s["v_cache"]))  # [rows, tokens, heads, dim]
    seen = at < lengths[:, None]
    if case["window"]:
        seen &= at >= lengths[:, None] - case["window"]
    q = s["q"].float().view(case["rows"], kv_heads, -1, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * dim ** -0.5
    score = torch.where(seen[:, None, None], score, -torch.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, v.transpose(1, 2)) / p.sum(-1, keepdim=True)
    return out.reshape(s["q"].shape).to(s["q"].dtype)


def _plain(s):
    op = s["case"]["op"]
    if op == "plan":
        return _plain_plan(s)
    if op == "attend":
        return _plain_attend(s)
    cos, sin = _plain_angles(s)
    dtype = s["q"].dtype
    if op == "rope":
        return [_plain_rotate(x.float(), cos, sin, s["case"]["interleaved"]).to(dtype) for x in (s["q"], s["k"])]
    q, k = _plain_norm_rope(s, s["q"], s["wq"], cos, sin).to(dtype), _plain_norm_rope(s, s["k"], s["wk"], cos, sin).to(dtype)
    if op == "norm":
        page = s["case"]["page"]
        return [q, _plain_store(s["k_cache"], k, s["slots"], page), _plain_store(s["v_cache"], s["v"], s["slots"], page)]
    dq, dwq = _plain_gradient(s, s["gq"], s["q"], s["wq"], cos, sin)
    dk, dwk = _plain_gradient(s, s["gk"], s["k"], s["wk"], cos, sin)
    return [q, k, dq, dk, dwq, dwk]


def _qlin():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-kernels-public_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qlin
    return qlin


def run(s):
    if not own:
        return _plain(s)
    q, case = _qlin(), s["case"]
    op = case["op"]
    if op == "plan":
        plan = q.paged_plan(s["context"], s["new"], s["table"], s["free"], case["page"], s["tokens"])
        return [plan.slots, plan.positions, plan.rows, plan.starts, plan.lengths, plan.used, s["table"]]
    if op == "attend":
        return q.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], window=case["window"])
    turn, inter = (s["positions"], s["freq"], s["axis"]), case["interleaved"]
    if op == "rope":
        return list(q.axis_rope(s["q"], s["k"], *turn, interleaved=inter))
    if op == "norm":
        out = q.qk_norm_rope_store(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["positions"], s["freq"], s["slots"], s["k_cache"],
                                   s["v_cache"], s["axis"], eps=EPS, interleaved=inter)
        return [out, s["k_cache"], s["v_cache"]]
    out = q.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], *turn, eps=EPS, interleaved=inter)
    return [*out, *q.qk_norm_rope_grad(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], *turn, eps=EPS, interleaved=inter)]


def work(case):
    op = case["op"]
    if op == "plan":
        context, new, page = _lengths(case), _spread(case["requests"], 1, case["new"]), case["page"]
        used = sum(new) // page + 1
        # lengths in and out, the partly filled pages' entries, free pages in, table entries out, 16 bytes a token out
        return {"bytes": case["requests"] * (4 + 4 + 4 + 4 + 4) + used * 8 + sum(new) * 16, "flops": 4 * sum(new) + 8 * len(context)}
    dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
    if op == "attend":
        lengths = [min(n, case["window"] or n) for n in _lengths(case)]
        pages = sum(_pages(n, case["page"]) for n in lengths)
        return {"bytes": 2 * 2 * sum(lengths) * kv_heads * dim + 2 * 2 * case["rows"] * heads * dim + 4 * pages,
                "flops": 4 * sum(lengths) * heads * dim}
    tokens, values = case["tokens"], case["tokens"] * (heads + kv_heads) * dim
    moved = {"rope": 2 * values, "norm": 2 * (values + tokens * kv_heads * dim), "train": 6 * values}[op]
    return {"bytes": 2 * moved + 4 * tokens * len(case["axes"].split(",")) + (8 * tokens if op == "norm" else 0),
            "flops": {"rope": 3, "norm": 7, "train": 20}[op] * values}


# ----------------------------------------------------------------------------- the results in 64 bits

def _turned(x, angle, interleaved):
    """x rotated by complex numbers of the pairs' angles."""
    n = 2 * angle.shape[-1]
    a = x[..., :n]
    a = a.unflatten(-1, (-1, 2)) if interleaved else a.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(a.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    a = torch.view_as_real(z)
    a = a if interleaved else a.transpose(-1, -2)
    return torch.cat([a.flatten(-2), x[..., n:]], -1)


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if op == "attend":
        rows = []
        for b, n in enumerate(s["lengths"].tolist()):
            first = max(0, n - case["window"]) if case["window"] else 0
            pages = s["table"][b, : _pages(n, case["page"])].long()
            k, v = (c[pages].double().flatten(0, 1)[first:n].transpose(0, 1) for c in (s["k_cache"], s["v_cache"]))
            q = s["q"][b].double().unflatten(0, (case["kv_heads"], -1))
            p = torch.softmax((q @ k.transpose(1, 2).contiguous()) / math.sqrt(case["dim"]), -1)
            rows.append((p @ v.contiguous()).flatten(0, 1))
        return torch.stack(rows)
    angle = s["positions"][s["axis"].long()].T.double() * s["freq"].double()
    if op == "rope":
        return [_turned(s[n].double(), angle, case["interleaved"]) for n in ("q", "k")]
    leaves = [s[n].double().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    q, k = (_turned(torch.nn.functional.rms_norm(x, (case["dim"],), w, EPS), angle, case["interleaved"])
            for x, w in zip(leaves[:2], leaves[2:]))
    if op == "train":
        grads = torch.autograd.grad((q, k), leaves, (s["gq"].double(), s["gk"].double()))
        return [q.detach(), k.detach(), *grads]
    caches = []
    for name, values in (("k_cache", k.detach()), ("v_cache", s["v"].double())):
        c = s[name].double()
        block, place = s["slots"].div(case["page"], rounding_mode="floor"), s["slots"].remainder(case["page"])
        for h in range(case["kv_heads"]):
            c[:, :, h].index_put_((block, place), values[:, h])
        caches.append(c)
    return [q.detach(), *caches]
