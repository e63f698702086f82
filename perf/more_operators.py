"""The operators of an attention layer that serves from a paged cache, as a list of cases that can be timed.

An operator is called as a program calls it: `hip.rotary` and `hip.rotary_backward` (rotary positions), `hip.kv_append` (keys
and values into the pages of their sequences, keys and queries rotated on the way), `hip.attention_paged` (single tokens,
chunks and prompts over the pages), and `hip.attention_shared` (the same for a batch whose sequences begin with one prefix).
With `own = False` the same outputs come from elementary torch operations in 32 bits.

Heads of 128 make the width of 4096 that this library's feed-forward layer is measured at; lengths are those of its products
(4095, 8192, 11007) and the odd ones that its kernels are tested at; between them they are drawn.
"""
import math

import torch

own = False

F32 = torch.float32
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token's queries, between a layer's product and its attention: what a launch costs
        dict(name="rotary_one_token", op="rotary", tokens=1, heads=32, d=128, dim=128, layout="half", factor=1.0, far=4096, dtype="bf16"),
        # a prompt's, at far positions of a context that was lengthened
        dict(name="rotary_prompt_far", op="rotary", tokens=8192, heads=32, d=128, dim=128, layout="half", factor=8.0, far=1000000, dtype="bf16"),
        # a training step's gradient: part of each head, neighbouring pairs, 32 bits, odd sizes
        dict(name="rotary_backward_part", op="rotary_backward", tokens=999, heads=13, d=80, dim=40, layout="interleaved", factor=1.0, far=4095, dtype="f32"),
        # a step of generation: a token for each sequence of a batch
        dict(name="append_tokens", op="append", batch=16, new=1, shortest=1, longest=4095, heads=32, kv_heads=8, d=128, page=16, dim=128, layout="half", idle=False, dtype="bf16"),
        # chunks of several prompts, of different lengths
        dict(name="append_prompts", op="append", batch=5, new=1638, shortest=1638, longest=8192, heads=32, kv_heads=8, d=128, page=64, dim=64, layout="interleaved", idle=False, dtype="f16"),
        # a token of one sequence: little to read, on the whole card
        dict(name="attention_one_token", op="attention", batch=1, new=1, shortest=4095, longest=4095, heads=32, kv_heads=8, d=128, page=16, idle=False, dtype="bf16"),
        # a token for each sequence of a batch, their lengths far apart, some places of the batch empty
        dict(name="attention_tokens", op="attention", batch=61, new=1, shortest=100, longest=11007, heads=32, kv_heads=8, d=128, page=16, idle=True, dtype="bf16"),
        # a token far into a long context, as many heads of keys as of queries
        dict(name="attention_long", op="attention", batch=1, new=1, shortest=131071, longest=131071, heads=16, kv_heads=16, d=64, page=256, idle=False, dtype="f16"),
        # a prompt
        dict(name="attention_prompt", op="attention", batch=1, new=8192, shortest=8192, longest=8192, heads=32, kv_heads=8, d=128, page=64, idle=False, dtype="bf16"),
        # chunks of prompts behind what is in the cache already, odd sizes
        dict(name="attention_chunks", op="attention", batch=5, new=500, shortest=700, longest=4095, heads=13, kv_heads=13, d=80, page=20, idle=False, dtype="f16"),
        # generation for a batch with one long prefix
        dict(name="shared_tokens", op="shared", batch=61, new=1, shortest=1, longest=500, prefix=8191, heads=32, kv_heads=8, d=128, page=16, idle=False, dtype="bf16"),
        # a few candidates of a few tokens each behind a prefix
        dict(name="shared_few", op="shared", batch=4, new=3, shortest=3, longest=61, prefix=1001, heads=16, kv_heads=4, d=64, page=32, idle=False, dtype="f16"),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform over [lo, hi]; every second one rounded to a multiple of 64 where it can be."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 256:
        v = v // 64 * 64
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(["rotary", "rotary_backward", "append", "attention", "attention", "attention", "shared", "shared"])
    if op.startswith("rotary"):
        d = 8 * _log(rng, 2, 32)
        while True:
            c = dict(op=op, tokens=_log(rng, 1, 16384), heads=_log(rng, 1, 64), d=d, dim=rng.choice([d, d // 2]), layout=rng.choice(["half", "interleaved"]),
                     factor=rng.choice([1.0, 4.0, 8.0]), far=_log(rng, 100, 1000000), dtype=rng.choice(["bf16", "f16", "f32"]))
            if c["tokens"] * c["heads"] * d * TYPES[c["dtype"]].itemsize <= 8192 * 32 * 128 * 2:
                return c
    while True:
        kv_heads = _log(rng, 1, 16)
        c = dict(op=op, batch=_log(rng, 1, 128), new=rng.choice([1, 1, _log(rng, 2, 4096)]), kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 2, 4, 8]),
                 d=rng.choice([64, 64, 128, 128, 128, 80, 256]), page=rng.choice([1, 16, 16, 20, 64, 256]), idle=rng.random() < 0.3, dtype=rng.choice(["bf16", "f16"]))
        c["longest"] = max(_log(rng, 16, 65536), c["new"])
        c["shortest"] = max(_log(rng, 1, c["longest"]), c["new"])
        if op == "append":
            c.update(dim=rng.choice([c["d"], c["d"] // 2]), layout=rng.choice(["half", "interleaved"]))
        if op == "shared":
            c["prefix"] = _log(rng, 16, 32768)
            c["longest"], c["shortest"] = max(c["longest"] // 16, c["new"]), max(c["shortest"] // 16, c["new"])
        if c["heads"] > 64 or c["batch"] * (c["longest"] + c["new"]) * kv_heads * c["d"] > 2 ** 28:
            continue
        w = work(c)
        if w["flops"] <= 4e11 and w["bytes"] <= 5e8:
            return c


# ---- what a program has before the call ------------------------------------------------------------------------------

def _news(case):
    """Tokens that each sequence brings; some places of a batch that has idle ones bring none."""
    return [0 if case["idle"] and b % 4 == 3 else case["new"] for b in range(case["batch"])]


def _lengths(case):
    """Keys of each sequence, the new ones among them: spread from the shortest to the longest, in no order."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [0 if new == 0 else hi if n == 1 else lo + (hi - lo) * (b * 37 % n) // (n - 1) for b, new in enumerate(_news(case))]


def _frequencies(dim, factor):
    """Radians from position to position of each pair, in 64 bits; slow ones (less than a turn in 4096) slowed by the factor, fast
    ones (from 4 turns on) as they are, in between in between."""
    f = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    keep = ((4096 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
    return f * keep + f / factor * (1 - keep)


def _plan(dim, layout, factor):
    from spoc_amd import hip
    return hip.Rotary(dim, layout=layout, scaling="ramp" if factor != 1.0 else None, factor=factor, trained=4096, low=1.0, high=4.0)


def _normal(gen, std, *shape):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, s, dtype = case["op"], dict(case), TYPES[case["dtype"]]
    if op.startswith("rotary"):
        first = torch.randint(0, max(case["far"] - case["tokens"], 1), (1,), device="cuda", generator=gen)
        s.update(x=_normal(gen, 1.0, case["tokens"], case["heads"], case["d"]).to(dtype),
                 positions=first + torch.arange(case["tokens"], device="cuda"), f=_frequencies(case["dim"], case["factor"]).cuda())
        if own:
            s["plan"] = _plan(case["dim"], case["layout"], case["factor"])
        return s
    page, lengths, news, kv_heads, d = case["page"], _lengths(case), _news(case), case["kv_heads"], case["d"]
    starts = [sum(news[:b]) for b in range(len(news) + 1)]
    held = [-(-n // page) for n in lengths]                        # pages of each sequence
    prefix = -(-case["prefix"] // page) if op == "shared" else 0
    order = torch.randperm(prefix + sum(held) + 3, device="cuda", generator=gen).to(torch.int32)
    pages = torch.full((len(held), max(max(held), 1)), 0, dtype=torch.int32, device="cuda")
    at = prefix
    for b, n in enumerate(held):
        pages[b, :n] = order[at:at + n]
        at += n
    s.update(host_lengths=lengths, host_starts=starts, host_held=held, pages=pages, lengths=_int(lengths),
             starts=None if case["new"] == 1 and not case["idle"] else _int(starts), prefix_pages=order[:prefix].contiguous(),
             keys=_normal(gen, 1.0, order.numel(), page, kv_heads, d).to(dtype), values=_normal(gen, 1.0, order.numel(), page, kv_heads, d).to(dtype),
             q=_normal(gen, 2.0, starts[-1], case["heads"], d).to(dtype))      # (some keys weigh much more than others)
    if op == "append":
        s.update(k=_normal(gen, 1.0, starts[-1], kv_heads, d).to(dtype), v=_normal(gen, 1.0, starts[-1], kv_heads, d).to(dtype),
                 f=_frequencies(case["dim"], 1.0).cuda())
    if own:
        from spoc_amd import hip
        s["cache"] = hip.KvCache(s["keys"], s["values"])
        if op == "append":
            s["plan"] = _plan(case["dim"], case["layout"], 1.0)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _rotated(x, positions, f, layout, sign=1.0):
    """Pairs turned by their angles, in 32 bits (the angles, which are of far positions, in 64); what is behind them as it is."""
    angle = positions.to(torch.float64)[:, None] * f
    cos, sin = torch.cos(angle).to(F32)[:, None], sign * torch.sin(angle).to(F32)[:, None]
    y, dim = x.to(F32), 2 * f.numel()
    if layout == "half":
        a, b = y[..., :dim // 2], y[..., dim // 2:dim]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = y[..., 0:dim:2], y[..., 1:dim:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, y[..., dim:]), -1).to(x.dtype)


def _attended(q, keys, values, hidden, scale):
    """[tokens, heads, d] queries over [length, kv_heads, d]: sums of exponents, their largest, and the weighted values; hidden:
    None, or which keys a token does not see."""
    tokens, heads, d = q.shape
    k, v = keys.to(F32).permute(1, 2, 0).contiguous(), values.to(F32).transpose(0, 1).contiguous()
    group = heads // k.shape[0]
    rows = q.to(F32).view(tokens, -1, group, d).permute(1, 0, 2, 3).reshape(k.shape[0], tokens * group, d)
    scores = torch.bmm(rows, k).mul_(scale)
    if hidden is not None:
        scores.view(k.shape[0], tokens, group, -1).masked_fill_(hidden[None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    back = lambda t: t.view(k.shape[0], tokens, group, -1).permute(1, 0, 2, 3).reshape(tokens, heads, -1)  # noqa: E731
    return back(top), back(p.sum(-1, keepdim=True)), back(torch.bmm(p, v))


def _positions(s):
    """The place in its sequence of each new token, and its page and slot."""
    place, page = [], []
    for b, n in enumerate(s["host_lengths"]):
        new = s["host_starts"][b + 1] - s["host_starts"][b]
        at = torch.arange(n - new, n, device="cuda")
        place.append(at)
        page.append(s["pages"][b].long()[at // s["page"]])
    place = torch.cat(place)
    return place, torch.cat(page), place % s["page"]


def _run_plain(s):
    op = s["op"]
    if op.startswith("rotary"):
        return _rotated(s["x"], s["positions"], s["f"], s["layout"], -1.0 if op == "rotary_backward" else 1.0)
    if op == "append":
        place, page, slot = _positions(s)
        s["keys"][page, slot] = _rotated(s["k"], place, s["f"], s["layout"])
        s["values"][page, slot] = s["v"]
        return {"q": _rotated(s["q"], place, s["f"], s["layout"]), "keys": s["keys"], "values": s["values"]}
    out, scale = torch.zeros_like(s["q"]), s["d"] ** -0.5
    gathered = lambda which, pages, n: which[pages.long()].flatten(0, 1)[:n]  # noqa: E731
    if op == "shared":
        before = _attended(s["q"], gathered(s["keys"], s["prefix_pages"], s["prefix"]), gathered(s["values"], s["prefix_pages"], s["prefix"]), None, scale)
    for b, n in enumerate(s["host_lengths"]):
        first, last = s["host_starts"][b], s["host_starts"][b + 1]
        if first == last:
            continue
        pages, new = s["pages"][b, :s["host_held"][b]], last - first
        hidden = None if new == 1 else torch.arange(n, device="cuda") > torch.arange(n - new, n, device="cuda")[:, None]
        top, total, o = _attended(s["q"][first:last], gathered(s["keys"], pages, n), gathered(s["values"], pages, n), hidden, scale)
        if op == "shared":
            most = torch.maximum(top, before[0][first:last])
            mine, other = torch.exp(top - most), torch.exp(before[0][first:last] - most)
            total, o = total * mine + before[1][first:last] * other, o * mine + before[2][first:last] * other
        out[first:last] = (o / total).to(out.dtype)
    return out


def _run_own(s):
    from spoc_amd import hip
    op = s["op"]
    if op == "rotary":
        return hip.rotary(s["x"], s["positions"], s["plan"])
    if op == "rotary_backward":
        return hip.rotary_backward(s["x"], s["positions"], s["plan"])
    if op == "append":
        q = hip.kv_append(s["k"], s["v"], s["cache"], s["pages"], s["lengths"], starts=s["starts"], rotary=s["plan"], q=s["q"])
        return {"q": q, "keys": s["keys"], "values": s["values"]}
    if op == "attention":
        return hip.attention_paged(s["q"], s["cache"], s["pages"], s["lengths"], starts=s["starts"])
    return hip.attention_shared(s["q"], s["cache"], s["prefix_pages"], s["prefix"], s["pages"], s["lengths"], starts=s["starts"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    op, d, size = case["op"], case["d"], TYPES[case["dtype"]].itemsize
    if op.startswith("rotary"):        # read and written once; positions; four products and two sums to a pair
        moved = case["tokens"] * case["heads"] * d
        return dict(bytes=2 * moved * size + 8 * case["tokens"], flops=3 * case["tokens"] * case["heads"] * case["dim"])
    heads, kv_heads, lengths, news = case["heads"], case["kv_heads"], _lengths(case), _news(case)
    table = 4 * sum(-(-n // case["page"]) for n in lengths) + 8 * len(lengths)
    if op == "append":
        tokens = sum(news)
        table = 4 * sum(-(-n // case["page"]) for n in news) + 8 * len(lengths)
        return dict(bytes=2 * tokens * (heads + 2 * kv_heads) * d * size + table, flops=3 * tokens * (heads + kv_heads) * case["dim"])
    seen = sum(new * n - new * (new - 1) // 2 for n, new in zip(lengths, news))        # pairs of a token and a key
    held = sum(lengths)
    if op == "shared":
        seen, held, table = seen + sum(news) * case["prefix"], held + case["prefix"], table + 4 * -(-case["prefix"] // case["page"])
    return dict(bytes=2 * sum(news) * heads * d * size + 2 * held * kv_heads * d * size + table, flops=4 * d * heads * seen)


# ---- the same from the definition, in 64 bits ------------------------------------------------------------------------

def _turn64(x, at, f, layout, direction):
    """Each pair as a complex number, times e^(i angle)."""
    dim = 2 * f.numel()
    x = x.double()
    pairs = x[:, :, :dim].unflatten(-1, (2, dim // 2)).transpose(-1, -2) if layout == "half" else x[:, :, :dim].unflatten(-1, (dim // 2, 2))
    angle = direction * at.double().outer(f)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
    z = torch.view_as_real(z)
    z = z.transpose(-1, -2).flatten(-2) if layout == "half" else z.flatten(-2)
    return torch.cat((z, x[:, :, dim:]), dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op.startswith("rotary"):
        return _turn64(s["x"], s["positions"], s["f"], s["layout"], -1 if op == "rotary_backward" else 1)
    lengths, starts, page, d = s["host_lengths"], s["host_starts"], s["page"], s["d"]
    if op == "append":
        keys, values, at = s["keys"].double(), s["values"].double(), torch.zeros(starts[-1], dtype=torch.int64, device="cuda")
        for b, n in enumerate(lengths):
            at[starts[b]:starts[b + 1]] = n - (starts[b + 1] - starts[b]) + torch.arange(starts[b + 1] - starts[b], device="cuda")
        k, v = _turn64(s["k"], at, s["f"], s["layout"], 1), s["v"].double()
        flat_keys, flat_values = keys.flatten(0, 1), values.flatten(0, 1)
        for b in range(len(lengths)):
            mine = slice(starts[b], starts[b + 1])
            where = s["pages"][b].long()[torch.div(at[mine], page, rounding_mode="floor")] * page + at[mine].remainder(page)
            flat_keys.index_copy_(0, where, k[mine])
            flat_values.index_copy_(0, where, v[mine])
        return {"q": _turn64(s["q"], at, s["f"], s["layout"], 1), "keys": keys, "values": values}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = s["heads"] // s["kv_heads"]
    for b, n in enumerate(lengths):
        new = starts[b + 1] - starts[b]
        if new == 0:
            continue
        row = torch.arange(n, device="cuda")
        where = s["pages"][b].long()[row // page] * page + row % page
        before = 0
        if op == "shared":
            before = s["prefix"]
            row = torch.arange(before, device="cuda")
            where = torch.cat((s["prefix_pages"].long()[row // page] * page + row % page, where))
        for h in range(s["heads"]):
            k, v = (s[name].flatten(0, 1)[where, h // group].double() for name in ("keys", "values"))
            for first in range(0, new, 2048):            # tokens at a time
                last = min(first + 2048, new)
                score = torch.mm(s["q"][starts[b] + first:starts[b] + last, h].double(), k.t()) / math.sqrt(d)
                if new > 1:
                    score += torch.full((last - first, before + n), -math.inf, dtype=torch.float64, device="cuda").triu(before + n - new + first + 1)
                out[starts[b] + first:starts[b] + last, h] = torch.mm(torch.exp(score - torch.logsumexp(score, 1, keepdim=True)), v)
    return out
