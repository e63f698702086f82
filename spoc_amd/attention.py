"""The attention layer of a transformer block that serves from a paged cache, on microscaled matrices: the residual's addition and the
root-mean-square norm, one product for queries, keys and values, rotary positions on the way into the cache, attention over it, and
the product back.

    python -m spoc_amd.attention [tokens] [width] [steps]    # a prompt, then steps of one token, checked against float64
"""
import torch

from . import hip


class MxAttention:
    """y = output(attention(qkv(norm(x + residual)))) with `qkv` [(heads + 2 kv_heads) head_dim, width] and `output` [width,
    heads head_dim] held in 4 bits (MxTensor "fp4"), a norm weight in the activations' type (bfloat16 or float16) and `rotary` a
    hip.Rotary or None.  It serves; the cache (a hip.KvCache of kv_heads heads) and the sequences' pages are the caller's."""

    def __init__(self, weight, qkv, output, heads, kv_heads, rotary=None, eps=1e-6):
        if weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("MxAttention: activations are bfloat16 or float16")
        if heads < 1 or kv_heads < 1 or heads % kv_heads or output.k % heads:
            raise ValueError(f"MxAttention: {heads} heads on {kv_heads}, {output.k} values")
        head_dim = output.k // heads
        if weight.shape != (qkv.k,) or output.rows != qkv.k or qkv.rows != (heads + 2 * kv_heads) * head_dim:
            raise ValueError(f"MxAttention: qkv is {qkv.rows} x {qkv.k}, output {output.rows} x {output.k}, the norm's weight {tuple(weight.shape)}")
        self.weight, self.qkv, self.output, self.rotary, self.eps = weight, qkv, output, rotary, eps
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim

    def __call__(self, x, cache, pages, lengths, starts=None, residual=None, prefix=None):
        """(y, h) for the tokens x [tokens, width]: the layer's output and h = x + residual.  pages, lengths and starts: as for
        hip.kv_append, lengths with the tokens among them.  prefix: (pages, length) of a prefix that all sequences share, as
        for hip.attention_shared."""
        tokens, q_heads, kv = x.shape[0], self.heads, self.kv_heads
        normed, h, _ = hip.rms_norm_mx(x, self.weight, residual=residual, eps=self.eps)
        qkv = hip.gemm_mx(normed, self.qkv, dtype=x.dtype).view(tokens, q_heads + 2 * kv, self.head_dim)
        q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv], qkv[:, q_heads + kv:]
        hip.kv_append(k, v, cache, pages, lengths, starts=starts, rotary=self.rotary, q=q, q_out=q, first=0 if prefix is None else prefix[1])
        # (attention leaves rows of no sequence alone, and a product would spread what is in fresh memory there)
        o = qkv.new_zeros(tokens, q_heads, self.head_dim) if starts is not None else qkv.new_empty(tokens, q_heads, self.head_dim)
        if prefix is None:
            hip.attention_paged(q, cache, pages, lengths, starts=starts, out=o)
        else:
            hip.attention_shared(q, cache, prefix[0], prefix[1], pages, lengths, starts=starts, out=o)
        y = hip.gemm_mx(hip.mx_quantize(o.flatten(1), "fp8"), self.output, dtype=x.dtype)
        return y, h


def main(argv=None):
    import sys
    sizes = [int(v) for v in (sys.argv[1:] if argv is None else argv)]
    tokens, width, steps = sizes + [100, 1024, 8][len(sizes):]
    heads, kv_heads, page = 8, 2, 16
    d = width // heads // 8 * 8
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    random = lambda std, *shape: torch.empty(shape, device="cuda").normal_(0, std, generator=gen)  # noqa: E731
    x = random(1, tokens + steps, width).bfloat16()
    weight = (1 + random(0.1, width)).bfloat16()
    qkv, output = hip.mx_quantize(random(0.05, (heads + 2 * kv_heads) * d, width), "fp4"), hip.mx_quantize(random(0.05, width, heads * d), "fp4")
    layer = MxAttention(weight, qkv, output, heads, kv_heads, hip.Rotary(d))
    count = -(-(tokens + steps) // page)
    cache = hip.KvCache.empty(count, page, kv_heads, d)
    pages = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)[None]
    int32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = [layer(x[:tokens], cache, pages, int32(tokens), starts=int32(0, tokens))[0]]
    got += [layer(x[n:n + 1], cache, pages, int32(n + 1))[0] for n in range(tokens, tokens + steps)]
    got = torch.cat(got).double()

    # float64 without the roundings to 8 bits, the whole sequence at once
    values = lambda q: hip.mx_dequantize(q, torch.float32).double()  # noqa: E731
    n = x.double() / (x.double().pow(2).mean(1, keepdim=True) + layer.eps).sqrt() * weight.double()
    all_heads = (n @ values(qkv).t()).view(-1, heads + 2 * kv_heads, d)
    angle = torch.arange(tokens + steps, device="cuda").double()[:, None] * layer.rotary.frequencies.cuda()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    turn = lambda t: torch.cat((t[..., :d // 2] * cos - t[..., d // 2:] * sin, t[..., :d // 2] * sin + t[..., d // 2:] * cos), -1)  # noqa: E731
    q, k, v = turn(all_heads[:, :heads]), turn(all_heads[:, heads:heads + kv_heads]), all_heads[:, heads + kv_heads:]
    rows = []
    for head in range(heads):
        kv = head // (heads // kv_heads)
        scores = (q[:, head] @ k[:, kv].t() / d ** 0.5).masked_fill(torch.ones(tokens + steps, tokens + steps, device="cuda", dtype=torch.bool).triu(1), float("-inf"))
        rows.append(scores.softmax(-1) @ v[:, kv])
    want = torch.stack(rows, 1).flatten(1) @ values(output).t()
    off = float((got - want).norm() / want.norm())
    # A rounding to e4m3 is off by up to 2^-4 of a value, 0.577 0.707 2^-4 = 0.0255 in the mean square over a mantissa's length.  A row of the norm brings
    # that into q, k and v; scores of std 0.05^2 width are then off by sqrt(2) 0.0255 of that, and o, a mean over weights that are off so
    # much each, by as much of itself; o's own rounding comes on top.  Half as much again for what a few rows are off from the mean.
    score = 2 ** 0.5 * 0.0255 * 0.05 ** 2 * width
    most = 1.5 * (score ** 2 + 2 * 0.0255 ** 2) ** 0.5
    print(f"{tokens} tokens and {steps} steps, {width} wide, {heads} heads on {kv_heads} of {d}: output within {off:.4f} (of the layer in float64 "
          f"without its roundings to 8 bits; {most:.4f} expected at most)")
    return 0 if off < most else 1


if __name__ == "__main__":
    raise SystemExit(main())
