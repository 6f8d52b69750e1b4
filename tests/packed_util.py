"""Plain 64-bit forms of the operators on packed sequences and the 4-bit cache, written from their definitions: one token, one head and
one sequence at a time, nibbles found where the layout puts them."""
import math

import torch

PAGE, GROUP = 32, 64


def word_indices(H):
    """Index of the code word and nibble of token t, dimension d: K and V, int64 [32, H]."""
    t, d = torch.arange(PAGE)[:, None], torch.arange(H)[None]
    k = t * (H // 8) + (d % 32) // 8 * (H // 32) + d // 32
    v = (((t // 8 * 8 + d % 64 // 8) * 4 + t % 4) * 2 + t % 8 // 4) * (H // 64) + d // 64
    return k, v, (d % 8).expand(PAGE, H)


def unpack_heads(raw):
    """raw uint8 [..., 36 H] -> codes, scales, minima of K, the same of V, fp64 [..., 32, H] each."""
    H = raw.shape[-1] // 36
    kw, vw, nib = (x.to(raw.device) for x in word_indices(H))
    run, par, out = PAGE * H // 2, PAGE * H // 16, []
    for base, word in ((0, kw), (run + par, vw)):
        byte = raw[..., (base + word * 4 + nib // 2).reshape(-1)].unflatten(-1, (PAGE, H)).long()
        code = (byte >> (4 * (nib % 2))) & 15
        p = raw[..., base + run:base + run + par].contiguous().view(torch.bfloat16).double().unflatten(-1, (PAGE, H // GROUP, 2))
        out += [code.double(), p[..., 0].repeat_interleave(GROUP, -1), p[..., 1].repeat_interleave(GROUP, -1)]
    return out


def pack_heads(codes, scales, minima):
    """The inverse for K and V: each argument a pair of [..., 32, H] (codes) and [..., 32, H / 64] (bf16 scales, minima)."""
    H = codes[0].shape[-1]
    kw, vw, nib = (x.to(codes[0].device) for x in word_indices(H))
    runs = []
    for c, s, z, word in ((codes[0], scales[0], minima[0], kw), (codes[1], scales[1], minima[1], vw)):
        words = torch.zeros(c.shape[:-2] + (PAGE * H // 8,), dtype=torch.int64, device=c.device)
        words.scatter_add_(-1, word.reshape(-1).expand(c.shape[:-2] + (-1,)), (c.long() << (4 * nib)).flatten(-2))
        by = torch.stack([(words >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2).to(torch.uint8)
        runs += [by, torch.stack([s, z], -1).to(torch.bfloat16).flatten(-3).contiguous().view(torch.uint8)]
    return torch.cat(runs, -1)


def quantised(x):
    """bf16 rows [..., H] -> (codes, scale, minimum) fp64 [..., H / 64, 64], [..., H / 64, 1] twice."""
    g = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).float().bfloat16().double()
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    s = torch.where(bad, math.nan, s)
    code = torch.where(s > 0, ((g - lo) / s).round().clamp(max=15), 0.0)
    return code, s, torch.where(bad, math.nan, lo)


def quantised_values(x):
    c, s, z = quantised(x)
    return (z + c * s).flatten(-2)


def norm_rope(x, w, eps, ep, pos):
    """x bf16 [T, heads, H] -> fp64, and what its fp32 arithmetic may be off by (absolute)."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs()
    if ep is not None:
        rot = ep.shape[2]
        inside = ((pos >= 0) & (pos < ep.shape[1]))[:, None, None]
        at = pos.clamp(0, ep.shape[1] - 1)
        c, s = (ep[i, at, :rot // 2].double()[:, None] for i in (0, 1))
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        both = a.abs() + b.abs()
        size = torch.cat([both, both, size[..., rot:]], -1)
        y = torch.where(inside, torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1), y)
    # statistics: H / 16 + 8 sums and a square root; two products of the norm, three operations of the rotation: far below 32 roundings
    return y, 32 * 2.0 ** -24 * size


def attention(q, k, v, before, causal, scale):
    """One sequence: q [n, heads, H], k and v [m, kv heads, H] fp64 -> output, weights [heads, n, m]. Token i sees keys 0 .. before + i."""
    n, heads, H = q.shape
    R = heads // k.shape[1]
    s = torch.einsum("nhd,mhd->hnm", q, k.repeat_interleave(R, 1)) * scale
    if causal:
        i, j = torch.arange(n, device=q.device)[:, None], torch.arange(k.shape[0], device=q.device)
        s = s.masked_fill(j > before + i, -math.inf)
    w = torch.softmax(s, -1).nan_to_num(0.0) if k.shape[0] else s
    return torch.einsum("hnm,mhd->nhd", w, v.repeat_interleave(R, 1)), w
