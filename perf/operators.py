"""Serving many sequences without padding, from a cache that is held in 4 bits, as cases that can be timed and checked.

Four operators, in the order in which a decoder layer calls them behind its q/k/v linear:
  norm_rope  RMS norm of every query and key head, then the rotation by the token's position, in one pass
  append     the same pass with the keys and values written to the cache in 4 bits, and the call's tokens read back from it
  packed     attention over whole prompts, causal, laid end to end without padding
  cache      attention of a few new tokens per sequence over the 4-bit cache

The cache of one layer is a pool of pages uint8 [pages, kv heads, 36 H] for head size H (64 or 128); a page holds 32 tokens of one
sequence, table[b, i] names the page of tokens 32 i .. 32 i + 31 of sequence b. 64 consecutive values of a key or value row share
a scale and a minimum (bf16); value = minimum + code * scale, code 0..15. One head of a page holds four runs of bytes:
  K codes   [32 tokens][4][H / 32] words: word (t, i) of a token holds its values 32 i + 8 t + 0..7, lowest nibble first
  K params  [32 tokens][H / 64] (scale, minimum)
  V codes   [4 groups of 8 tokens][8][4][2][H / 64] words: word (g, t, u, h) of a group holds values 64 h + 8 g + 0..7 of its token t + 4 u
  V params  as K params"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 5e5
PAGE = 32
GROUP = 64
MOST_SCORES = 32 * 8192 * 8192  # heads x tokens x tokens of one padded batch of prompts


def _case(name, op, heads, kv_heads, head_dim, batch, tokens, cached=0, ragged=False, salt=0):
    return dict(name=name, op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, tokens=tokens, cached=cached, ragged=ragged, salt=salt)


def listed():
    return [
        # one decoding sequence of a grouped-head decoder: a launch and little else
        _case("norm rope 1", "norm_rope", 32, 8, 128, 1, 1),
        # a prompt of odd length: the pass over its q/k/v rows
        _case("norm rope 8191", "norm_rope", 32, 8, 128, 1, 8191),
        # a decode step of 64 sequences: every sequence appends one token behind what it has cached
        _case("append 64x1", "append", 32, 8, 128, 64, 1, 2000, ragged=True, salt=1),
        # prompts of unequal lengths, some of them behind earlier turns of their conversation
        _case("append 16 prompts", "append", 32, 8, 128, 16, 2048, 600, ragged=True, salt=2),
        # a handful of chat prompts on a decoder with one key head per query head of 64
        _case("packed 24 short 64", "packed", 32, 32, 64, 24, 300, ragged=True, salt=3),
        # a batch of prompts of unequal lengths
        _case("packed 16 prompts", "packed", 32, 8, 128, 16, 2048, ragged=True, salt=4),
        # one long prompt
        _case("packed 1x8192", "packed", 32, 8, 128, 1, 8192),
        # interactive chat: one sequence, one token
        _case("cache 1x1024", "cache", 32, 8, 128, 1, 1, 1024),
        # a serving engine's decode step
        _case("cache 16x2048", "cache", 32, 8, 128, 16, 1, 2048),
        # the same on a wide decoder, sequences of any age
        _case("cache 64 ragged", "cache", 64, 8, 128, 64, 1, 4096, ragged=True, salt=5),
        # one token behind a very long document
        _case("cache 1x131072", "cache", 32, 8, 128, 1, 1, 131072),
        # five drafted tokens per sequence are verified, one key head per query head of 64
        _case("cache 8x5 drafted 64", "cache", 32, 32, 64, 8, 5, 1500, ragged=True, salt=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm_rope", "append", "packed", "packed", "cache", "cache", "cache"))
    kv, group = rng.choice((1, 2, 4, 5, 8, 16, 32)), rng.choice((1, 1, 2, 3, 4, 4, 5, 7, 8, 12, 16))
    while kv * group > 64:
        kv //= 2
    dim, salt = rng.choice((64, 128, 128)), rng.randrange(1 << 30)
    heads = kv * group
    ragged = rng.random() < 0.7
    if op == "norm_rope":
        return _case("", op, heads, kv, dim, 1, _log(rng, 1, 8000)) | {"salt": salt}
    if op == "append":
        batch = _log(rng, 1, 48)
        return _case("", op, heads, kv, dim, batch, _log(rng, 1, max(2, 16000 // batch)), rng.choice((0, _log(rng, 1, 2000))), ragged, salt)
    if op == "packed":
        batch = _log(rng, 1, 64)
        most = int(math.sqrt(MOST_SCORES / 2 / (batch * heads)))
        return _case("", op, heads, kv, dim, batch, _log(rng, 1, min(6000, most)), 0, ragged, salt)
    batch = _log(rng, 1, 128)
    tokens = rng.choice((1, 1, 1, 2, 3, 4, 8))
    most = 64 * 4096 * 8 // (batch * kv)
    return _case("", op, heads, kv, dim, batch, tokens, _log(rng, 1, max(2, min(100000, most))), ragged, salt)


def _lengths(case):
    """New tokens of every sequence, and the tokens that it has cached before."""
    n, rng = case["batch"], random.Random(case["salt"])
    new, old = [case["tokens"]] * n, [case["cached"]] * n
    if case["ragged"]:
        if case["op"] in ("append", "packed"):
            new = [_log(rng, 1, case["tokens"]) for _ in range(n - 1)] + [case["tokens"]]
        old = [_log(rng, 1, case["cached"] + 1) - 1 for _ in range(n - 1)] + [case["cached"]]
        rng.shuffle(new)
        rng.shuffle(old)
    return new, old


def _width(case):
    return (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]


def _values(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rope_table(positions, dim):
    """fp32 [2, positions, dim]: cosines, then sines, of the half-split rotation."""
    freq = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()]).repeat(1, 1, 2).float().contiguous()


def _pool(gen, case, pages):
    """Pages as a program finds them: rows whose channels have means and sizes of their own, in codes, scales and minima."""
    kv, dim = case["kv_heads"], case["head_dim"]
    runs = []
    for _ in range(2):
        codes = (_values(gen, pages, kv, PAGE * dim // 2, 2) * 3.2 + 7.5).round().clamp(0, 15).to(torch.uint8)
        runs.append(codes[..., 0] | codes[..., 1] << 4)
        scale = (_values(gen, pages, kv, PAGE, dim // GROUP) * 0.2).exp() * 0.32
        least = -7.5 * scale * (1 + 0.1 * _values(gen, pages, kv, PAGE, dim // GROUP))
        runs.append(torch.stack([scale, least], -1).bfloat16().flatten(2).view(torch.uint8))
    return torch.cat(runs, -1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    heads, kv, dim, op = case["heads"], case["kv_heads"], case["head_dim"], case["op"]
    new, old = _lengths(case)
    total = sum(new)
    s = dict(op=op, heads=heads, kv_heads=kv, head_dim=dim, longest=max(new))
    if op in ("norm_rope", "append"):
        scale = (_values(gen, heads + 2 * kv, 1) * 0.3).exp()
        s["qkv"] = (_values(gen, total, heads + 2 * kv, dim) * scale).bfloat16().flatten(1)
        s["q_norm"], s["k_norm"] = ((1 + 0.2 * _values(gen, dim)).bfloat16() for _ in range(2))
        s["table"] = _rope_table(max(a + b for a, b in zip(new, old)), dim)
    if op != "norm_rope":
        s["cu"] = torch.tensor([0] + new).cumsum(0).to("cuda", torch.int32)
    if op == "norm_rope":
        s["pos"] = torch.arange(total, device="cuda")
    if op == "packed":
        # as the pass in front leaves them: q and k in tensors of their own, v still among the rows of the linear
        s["q"], s["k"] = ((_values(gen, total, n, dim) * 1.5).bfloat16() for n in (heads, kv))
        s["v"] = _values(gen, total, heads + 2 * kv, dim).bfloat16()[:, heads + kv:]
    if op in ("append", "cache"):
        need = [(a + b + PAGE - 1) // PAGE for a, b in zip(new, old)]
        order = torch.randperm(sum(need), generator=gen, device="cuda").to(torch.int32).split(need)
        s["pages"] = torch.nn.utils.rnn.pad_sequence(list(order), batch_first=True, padding_value=-1).contiguous()
        s["lengths"] = torch.tensor(old, device="cuda", dtype=torch.int32)
        s["pool"] = _pool(gen, case, sum(need))
        if op == "cache":
            s["q"] = (_values(gen, total, heads, dim) * 1.5).bfloat16()
    return s


# ---------------------------------------------------------------- plain forms

def _norm_rope(s, pos):
    """q, k, v [tokens, heads, dim], bf16."""
    heads, kv, dim = s["heads"], s["kv_heads"], s["head_dim"]
    x = s["qkv"].float().view(-1, heads + 2 * kv, dim)
    qk = x[:, :heads + kv]
    w = torch.cat([s["q_norm"].float().expand(heads, dim), s["k_norm"].float().expand(kv, dim)])
    y = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    lo, hi = y.chunk(2, -1)
    c, sn = s["table"][:, pos, None, :dim // 2]
    y = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1).bfloat16()
    return y[:, :heads], y[:, heads:], s["qkv"].view(-1, heads + 2 * kv, dim)[:, heads + kv:]


def _in_4_bits(x):
    """The values that the cache holds in the place of x, bf16."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((0.5 * hi - 0.5 * lo) / 7.5).bfloat16().float()
    code = ((0.5 * g - 0.5 * lo) / (0.5 * scale)).round().clamp(0, 15)
    return (lo + torch.where(scale > 0, code, 0) * scale).bfloat16().flatten(-2)


def _place(s, total):
    """Sequence and index within it of every token of the call."""
    at = torch.arange(total, device="cuda")
    seq = torch.searchsorted(s["cu"][1:].contiguous(), at.to(torch.int32), right=True)
    return seq, at - s["cu"][seq]


def _cached(s):
    """Keys and values of every sequence, fp32 [batch, capacity, kv heads, dim] each."""
    kv, dim = s["kv_heads"], s["head_dim"]
    page = s["pool"][s["pages"].clamp(min=0).long()]
    batch, n = page.shape[:2]
    words, params = PAGE * dim // 2, PAGE * dim // GROUP * 4
    kc, kp, vc, vp = page.split([words, params, words, params], -1)

    def nibbles(codes, *shape):
        return torch.stack([codes & 15, codes >> 4], -1).reshape(batch, n, kv, *shape, 8).float()

    # to [batch, page, tokens .., kv heads, values ..]
    k = nibbles(kc, PAGE, 4, dim // 32).permute(0, 1, 3, 2, 5, 4, 6)
    v = nibbles(vc, 4, 8, 4, 2, dim // 64).permute(0, 1, 3, 6, 5, 2, 7, 4, 8)

    def valued(codes, p):
        p = p.contiguous().view(torch.bfloat16).float().view(batch, n, kv, PAGE, dim // GROUP, 2)
        p = p.transpose(2, 3).reshape(batch, n * PAGE, kv, dim // GROUP, 2)
        return (codes.reshape(batch, n * PAGE, kv, dim // GROUP, GROUP) * p[..., :1] + p[..., 1:]).flatten(-2)

    return valued(k, kp), valued(v, vp)


def _attend(q, k, v, visible):
    """q [b, n, heads, d], k and v [b, m, kv, d], fp32; visible [b, n, m]."""
    b, n, heads, d = q.shape
    q = q.view(b, n, k.shape[2], -1, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    p = q @ k.permute(0, 2, 3, 1) * d ** -0.5
    p = p.view(b, k.shape[2], -1, n, k.shape[1]).masked_fill_(~visible[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).flatten(2, 3)
    o = p @ v.transpose(1, 2)
    return o.view(b, k.shape[2], -1, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)


def _padded(s, x, seq, at):
    y = x.new_zeros((s["cu"].numel() - 1, s["longest"]) + x.shape[1:], dtype=torch.float32)
    y[seq, at] = x.float()
    return y


def _plain(s):
    op = s["op"]
    if op == "norm_rope":
        return _norm_rope(s, s["pos"])[:2]
    total = (s["qkv"] if op == "append" else s["q"]).shape[0]
    seq, at = _place(s, total)
    if op == "append":
        q, k, v = _norm_rope(s, s["lengths"][seq] + at)
        return q, k, _in_4_bits(k), _in_4_bits(v)
    q = _padded(s, s["q"], seq, at)
    n = torch.arange(s["longest"], device="cuda")
    if op == "packed":
        k, v = _padded(s, s["k"], seq, at), _padded(s, s["v"], seq, at)
        visible = (n[:, None] >= n).expand(q.shape[0], -1, -1)
    else:
        k, v = _cached(s)
        m = torch.arange(k.shape[1], device="cuda")
        visible = m <= s["lengths"][:, None, None] + n[:, None]
    return _attend(q, k, v, visible)[seq, at].bfloat16()


def _own(s):
    from tpp_pytorch_extension_b200._C import _packed_attn as P
    heads, kv, dim, op = s["heads"], s["kv_heads"], s["head_dim"], s["op"]
    if op == "norm_rope":
        return P.qk_norm_rope(s["qkv"], heads, kv, dim, s["q_norm"], s["k_norm"], EPS, s["table"], s["pos"])
    if op == "packed":
        return P.attention_packed(s["q"], s["k"], s["v"], s["cu"])
    cache = P.Int4Cache.over([s["pool"]], s["pages"], s["lengths"])
    one = s["longest"] == 1
    if op == "append":
        q, k = P.qk_norm_rope(s["qkv"], heads, kv, dim, s["q_norm"], s["k_norm"], EPS, s["table"], cu_seqlens=None if one else s["cu"], cache=cache)
        return q, k, *P.read_int4(cache, 0, s["qkv"].shape[0], None if one else s["cu"])
    return P.attention_int4(s["q"], cache, 0, None if one else s["cu"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    heads, kv, dim, op = case["heads"], case["kv_heads"], case["head_dim"], case["op"]
    new, old = _lengths(case)
    total, held = sum(new), 2 * kv * (dim // 2 + 4 * dim // GROUP)  # bytes of a cached token
    if op in ("norm_rope", "append"):
        moved = total * (2 * heads + (2 if op == "norm_rope" else 3) * kv) * dim * 2  # q, k (v) in, q, k out
        moved += total * 8 if op == "norm_rope" else total * (2 * kv * dim * 2 + held)  # positions; cached, and read back as bf16
        return {"bytes": moved + max(a + b for a, b in zip(new, old)) * dim * 4, "flops": total * (heads + kv) * dim * 8}
    if op == "packed":
        pairs = sum(n * (n + 1) // 2 for n in new)
        return {"bytes": total * (2 * heads + 2 * kv) * dim * 2, "flops": 4 * heads * dim * pairs}
    pairs = sum(n * m + n * (n + 1) // 2 for n, m in zip(new, old))
    return {"bytes": total * 2 * heads * dim * 2 + sum(a + b for a, b in zip(new, old)) * held, "flops": 4 * heads * dim * pairs}


# ---------------------------------------------------------------- in 64 bits

def _exact_rows(s, heads, offset, weight, pos):
    dim = s["head_dim"]
    x = s["qkv"].double().unflatten(1, (-1, dim))[:, offset:offset + heads]
    if weight is None:
        return x
    x = x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
    turn = torch.complex(s["table"][0, pos, :dim // 2].double(), s["table"][1, pos, :dim // 2].double())[:, None]
    z = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) * turn
    return torch.cat([z.real, z.imag], -1)


def _exact_4_bits(x):
    """The cache quantises what a bf16 cache would hold, with a scale that is rounded to bf16."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], GROUP):
        part = x[..., g:g + GROUP].bfloat16().double()
        least, most = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        scale = ((most - least) / 15).bfloat16().double()
        steps = torch.round((part - least) / torch.where(scale == 0, 1.0, scale))
        out[..., g:g + GROUP] = least + torch.minimum(steps, torch.full_like(steps, 15)) * scale
    return out


def _exact_attention(q, k, v, before):
    """One sequence: q [n, heads, d], k and v [before + n, kv, d], 64 bits."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    out = torch.empty_like(q)
    hidden = torch.arange(k.shape[0], device="cuda")[None] > before + torch.arange(n, device="cuda")[:, None]
    for h in range(heads):
        score = (q[:, h] @ k[:, h // group].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
        out[:, h] = torch.softmax(score, 1) @ v[:, h // group]
    return out


def _exact_page(s, index):
    """Keys and values of one page, fp64 [32, kv heads, dim] each, from where the layout puts every nibble."""
    kv, dim = s["kv_heads"], s["head_dim"]
    raw = s["pool"][index]
    token, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(dim, device="cuda")[None]
    k_word = token * (dim // 8) + (d % 32 // 8) * (dim // 32) + d // 32
    v_word = ((((token // 8) * 8 + d % 64 // 8) * 4 + token % 4) * 2 + token % 8 // 4) * (dim // 64) + d // 64
    got, base = [], 0
    for word in (k_word, v_word):
        byte = raw[..., (base + word * 4 + d % 8 // 2).flatten()].unflatten(-1, (PAGE, dim)).to(torch.int32)
        code = torch.where(d % 2 == 1, byte >> 4, byte & 15).double()
        base += PAGE * dim // 2
        params = raw[..., base:base + PAGE * dim // 16].contiguous().view(torch.bfloat16).double().unflatten(-1, (PAGE, dim // GROUP, 2))
        base += PAGE * dim // 16
        got.append((code * params[..., 0].repeat_interleave(GROUP, -1) + params[..., 1].repeat_interleave(GROUP, -1)).movedim(-3, -2))
    return [x.flatten(0, 1) for x in got]


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv = s["heads"], s["kv_heads"]
    new, old = _lengths(case)
    if s["op"] in ("norm_rope", "append"):
        pos = torch.cat([torch.arange(m, m + n, device="cuda") for n, m in zip(new, old)])
        q, k = _exact_rows(s, heads, 0, s["q_norm"], pos), _exact_rows(s, kv, heads, s["k_norm"], pos)
        if s["op"] == "norm_rope":
            return q, k
        return q, k, _exact_4_bits(k), _exact_4_bits(_exact_rows(s, kv, heads + kv, None, pos))
    out, at = [], 0
    for b, (n, m) in enumerate(zip(new, old)):
        q = s["q"][at:at + n].double()
        if s["op"] == "packed":
            k, v, m = s["k"][at:at + n].double(), s["v"][at:at + n].double(), 0
        else:
            k, v = _exact_page(s, s["pages"][b, :(m + n + PAGE - 1) // PAGE].long())
            k, v = k[:m + n], v[:m + n]
        out.append(_exact_attention(q, k, v, m))
        at += n
    return torch.cat(out)
