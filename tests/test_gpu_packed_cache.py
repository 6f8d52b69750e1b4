"""Head norms with rotation, the append to the 4-bit cache, its read-back, and attention over it, against 64-bit forms."""
import math

import pytest
import torch

from tests import packed_util as U

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8  # a rounding to bf16


def P():
    from tpp_pytorch_extension_b200._C import _packed_attn
    return _packed_attn


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def table(positions, rot, theta=1e4):
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.stack([a.cos(), a.sin()]).repeat(1, 1, 2).float().contiguous()


def close_rounded(got, want, extra):
    """got is want rounded to bf16, of a value that was `extra` off."""
    err = (got.double() - want).abs()
    assert bool((err <= BF16 * want.abs() + 1.01 * extra + 2.0 ** -130).all()), float((err - BF16 * want.abs() - 1.01 * extra).max())


@pytest.mark.parametrize("T", [1, 2, 37, 700])
@pytest.mark.parametrize("Nq,Nkv,H", [(32, 8, 128), (1, 1, 64), (7, 1, 128), (5, 5, 64), (3, 2, 96), (4, 2, 80), (2, 1, 16), (4, 4, 256), (3, 3, 32)])
def test_norm_rope(Nq, Nkv, H, T):
    g = gen(T, Nq, Nkv, H)
    wide = (Nq + 2 * Nkv) * H + 8
    qkv = (rand(g, T, wide) * 3).bfloat16()[:, :wide - 8]  # strided rows
    f32 = T % 2 == 0
    qw, kw = ((1 + 0.3 * rand(g, H)).to(torch.float32 if f32 else torch.bfloat16) for _ in range(2))
    ep = table(900, H)
    pos = torch.randint(-2, 905, (T,), generator=g, device="cuda")
    q, k = P().qk_norm_rope(qkv, Nq, Nkv, H, qw, kw, 1e-5, ep, pos)
    x = qkv.reshape(T, -1, H)
    for got, part, w in ((q, x[:, :Nq], qw), (k, x[:, Nq:Nq + Nkv], kw)):
        close_rounded(got, *U.norm_rope(part, w, 1e-5, ep, pos))


@pytest.mark.parametrize("H,rot", [(128, 32), (128, 64), (64, 16), (96, 48), (256, 64)])
@pytest.mark.parametrize("normed", [True, False])
def test_partial_rotation_and_no_norm(H, rot, normed):
    g = gen(H, rot, normed)
    T, Nq, Nkv = 65, 3, 1
    qkv = rand(g, T, (Nq + 2 * Nkv) * H).bfloat16()
    w = rand(g, H) if normed else None
    ep, pos = table(70, rot), torch.arange(T, device="cuda")
    q, k = P().qk_norm_rope(qkv, Nq, Nkv, H, w, None, 1e-6, ep, pos)
    x = qkv.view(T, -1, H)
    close_rounded(q, *U.norm_rope(x[:, :Nq], w, 1e-6, ep, pos))
    close_rounded(k, *U.norm_rope(x[:, Nq:Nq + Nkv], None, 1e-6, ep, pos))
    q, k = P().qk_norm_rope(qkv, Nq, Nkv, H)  # nothing at all: the heads as they are
    assert torch.equal(q, x[:, :Nq]) and torch.equal(k, x[:, Nq:Nq + Nkv])


def test_norm_of_zero_rows_large_rows_and_nan_stays_in_its_head():
    H, Nq, Nkv = 128, 2, 1
    qkv = torch.ones(6, (Nq + 2 * Nkv) * H, device="cuda").bfloat16()
    qkv[0] = 0
    qkv[1, :H] = 2.0 ** 60
    qkv[2, 5] = math.nan
    qkv[3, H + 7] = math.inf
    q, k = P().qk_norm_rope(qkv, Nq, Nkv, H, torch.ones(H, device="cuda"), torch.ones(H, device="cuda"), 1e-6, None, None)
    assert not q[0].any() and not k[0].any()
    assert bool((q[1, 0] == 1).all())
    assert q[2, 0].isnan().all() and q[2, 1].isfinite().all() and k[2].isfinite().all()
    assert q[3, 0].isfinite().all() and not q[3, 1].isfinite().all()


def new_cache(lengths, new, Nkv, H, g, spare_columns=1, layers=1):
    need = [-(-(a + b) // 32) for a, b in zip(lengths, new)]
    cols, n = max(need) + spare_columns, sum(need) + 3
    cache = P().Int4Cache(layers, n, Nkv, H, len(lengths), cols)
    order = torch.randperm(n, generator=g, device="cuda").tolist()
    rows = []
    for k in need:
        rows.append([order.pop() for _ in range(k)] + [-1] * (cols - k))
    cache.table.copy_(torch.tensor(rows, dtype=torch.int32))
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    for pool in cache.pools:
        pool.fill_(255)  # every scale and minimum a NaN until it is written
    return cache


def cu_of(new, first=0):
    return torch.tensor([first] + new, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def sequence_heads(cache, b, tokens, layer=0):
    """codes, scales, minima of K and V of the first `tokens` tokens, [tokens, Nkv, H] each."""
    pages = cache.table[b, :-(-tokens // 32)].long()
    return [x.transpose(1, 2).flatten(0, 1)[:tokens] for x in U.unpack_heads(cache.pools[layer][pages])]


LENGTHS = [([0], [1]), ([31, 0, 64], [1, 1, 1]), ([0, 31, 32, 33, 5], [70, 1, 0, 31, 64]), ([0, 0, 0], [0, 33, 0]), ([1000], [200])]


@pytest.mark.parametrize("lengths,new", LENGTHS)
@pytest.mark.parametrize("Nkv,H", [(1, 128), (3, 64), (8, 128)])
def test_append_and_read(Nkv, H, lengths, new):
    g = gen(Nkv, H, *lengths, *new)
    cache = new_cache(lengths, new, Nkv, H, g)
    before = cache.pools[0].clone()
    T = sum(new) + 3  # a row in front of the first sequence, two behind the last
    k, v = ((rand(g, T, Nkv + 1, H) * torch.exp(rand(g, T, Nkv + 1, 1) * 3)).bfloat16()[:, :Nkv] for _ in range(2))
    cu = cu_of(new, 1)
    P().append_int4(k, v, cache, 0, cu)
    rk, rv = P().read_int4(cache, 0, T, cu)
    for b, (n, at) in enumerate(zip(new, cu.tolist())):
        heads = sequence_heads(cache, b, lengths[b] + n)
        for x, (c, s, z), r in ((k, heads[:3], rk), (v, heads[3:], rv)):
            wc, ws, wz = U.quantised(x[at:at + n])
            got = [t[lengths[b]:] for t in (c, s, z)]
            assert torch.equal(got[0], wc.flatten(-2))
            assert torch.equal(got[1].unflatten(-1, (-1, 64))[..., :1], ws) and torch.equal(got[2].unflatten(-1, (-1, 64))[..., :1], wz)
            close_rounded(r[at:at + n], (wz + wc * ws).flatten(-2), 2.0 ** -24 * (wz.abs() + wc * ws).flatten(-2))
        # nothing else of the sequence's pages changed: put the new places back
    again = cache.pools[0].clone()
    cache.pools[0].copy_(before)
    P().append_int4(k, v, cache, 0, cu)
    assert torch.equal(again, cache.pools[0])
    untouched = new_cache(lengths, new, Nkv, H, gen(Nkv, H, *lengths, *new))
    assert torch.equal(untouched.table, cache.table)
    for b, n in enumerate(new):  # old places still hold NaN parameters and codes of 15
        if lengths[b]:
            c, s, z, c2, s2, z2 = (t[:lengths[b]] for t in sequence_heads(cache, b, lengths[b]))
            assert bool((c == 15).all()) and bool((c2 == 15).all()) and s.isnan().all() and z2.isnan().all()


@pytest.mark.parametrize("Nq,Nkv,H,rot", [(8, 2, 128, 128), (3, 3, 64, 64), (4, 1, 128, 64), (2, 1, 128, 32)])
def test_norm_rope_appends_what_it_returns(Nq, Nkv, H, rot):
    lengths, new = [0, 40, 7], [33, 1, 0]
    g = gen(Nq, Nkv, H, rot)
    cache, other = (new_cache(lengths, new, Nkv, H, gen(1), layers=2) for _ in range(2))
    T, cu = sum(new), cu_of(new)
    qkv = rand(g, T, (Nq + 2 * Nkv) * H).bfloat16()
    w = (1 + 0.1 * rand(g, H)).bfloat16()
    ep = table(128, rot)
    q, k = P().qk_norm_rope(qkv, Nq, Nkv, H, w, w, 1e-6, ep, None, cu, cache, 1)
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(lengths, new)]).cuda()
    q2, k2 = P().qk_norm_rope(qkv, Nq, Nkv, H, w, w, 1e-6, ep, pos)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    P().append_int4(k, qkv.view(T, -1, H)[:, Nq + Nkv:], other, 1, cu)
    assert torch.equal(cache.pools[1], other.pools[1]) and bool((cache.pools[0] == 255).all())
    q3, k3 = P().qk_norm_rope(qkv, Nq, Nkv, H, w, w, 1e-6, ep, None, cu, other, 0, want_k=False)
    assert k3 is None and torch.equal(q3, q) and torch.equal(other.pools[0], cache.pools[1])
    assert cache.lengths.tolist() == lengths
    cache.advance(cu)
    assert cache.lengths.tolist() == [a + n for a, n in zip(lengths, new)]


def test_append_of_equal_tiny_huge_and_infinite_values():
    H = 64
    k = torch.zeros(8, 1, H, device="cuda").bfloat16()
    k[0] = 3.0
    k[1, 0, 0], k[1, 0, 1] = 2.0 ** -133, -(2.0 ** -133)   # the scale vanishes
    k[2, 0, ::2], k[2, 0, 1::2] = 3e38, -3e38              # the range passes the largest float
    k[3, 0, 5] = math.inf
    k[4, 0, 6] = math.nan
    k[5, 0, 7] = -math.inf
    k[6] = torch.arange(64, device="cuda").bfloat16() * 2.0 ** -130
    k[7, 0, :3] = torch.tensor([1.0, 2.0 ** -20, -2.0 ** -40])
    cache = new_cache([0], [8], 1, H, gen(3))
    P().append_int4(k, k.flip(0), cache, 0, cu_of([8]))
    c, s, z, c2, s2, z2 = sequence_heads(cache, 0, 8)
    for got, x in (((c, s, z), k), ((c2, s2, z2), k.flip(0))):
        wc, ws, wz = U.quantised(x)
        bad = ws.isnan()[..., 0, 0]
        assert torch.equal(got[1].isnan().all(-1), bad) and torch.equal(got[2].isnan().all(-1), bad)
        for a, b in zip(got, (wc.flatten(-2), ws.expand(-1, -1, -1, 64).flatten(-2), wz.expand(-1, -1, -1, 64).flatten(-2))):
            assert torch.equal(a[~bad], b[~bad])


def test_places_without_a_page_are_dropped():
    cache = new_cache([30, 0, 62], [6, 40, 6], 2, 64, gen(4), spare_columns=0)
    cache.table[0, 1], cache.table[1, 0], cache.table[1, 1] = -1, cache.pages, 1 << 30  # no pages
    cache.lengths[2] = 1 << 30                                                          # far behind the table
    before = cache.pools[0].clone()
    T, cu = 52, cu_of([6, 40, 6])
    k, v = (rand(gen(5), T, 2, 64).bfloat16() for _ in range(2))
    P().append_int4(k, v, cache, 0, cu)
    changed = (cache.pools[0] != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(cache.table[0, 0])]
    rk, rv = P().read_int4(cache, 0, T, cu)
    assert bool((rk[2:] == 0).all()) and bool((rv[2:] == 0).all()) and bool((rk[:2] != 0).any())
    out = P().attention_int4(rand(gen(6), T, 2, 64).bfloat16(), cache, 0, cu)
    assert not out[6:46].any()  # a sequence that has no page at all


# ---------------------------------------------------------------- attention over the cache

def fill(cache, g, old, new, mean=0.3):
    """Every place of the sequences gets codes, scales and minima of its own; places behind the last token stay NaN."""
    n, Nkv, H = cache.pages, cache.kv_heads, cache.head_dim
    codes = [torch.randint(0, 16, (n, Nkv, 32, H), generator=g, device="cuda") for _ in range(2)]
    scales = [(torch.exp(0.3 * rand(g, n, Nkv, 32, H // 64)) * 0.3).bfloat16() for _ in range(2)]
    minima = [(-7.5 * s.float() + mean * rand(g, n, Nkv, 32, H // 64)).bfloat16() for s in scales]
    for b, (a, k) in enumerate(zip(old, new)):
        m = a + k
        for i, page in enumerate(cache.table[b].tolist()):
            if page >= 0 and m < 32 * (i + 1):
                for t in scales + minima:
                    t[page, :, max(m - 32 * i, 0):] = math.nan
    cache.pools[0].copy_(U.pack_heads(codes, scales, minima))


def check_attention(cache, q, out, old, new, cu, causal, scale, rows=None):
    R = q.shape[1] // cache.kv_heads
    for b, (m, n) in enumerate(zip(old, new)):
        if n == 0 or (rows is not None and b not in rows):
            continue
        at = int(cu[b])
        kc, ks, kz, vc, vs, vz = sequence_heads(cache, b, m + n)
        x = q[at:at + n].double()
        want, w = U.attention(x, kz + kc * ks, vz + vc * vs, m, causal, scale)
        # scores: q as whole numbers of 2^-17 of its row's largest value or finer (half a step off at most, times a code of up to 15 and
        # its scale), then some ten roundings of sums and products in fp32
        size = torch.einsum("nhd,mhd->hnm", x.abs(), (kz.abs() + 15 * ks).repeat_interleave(R, 1)) * abs(scale)
        steps = x.abs().amax(-1).T[..., None] * (15 * ks).repeat_interleave(R, 1).sum(-1).T[:, None] * abs(scale)
        delta = (16 * 2.0 ** -24 * size + 2.0 ** -18 * steps).amax(-1)                 # [heads, n]
        rounded = torch.einsum("hnm,mhd->nhd", w, (vs * (vc - 8).abs()).repeat_interleave(R, 1))  # weights times scales are rounded
        plain = torch.einsum("hnm,mhd->nhd", w, (vz.abs() + 8 * vs + vs * vc).repeat_interleave(R, 1))
        # sums in fp32 over the keys, weights off by their scores' error and that of the exponential (2^-22)
        sums = (2 * delta + 2.0 ** -20 + 2.0 ** -23 * (m + n) / 16).T[..., None] * plain
        err = (out[at:at + n].double() - want).abs()
        limit = BF16 * want.abs() + 1.02 * BF16 * rounded + 2 * sums
        assert bool((err <= limit).all()), (b, m, n, float((err - limit).max()), float(err.max()))


SHAPES = [(32, 8, 128), (4, 4, 128), (7, 1, 128), (8, 1, 64), (12, 1, 128), (16, 1, 64), (20, 1, 128), (3, 3, 64)]


@pytest.mark.parametrize("old", [[0], [31], [32], [700, 0, 63], [5000, 17]])
@pytest.mark.parametrize("Nq,Nkv,H", SHAPES)
def test_one_token(Nq, Nkv, H, old):
    g = gen(Nq, Nkv, H, *old)
    new = [1] * len(old)
    cache = new_cache(old, new, Nkv, H, g)
    fill(cache, g, old, new)
    wide = rand(g, len(old), Nq * H + 16).bfloat16() * 2
    q = wide[:, :Nq * H].unflatten(1, (Nq, H))  # strided rows
    out = P().attention_int4(q, cache, 0)
    check_attention(cache, q, out, old, new, range(len(old)), True, H ** -0.5)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("old,new", [([40, 0, 33], [2, 5, 9]), ([0, 0], [64, 1]), ([300, 7, 0, 90], [0, 17, 3, 1]), ([2000], [33])])
@pytest.mark.parametrize("Nq,Nkv,H", [(32, 8, 128), (2, 2, 64), (7, 1, 128), (16, 1, 64)])
def test_several_tokens(Nq, Nkv, H, old, new, causal):
    g = gen(Nq, Nkv, H, *old, *new)
    cache = new_cache(old, new, Nkv, H, g)
    fill(cache, g, old, new)
    T, cu = sum(new) + 5, cu_of(new, 2)
    q = rand(g, T, Nq, H).bfloat16()
    out = torch.full_like(q, 7.0)
    got = P().attention_int4(q, cache, 0, cu, causal, 0.11, out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[:2] == 7).all()) and bool((out[T - 3:] == 7).all())  # rows of no sequence
    check_attention(cache, q, out, old, new, cu, causal, 0.11)


def test_many_ragged_sequences():
    g = gen(9)
    old = [(i * i * 7) % 901 for i in range(300)]
    new = [1] * 300
    cache = new_cache(old, new, 2, 64, g)
    fill(cache, g, old, new)
    q = rand(g, 300, 8, 64).bfloat16()
    check_attention(cache, q, P().attention_int4(q, cache, 0), old, new, range(300), True, 0.125, set(range(0, 300, 7)))


@pytest.mark.parametrize("grow", [2.0 ** 4, 2.0 ** 10, 2.0 ** -20, 0.0])
def test_scores_of_any_size(grow):
    """Scores far apart, tiny ones and equal ones: the largest may come first or last, in any warp's keys."""
    g = gen(11)
    old, new = [1500, 64], [1, 1]
    cache = new_cache(old, new, 1, 128, g)
    fill(cache, g, old, new)
    q = (rand(g, 2, 4, 128) * grow).bfloat16()
    check_attention(cache, q, P().attention_int4(q, cache, 0), old, new, range(2), True, 128 ** -0.5)


def test_nan_and_infinity_reach_those_who_see_them():
    g = gen(12)
    old, new = [70, 70], [3, 3]
    cache = new_cache(old, new, 1, 64, g)
    k, v = (rand(g, 73, 1, 64).bfloat16() for _ in range(2))
    start = cache.lengths.clone()
    cache.lengths.zero_()
    two = lambda t: torch.cat([t, t])  # noqa: E731
    k[72, 0, 3], v[71, 0, 5] = math.nan, math.inf     # of the call's last two tokens
    P().append_int4(two(k), two(v), cache, 0, cu_of([73, 73]))
    cache.lengths.copy_(start)
    out = P().attention_int4(two(rand(g, 3, 2, 64).bfloat16()), cache, 0, cu_of(new))
    for b in range(2):
        assert out[3 * b].isfinite().all()                                    # sees neither
        assert out[3 * b + 1].isnan().all() and out[3 * b + 2].isnan().all()  # the infinity; the NaN too


@pytest.mark.parametrize("old", [[0, 40], [5000, 0], [20000, 3], [3] * 300])
@pytest.mark.parametrize("what", ["query", "keys"])
def test_scores_that_are_all_nan_give_nan(what, old):
    """A row whose every score is a NaN has no largest score, but it is not a row without keys: by one warp, a block and many blocks."""
    g, H = gen(23, len(old), old[0]), 64
    n = len(old)
    cache = new_cache(old, [1] * n, 2, H, g)
    k, v = (rand(g, sum(old) + n, 2, H).bfloat16() for _ in range(2))
    q = rand(g, n, 4, H).bfloat16()
    cu = cu_of([m + 1 for m in old])
    if what == "query":
        q[0, 1, 7] = math.nan
    else:
        k[:int(cu[1]), 0] = math.nan
    start = cache.lengths.clone()
    cache.lengths.zero_()
    P().append_int4(k, v, cache, 0, cu)
    cache.lengths.copy_(start)
    out = P().attention_int4(q, cache, 0)
    bad = torch.zeros((n, 4), dtype=torch.bool, device="cuda")
    bad[0, 1 if what == "query" else slice(0, 2)] = True
    assert torch.equal(out.isnan().all(-1), bad) and bool(out[~bad].isfinite().all())


def test_offsets_behind_two_gigabytes():
    old, new, H = [100, 40], [1, 1], 128
    pages = 2 ** 31 // 4608 + 40
    pool = torch.empty((pages, 1, 36 * H), dtype=torch.uint8, device="cuda")
    tab = torch.tensor([[pages - 1, pages - 5, pages - 2, pages - 9], [3, pages - 30, -1, -1]], dtype=torch.int32, device="cuda")
    big = P().Int4Cache.over([pool], tab, torch.tensor(old, dtype=torch.int32, device="cuda"))
    g = gen(13)
    k, v = (rand(g, 142, 1, H).bfloat16() for _ in range(2))
    big.lengths.zero_()
    P().append_int4(k, v, big, 0, cu_of([101, 41]))
    rk, _ = P().read_int4(big, 0, 142, cu_of([101, 41]))
    close_rounded(rk, U.quantised_values(k), 2.0 ** -20 * k.double().abs().amax())
    big.lengths.copy_(torch.tensor(old, dtype=torch.int32))
    q = rand(g, 2, 4, H).bfloat16()
    check_attention(big, q, P().attention_int4(q, big, 0), old, new, range(2), True, H ** -0.5)


def test_two_streams_and_two_graphs_at_once():
    """Calls that run at the same time share nothing; a replayed one reads the lengths of its replay."""
    g = gen(14)
    old, new = [3000, 900, 50], [1, 1, 1]
    caches, qs, want = [], [], []
    for i in range(2):
        c = new_cache([x + 64 for x in old], new, 2, 128, g)
        fill(c, g, [x + 64 for x in old], new)
        c.lengths.copy_(torch.tensor(old, dtype=torch.int32))
        caches.append(c)
        qs.append(rand(g, 3, 8, 128).bfloat16())
        want.append(P().attention_int4(qs[i], c, 0))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append([P().attention_int4(qs[i], caches[i], 0) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(P().attention_int4(qs[i], caches[i], 0))
        graphs.append(gr)
    for step in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            check_attention(caches[i], qs[i], outs[i], [x + step for x in old], new, range(3), True, 128 ** -0.5)
            caches[i].lengths.add_(1)
        torch.cuda.synchronize()


def test_one_result_whatever_the_order_of_arrival():
    g = gen(15)
    old, new = [20000, 3, 7000], [1, 1, 1]
    cache = new_cache(old, new, 4, 64, g)
    fill(cache, g, old, new)
    q = rand(g, 3, 8, 64).bfloat16()
    first = P().attention_int4(q, cache, 0)
    assert all(torch.equal(first, P().attention_int4(q, cache, 0)) for _ in range(30))


def test_empty_calls():
    cache = new_cache([4, 5], [0, 0], 1, 64, gen(16))
    cu = cu_of([0, 0])
    none = torch.empty(0, 1, 64, device="cuda", dtype=torch.bfloat16)
    P().append_int4(none, none, cache, 0, cu)
    assert P().attention_int4(none, cache, 0, cu).shape == (0, 1, 64)
    assert P().read_int4(cache, 0, 0, cu)[0].shape == (0, 1, 64)
    q, k = P().qk_norm_rope(torch.empty(0, 3 * 64, device="cuda", dtype=torch.bfloat16), 1, 1, 64)
    assert q.shape == (0, 1, 64)


def test_refused_tensors():
    """What the host sees of a call that cannot work: none of these launches anything."""
    from tpp_pytorch_extension_b200._lib import TpxError
    g, old = gen(31), [40, 0]
    cache = new_cache(old, [1, 1], 2, 64, g)
    qkv = rand(g, 2, 8 * 64).bfloat16()
    q, k = qkv[:, :256].contiguous().view(2, 4, 64), qkv[:, 256:384].contiguous().view(2, 2, 64)
    ep = table(64, 64)
    prep = lambda x=qkv, **kw: P().qk_norm_rope(x, 4, 2, 64, ep=ep, cache=cache, **kw)  # noqa: E731
    cu = cu_of([1, 1])
    refused = [
        lambda: prep(qkv.cpu()), lambda: prep(qkv.float()), lambda: prep(qkv[:, :448]), lambda: prep(qkv[:1]), lambda: prep(qkv.clone().requires_grad_()),
        lambda: prep(q_out=qkv[:, :256].view(2, 4, 64)), lambda: prep(q_out=torch.empty_like(q).float()), lambda: prep(q_out=torch.empty_like(k)),
        lambda: prep(q_out=qkv.view(-1)[:512].view(2, 4, 64)), lambda: prep(q_out=q, k_out=q.view(-1)[:256].view(2, 2, 64)),
        lambda: prep(positions=torch.zeros(2, dtype=torch.int32, device="cuda")), lambda: prep(positions=torch.zeros(3, dtype=torch.int64, device="cuda")),
        lambda: prep(q_norm=torch.ones(64, device="cuda"), k_norm=torch.ones(64, device="cuda").bfloat16()), lambda: prep(q_norm=torch.ones(32, device="cuda")),
        lambda: prep(cu_seqlens=cu.long()), lambda: prep(cu_seqlens=cu[:2]),
        lambda: P().qk_norm_rope(qkv, 4, 2, 64, ep=ep), lambda: P().qk_norm_rope(qkv, 4, 2, 64, cu_seqlens=cu),
        lambda: P().qk_norm_rope(qkv, 8, 4, 32, cache=cache), lambda: P().qk_norm_rope(qkv, 2, 3, 64, cache=cache),
        lambda: P().append_int4(k, k[:1], cache, 0), lambda: P().append_int4(k[:, :1], k[:, :1], cache, 0), lambda: P().append_int4(k.float(), k.float(), cache, 0),
        lambda: P().append_int4(k.transpose(0, 1), k.transpose(0, 1), cache, 0), lambda: P().append_int4(k[:1], k[:1], cache, 0),
        lambda: P().read_int4(cache, 0, 3), lambda: P().read_int4(cache, 0, 2, lengths=cu), lambda: P().read_int4(cache, 0, -1),
        lambda: P().attention_int4(q[:, :3], cache, 0), lambda: P().attention_int4(q[:1], cache, 0), lambda: P().attention_int4(q.float(), cache, 0),
        lambda: P().attention_int4(q, cache, 0, scale=math.inf), lambda: P().attention_int4(q, cache, 0, scale=math.nan),
        lambda: P().attention_int4(q, cache, 0, out=q), lambda: P().attention_int4(q, cache, 0, out=cache.pools[0].view(-1)[:1024].view(torch.bfloat16).view(2, 4, 64)),
        lambda: P().attention_int4(q.expand(2, 4, 64)[:, :, ::2], cache, 0), lambda: P().attention_int4(q.detach().requires_grad_(), cache, 0),
    ]
    before = cache.pools[0].clone()
    for i, call in enumerate(refused):
        with pytest.raises(TpxError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert torch.equal(before, cache.pools[0])
    with torch.no_grad():  # leaves that want a gradient may be used where none is recorded
        P().attention_int4(q.clone().requires_grad_(), cache, 0)
