"""Head norms with rotation, the append and the read-back on either side of the number of tokens from which resident warps walk them, and what the
append leaves alone: the whole pool against one that is put together from the definition."""
import pytest
import torch

from tests import packed_util as U
from tests import test_gpu_packed_cache as C

pytestmark = pytest.mark.gpu


def tokens(heads, H, beyond):
    """The least number of tokens that gives every resident warp an item, or one less."""
    lanes = 1 if H <= 16 else 2 if H <= 32 else 4 if H <= 64 else 8 if H <= 128 else 16
    each = heads * lanes
    return -(-torch.cuda.get_device_properties(0).multi_processor_count * 2048 // each) - (0 if beyond else 1)


@pytest.mark.parametrize("beyond", [False, True])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("Nq,Nkv,H,rot", [(32, 8, 128, 128), (33, 3, 128, 64), (7, 1, 128, 32), (5, 5, 64, 64), (18, 2, 64, 16), (3, 2, 96, 96), (4, 2, 80, 48),
                                         (2, 1, 16, 16), (4, 4, 256, 256), (9, 1, 256, 64), (3, 3, 32, 32), (16, 0, 64, 32)])
def test_norm_rope(Nq, Nkv, H, rot, normed, beyond):
    T = tokens(Nq + Nkv, H, beyond) + (37 if beyond else 0)
    g = C.gen(T, Nq, H, rot, normed)
    wide = (Nq + 2 * Nkv) * H + 24
    qkv = (C.rand(g, T, wide) * 2).bfloat16()[:, :wide - 24]  # strided rows
    ws = [(1 + 0.3 * C.rand(g, H)).to(torch.bfloat16 if rot == H else torch.float32) for _ in range(2)] if normed else [None, None]
    ep, pos = C.table(900, rot), torch.randint(-3, 905, (T,), generator=g, device="cuda")
    q, k = C.P().qk_norm_rope(qkv, Nq, Nkv, H, ws[0], ws[1], 1e-5, ep, pos)
    x = qkv.reshape(T, -1, H)
    C.close_rounded(q, *U.norm_rope(x[:, :Nq], ws[0], 1e-5, ep, pos))
    C.close_rounded(k, *U.norm_rope(x[:, Nq:Nq + Nkv], ws[1], 1e-5, ep, pos)) if Nkv else None
    q2, _ = C.P().qk_norm_rope(qkv, Nq, Nkv, H, ws[0], ws[1], 1e-5)  # norms alone
    C.close_rounded(q2, *U.norm_rope(x[:, :Nq], ws[0], 1e-5, None, None))


def expected_pool(before, cache, old, new, cu, k, v):
    """The bytes of the pool with the call's keys and values in their places: a mask of the nibbles and parameters that are theirs, and what they become."""
    n, Nkv, H = before.shape[0], before.shape[1], before.shape[2] // 36
    codes, mask = ([torch.zeros(n, Nkv, 32, H, device="cuda") for _ in range(2)] for _ in range(2))
    scales, minima, whole = ([torch.zeros(n, Nkv, 32, H // 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)] for _ in range(3))
    at = torch.cat([torch.arange(int(c), int(c) + b) for c, b in zip(cu.tolist(), new)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    place = torch.cat([torch.arange(a, a + b) for a, b in zip(old, new)]).cuda()
    page, t = cache.table[seq, place // 32].long(), place % 32
    for i, x in enumerate((k, v)):
        c, s, z = U.quantised(x[at])
        codes[i][page, :, t], mask[i][page, :, t] = c.flatten(-2).float(), 15.0
        scales[i][page, :, t], minima[i][page, :, t] = s[..., 0].bfloat16(), z[..., 0].bfloat16()
        whole[i].view(torch.int16)[page, :, t] = -1
    value, own = U.pack_heads(codes, scales, minima), U.pack_heads(mask, whole, whole)
    return before & ~own | value & own


CALLS = [([0], [1]), ([31, 0, 64], [1, 1, 1]), ([0, 31, 32, 33, 5], [70, 1, 0, 31, 64]), ([1000], [200]),
         ([0, 9, 600, 32, 0, 64], [2000, 1, 900, 0, 33, 1700]), ([77, 31], [3, 9000])]


@pytest.mark.parametrize("old,new", CALLS)
@pytest.mark.parametrize("Nq,Nkv,H,rot", [(32, 8, 128, 128), (5, 5, 64, 64), (7, 1, 128, 64), (0, 3, 64, 0), (6, 3, 128, 0)])
def test_the_append_writes_its_places_and_nothing_else(Nq, Nkv, H, rot, old, new):
    g = C.gen(111, Nq, H, *old, *new)
    cache = C.new_cache(old, new, Nkv, H, g, layers=2)
    for pool in cache.pools:
        pool.copy_(torch.randint(0, 256, pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    before = [p.clone() for p in cache.pools]
    T, cu = sum(new) + 5, C.cu_of(new, 2)  # two rows in front, three behind
    qkv = C.rand(g, T, (Nq + 2 * Nkv) * H).bfloat16()
    x = qkv.view(T, -1, H)
    if Nq:
        w, ep = 1 + 0.1 * C.rand(g, H), C.table(700, rot) if rot else None  # the last places lie behind the table
        q, k = torch.full((T, Nq, H), 4.0, device="cuda").bfloat16(), torch.full((T, Nkv, H), 4.0, device="cuda").bfloat16()
        C.P().qk_norm_rope(qkv, Nq, Nkv, H, w, w, 1e-6, ep, None, cu, cache, 1, q_out=q, k_out=k)
        inside = torch.zeros(T, dtype=torch.bool, device="cuda")
        inside[2:T - 3] = True
        assert bool((q[~inside] == 4).all()) and bool((k[~inside] == 4).all())
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(old, new)]).cuda()
        C.close_rounded(q[inside], *U.norm_rope(x[inside, :Nq], w, 1e-6, ep, pos))
        C.close_rounded(k[inside], *U.norm_rope(x[inside, Nq:Nq + Nkv], w, 1e-6, ep, pos))
    else:
        k = x[:, :Nkv]
        C.P().append_int4(k, x[:, Nkv:], cache, 1, cu)
    v = x[:, Nq + Nkv:]
    assert torch.equal(cache.pools[0], before[0])
    want = expected_pool(before[1], cache, old, new, cu, k, v)
    assert torch.equal(cache.pools[1], want)
    rk, rv = C.P().read_int4(cache, 1, T, cu)
    for got, src in ((rk, k), (rv, v)):
        c, s, z = U.quantised(src[2:T - 3])
        C.close_rounded(got[2:T - 3], (z + c * s).flatten(-2), 2.0 ** -24 * (z.abs() + c * s).flatten(-2))


@pytest.mark.parametrize("beyond", [False, True])
@pytest.mark.parametrize("Nkv,H", [(1, 64), (8, 128), (5, 128), (6, 64), (2, 128)])
def test_read_back(Nkv, H, beyond):
    """Heads that four per thread do and do not divide, sequences without pages, rows of no sequence."""
    T = -(-torch.cuda.get_device_properties(0).multi_processor_count * 2048 // (Nkv * (H // 8))) - (0 if beyond else 1)
    new = [T // 2, 0, T // 3, 5]
    new.append(T - 3 - sum(new))
    old = [0, 3, 40, 31, 7]
    g = C.gen(112, T, Nkv, H)
    cache = C.new_cache(old, new, Nkv, H, g)
    cu = C.cu_of(new, 3)
    k, v = (C.rand(g, T, Nkv, H).bfloat16() for _ in range(2))
    C.P().append_int4(k, v, cache, 0, cu)
    cache.table[3].fill_(-1)
    rk, rv = C.P().read_int4(cache, 0, T, cu)
    at = cu.tolist()
    for got, src in ((rk, k), (rv, v)):
        c, s, z = U.quantised(src)
        want, off = (z + c * s).flatten(-2), 2.0 ** -24 * (z.abs() + c * s).flatten(-2)
        want[at[3]:at[4]], off[at[3]:at[4]] = 0, 0
        C.close_rounded(got[3:], want[3:], off[3:])


def test_what_is_not_finite_among_many_tokens():
    """Codes and parameters of rows of every kind, by the resident warps: equal, tiny, huge, infinite and NaN."""
    H, Nkv, n = 64, 4, 12000
    assert n > tokens(2 * Nkv, H, True)
    g = C.gen(113)
    k = C.rand(g, n, Nkv, H).bfloat16()
    k[5], k[6, :, ::2], k[6, :, 1::2] = 3.0, 3e38, -3e38
    k[7, 1, 5], k[8, 2, 6], k[9, 3, 7] = float("inf"), float("nan"), float("-inf")
    k[10] = torch.arange(64, device="cuda").bfloat16() * 2.0 ** -130
    cache = C.new_cache([0], [n], Nkv, H, g)
    C.P().append_int4(k, k.flip(0), cache, 0, C.cu_of([n]))
    heads = C.sequence_heads(cache, 0, n)
    for got, x in ((heads[:3], k), (heads[3:], k.flip(0))):
        wc, ws, wz = (t.expand(-1, -1, -1, 64).flatten(-2) for t in U.quantised(x))
        bad = ws.isnan()
        assert torch.equal(got[1].isnan(), bad) and torch.equal(got[2].isnan(), bad)
        for a, b in zip(got, (wc, ws, wz)):
            assert torch.equal(a[~bad], b[~bad])
