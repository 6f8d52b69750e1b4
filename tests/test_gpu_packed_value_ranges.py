"""Attention over the 4-bit cache where values differ in size by many powers of two: the groups of a head, the tokens of a sequence, and the
rows that look at them. What a row takes from a group is as exact as that group's own values allow."""
import pytest
import torch

from tests import test_gpu_packed_cache as C
from tests import packed_util as U

pytestmark = pytest.mark.gpu


def filled(g, old, new, Nkv, H, change):
    """A cache whose scales and minima of values `change(page, scale, minimum)` has had its way with, fp32 [kv heads, 32, H / 64]."""
    cache = C.new_cache(old, new, Nkv, H, g)
    C.fill(cache, g, old, new)
    c, s, z, c2, s2, z2 = U.unpack_heads(cache.pools[0])
    s, z, s2, z2 = (t[..., ::64].float() for t in (s, z, s2, z2))
    s2, z2 = change(s2, z2)
    cache.pools[0].copy_(U.pack_heads((c, c2), (s, s2), (z, z2)))
    return cache


@pytest.mark.parametrize("ratio", [-10, -20, -24, -28, -45, -90, 24, 60])
@pytest.mark.parametrize("Nq,Nkv", [(4, 1), (8, 1), (16, 1), (7, 1), (8, 2)])
@pytest.mark.parametrize("old", [[4095], [40, 700, 3]])
def test_groups_of_different_sizes(old, Nq, Nkv, ratio):
    """One group of 64 values of a head is 2^ratio times as large as the other."""
    g, new = C.gen(71, ratio + 100, Nq, *old), [1] * len(old)
    factor = torch.tensor([1.0, 2.0 ** ratio], device="cuda")
    cache = filled(g, old, new, Nkv, 128, lambda s, z: (s * factor, z * factor))
    for grow in (0.0, 1.0, 4.0):  # even weights, ordinary ones, much of them on a few keys
        q = (C.rand(g, len(old), Nq, 128) * grow).bfloat16()
        C.check_attention(cache, q, P().attention_int4(q, cache, 0), old, new, range(len(old)), True, 128 ** -0.5)


def P():
    return C.P()


@pytest.mark.parametrize("H,Nq", [(64, 4), (64, 8), (64, 16), (128, 4), (128, 8), (128, 16)])
@pytest.mark.parametrize("at", [0, 9, 500, 1499])
@pytest.mark.parametrize("ratio", [12, 24, 40])
def test_one_large_token_that_half_of_the_rows_leave_alone(ratio, at, H, Nq):
    """Values of one token are 2^ratio times as large as the others'. Its key is one number in all places, so rows whose query is positive give it
    next to no weight, rows with the sign turned give it nearly all of theirs."""
    g, old, new = C.gen(72, ratio, at, H, Nq), [1500, 33], [1, 1]
    cache = filled(g, old, new, 1, H, lambda s, z: (s, z))
    c, s, z, c2, s2, z2 = U.unpack_heads(cache.pools[0])
    s, z, s2, z2 = (t[..., ::64].float() for t in (s, z, s2, z2))
    page, t = int(cache.table[0, at // 32]), at % 32
    s[page, :, t], z[page, :, t] = 0.0, -4.0
    s2[page, :, t] *= 2.0 ** ratio
    z2[page, :, t] *= 2.0 ** ratio
    cache.pools[0].copy_(U.pack_heads((c, c2), (s, s2), (z, z2)))
    q = C.rand(g, 2, Nq, H).abs() * 1.5
    q[:, ::2] *= -1
    q = q.bfloat16()
    scale = H ** -0.5
    x, n = q[0, 1].double(), old[0] + 1
    kc, ks, kz = C.sequence_heads(cache, 0, n)[:3]
    _, w = U.attention(q[:1].double(), kz + kc * ks, torch.zeros_like(kz), old[0], True, scale)
    assert float(w[1, 0, at]) < 2.0 ** (-ratio / 2) and float(w[0, 0, at]) > 0.5 and x.sum() > 0
    C.check_attention(cache, q, P().attention_int4(q, cache, 0), old, new, range(2), True, scale)


@pytest.mark.parametrize("H", [64, 128])
@pytest.mark.parametrize("step", [2.0, -2.0, 0.25])
def test_values_that_grow_and_shrink_along_the_sequence(H, step):
    """Every page's values are 2^step times those of the page in front, scores likewise in either direction."""
    g, old, new = C.gen(73, H, int(8 * step + 99)), [1200, 31], [1, 1]
    cache = C.new_cache(old, new, 2, H, g)
    C.fill(cache, g, old, new)
    c, s, z, c2, s2, z2 = U.unpack_heads(cache.pools[0])
    s, z, s2, z2 = (t[..., ::64].float() for t in (s, z, s2, z2))
    for i, page in enumerate(cache.table[0].tolist()):
        if page >= 0:
            s2[page] *= 2.0 ** (step * (i - 19))
            z2[page] *= 2.0 ** (step * (i - 19))
    cache.pools[0].copy_(U.pack_heads((c, c2), (s, s2), (z, z2)))
    for grow in (0.25, 4.0, 16.0):
        q = (C.rand(g, 2, 8, H) * grow).bfloat16()
        C.check_attention(cache, q, P().attention_int4(q, cache, 0), old, new, range(2), True, H ** -0.5)


@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** 40, 2.0 ** -60, 2.0 ** -100])
def test_values_of_any_size(size):
    g, old, new = C.gen(74), [700, 2], [1, 1]
    cache = filled(g, old, new, 2, 128, lambda s, z: (s * size, z * size))
    q = C.rand(g, 2, 8, 128).bfloat16()
    C.check_attention(cache, q, P().attention_int4(q, cache, 0), old, new, range(2), True, 128 ** -0.5)
