"""Attention over the 4-bit cache for every way in which its blocks share the work: warps with segments of their own, groups of four warps, whole
blocks; segments that are cut between them and joined by who is last. A segment is a key head of a sequence, 4, 8 or 16 query rows at a time."""
import math

import pytest
import torch

from tests import test_gpu_packed_cache as C

pytestmark = pytest.mark.gpu


def arrangement(old, new, Nq, Nkv):
    """Warps that work on a segment together, and whether it is dealt in pieces of four quanta, as the kernel's rule has it."""
    sms, R, B = torch.cuda.get_device_properties(0).multi_processor_count, Nq // Nkv, len(old)
    per = -(-sum(new) // B) * R
    rows = 4 if per <= 4 else 8 if per <= 8 else 16
    warps = 8 if rows == 16 else 16
    segments = [(-(-n * R // rows) * Nkv, -(-(m + n) // 32)) for m, n in zip(old, new)]
    even = -(-sum(s * p for s, p in segments) // (sms * warps))
    most = max(p for s, p in segments)
    wide = warps if sum(s for s, _ in segments) < sms else 1 if most <= 8 * even else 4 if most <= 64 * even else warps
    quanta = [(s, -(-p // wide)) for s, p in segments]
    pieces = sum(s * -(-q // 4) for s, q in quanta)
    workers = sms * warps // wide
    few = pieces <= workers
    units = pieces if few else sum(s * (q + 2) for s, q in quanta)
    cut = any((-(-q // 4) if few else q + 2) > 1 for s, q in quanta) and units > workers or few and any(q > 4 for _, q in quanta)
    return wide if wide < warps else "block", few, cut


def spread(n, lo, hi, *long):
    """n lengths between lo and hi, the given ones among them."""
    x = [lo + (i * i * 37 + 11 * i) % (hi - lo + 1) for i in range(n)]
    for i, m in enumerate(long):
        x[(i * 29 + 13) % n] = m
    return x


CASES = [  # lengths, key heads, warps per segment, pieces
    (spread(100, 140, 255), 2, 1, True),
    (spread(100, 33, 200, 1900), 2, 4, True),
    (spread(100, 0, 60, 3300), 2, "block", False),
    (spread(64, 1000, 1999), 8, 1, False),
    (spread(64, 40, 1800, 4095, 3000), 8, 4, False),
    (spread(300, 0, 50, 13000), 8, "block", False),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("H", [64, 128])
@pytest.mark.parametrize("R", [4, 7, 16])
def test_one_token_of_many_sequences(R, H, case):
    old, Nkv, wide, few = CASES[case]
    new, Nq, g = [1] * len(old), R * Nkv, C.gen(81, R, H, case)
    assert arrangement(old, new, Nq, Nkv)[:2] == (wide, few)
    cache = C.new_cache(old, new, Nkv, H, g)
    C.fill(cache, g, old, new)
    q = C.rand(g, len(old), Nq, H).bfloat16()
    out = C.P().attention_int4(q, cache, 0)
    longest = {i for i, m in enumerate(old) if m >= sorted(old)[-8]}
    C.check_attention(cache, q, out, old, new, range(len(old)), True, H ** -0.5, longest | set(range(0, len(old), max(1, len(old) // 64))))
    for _ in range(10):
        assert torch.equal(out, C.P().attention_int4(q, cache, 0))


@pytest.mark.parametrize("H", [64, 128])
@pytest.mark.parametrize("R,most,wide", [(1, 3, 1), (2, 5, 1), (4, 9, 1), (4, 9, 4), (1, 3, 4), (2, 5, "block")])
def test_several_tokens_of_many_sequences(R, most, wide, H):
    """Sequences of no token, of one and of several, so that some have more row chunks than others."""
    g, Nkv = C.gen(82, R, H, most), 3
    old = spread(90, 100, 240) if wide == 1 else spread(90, 20, 140, 2000) if wide == 4 else spread(90, 0, 20, 5000)
    new = [(i * 7) % (most + 1) for i in range(90)]
    new[13] = most
    Nq = R * Nkv
    assert arrangement(old, new, Nq, Nkv)[0] == wide
    cache = C.new_cache(old, new, Nkv, H, g)
    C.fill(cache, g, old, new)
    T, cu = sum(new) + 3, C.cu_of(new, 1)
    q = C.rand(g, T, Nq, H).bfloat16()
    for causal in (True, False):
        out = torch.full_like(q, 3.0)
        C.P().attention_int4(q, cache, 0, cu, causal, 1 / math.sqrt(H), out)
        assert bool((out[:1] == 3).all()) and bool((out[T - 2:] == 3).all())
        C.check_attention(cache, q, out, old, new, cu, causal, 1 / math.sqrt(H))
        again = torch.full_like(q, 3.0)
        for _ in range(5):
            assert torch.equal(out, C.P().attention_int4(q, cache, 0, cu, causal, 1 / math.sqrt(H), again))
