"""Calls of two host threads at once, and pages that several sequences read."""
import threading

import pytest
import torch

from tests import packed_util as U
from tests import test_gpu_packed_cache as C
from tests import test_gpu_packed_prompts as S

pytestmark = pytest.mark.gpu


def test_two_host_threads():
    """Each on its own stream and cache: append, read back, both attentions, over and over."""
    P, problems = C.P(), []
    start = torch.cuda.Event()
    start.record()

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                g = C.gen(121, seed)
                old, new = [900, 40 + seed, 0], [3, 1, 70]
                cache = C.new_cache(old, new, 2, 128, g)
                C.fill(cache, g, old, new)
                cu = C.cu_of(new)
                q, k, v = S.inputs(g, sum(new), 8, 2, 128)
                first = None
                for _ in range(50):
                    P.append_int4(k, v, cache, 0, cu)
                    got = [P.attention_int4(q, cache, 0, cu), P.attention_packed(q, k, v, cu), *P.read_int4(cache, 0, sum(new), cu)]
                    first = first or got
                    assert all(torch.equal(a, b) for a, b in zip(first, got))
                C.check_attention(cache, q, first[0], old, new, cu, True, 128 ** -0.5)
                S.check(q, k, v, first[1], new, cu)
                C.close_rounded(first[2], U.quantised_values(k), 2.0 ** -22 * k.double().abs().amax())
        except BaseException as e:
            problems.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not problems, problems[0]


@pytest.mark.parametrize("Nq,Nkv,H", [(8, 2, 128), (4, 4, 64)])
def test_a_prefix_that_sequences_share(Nq, Nkv, H):
    """The first pages of three sequences are the same ones; their last pages are their own."""
    g, old, new = C.gen(122, H), [320 + 5, 320, 320 + 31], [1, 1, 1]
    cache = C.new_cache(old, new, Nkv, H, g)
    cache.table[1:, :10] = cache.table[0, :10]
    C.fill(cache, g, old, new)
    q = C.rand(g, 3, Nq, H).bfloat16()
    shared = cache.pools[0][cache.table[0, :10].long()].clone()
    k, v = (C.rand(g, 3, Nkv, H).bfloat16() for _ in range(2))
    C.P().append_int4(k, v, cache, 0)
    assert torch.equal(cache.pools[0][cache.table[0, :10].long()], shared)
    C.check_attention(cache, q, C.P().attention_int4(q, cache, 0), old, new, range(3), True, H ** -0.5)
