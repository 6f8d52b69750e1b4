"""A slot of the 4-bit cache that is released and taken by the next prompt while the other sequences decode, step by step and from a recorded step."""
import pytest
import torch

from tests import packed_util as U
from tests import test_gpu_packed_cache as C

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [False, True])
def test_a_released_slot_is_taken_by_the_next_prompt(recorded):
    P, g = C.P(), C.gen(91, recorded)
    Nq, Nkv, H, B = 8, 2, 64, 3
    cache = P.Int4Cache(1, 20, Nkv, H, B, 5)
    said = [[], [], []]  # keys and values of each sequence, bf16 [tokens, Nkv, H]
    row = torch.zeros(B, (Nq + 2 * Nkv) * H, device="cuda", dtype=torch.bfloat16)

    def prompts(new):
        qkv = C.rand(g, sum(new), (Nq + 2 * Nkv) * H).bfloat16()
        cu = C.cu_of(new)
        P.qk_norm_rope(qkv, Nq, Nkv, H, cu_seqlens=cu, cache=cache)
        cache.advance(cu)
        for b, part in enumerate(qkv.view(-1, Nq + 2 * Nkv, H)[:, Nq:].split(new)):
            said[b] += list(part)

    def work():
        q, _ = P.qk_norm_rope(row, Nq, Nkv, H, cache=cache, want_k=False)
        out = P.attention_int4(q, cache, 0)
        cache.advance()
        return out

    def step(live, graph, out):
        row.copy_(C.rand(g, *row.shape))
        old = [len(x) for x in said]
        graph.replay() if graph else out.copy_(work())
        x = row.view(B, -1, H)
        for b in live:
            said[b].append(x[b, Nq:].clone())
        assert cache.lengths.tolist() == [len(x) for x in said]
        before = cache.lengths.clone()
        cache.lengths.copy_(torch.tensor(old, dtype=torch.int32))  # what the attention of the step saw
        C.check_attention(cache, x[:, :Nq], out, old, [int(b in live) for b in range(B)], range(B), True, H ** -0.5)
        cache.lengths.copy_(before)
        assert not any(out[b].any() for b in range(B) if b not in live)

    cache.add_pages([100, 90, 100])
    prompts([40, 64, 3])
    graph, out = None, torch.empty(B, Nq, H, device="cuda", dtype=torch.bfloat16)
    if recorded:
        work()
        cache.lengths.copy_(torch.tensor([40, 64, 3], dtype=torch.int32))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
    for _ in range(3):
        step([0, 1, 2], graph, out)
    cache.release(1)
    said[1].clear()
    for _ in range(5):
        step([0, 2], graph, out)
    cache.add_pages([100, 45, 100])
    prompts([0, 40, 0])
    for _ in range(4):
        step([0, 1, 2], graph, out)
    lens = [len(x) for x in said]
    rk, rv = P.read_int4(cache, 0, sum(lens), C.cu_of(lens), torch.zeros(B, device="cuda", dtype=torch.int32))
    whole = torch.stack([t for x in said for t in x])
    for got, want in ((rk, whole[:, :Nkv]), (rv, whole[:, Nkv:])):
        C.close_rounded(got, U.quantised_values(want), 2.0 ** -22 * want.double().abs().amax())
