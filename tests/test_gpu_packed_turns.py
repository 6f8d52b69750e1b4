"""Tokens behind cached ones: later turns, drafted tokens and resting sequences in one call with new prompts, by the operators and by the layer."""
import pytest
import torch

from tests import test_gpu_packed_cache as C
from tests import test_gpu_packed_model as M
from tests import test_gpu_packed_prompts as S
from tests.gpu_util import assert_no_kernel_error

pytestmark = pytest.mark.gpu

MIXED = [([0, 40, 0, 7, 33], [70, 5, 0, 1, 0]), ([100, 0], [0, 0]), ([0, 0, 0], [1, 200, 3]), ([64, 1, 31], [129, 1, 40]), ([0, 300] * 70, [2, 1] * 70)]


@pytest.mark.parametrize("old,new", MIXED)
@pytest.mark.parametrize("Nq,Nkv,H", [(8, 2, 128), (3, 3, 64), (7, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_the_two_halves_of_a_call(Nq, Nkv, H, old, new, causal):
    """Each writes its own sequences' rows and leaves the others'."""
    g = C.gen(101, Nq, H, *old[:4], *new[:4])
    cache = C.new_cache(old, new, Nkv, H, g)
    C.fill(cache, g, old, new)
    T, cu = sum(new) + 4, C.cu_of(new, 1)
    q, k, v = S.inputs(g, T, Nq, Nkv, H)
    out = torch.full_like(q, 9.0)
    C.P().attention_packed(q, k, v, cu, causal, None, out, cache.lengths)
    behind = torch.zeros(T, dtype=torch.bool, device="cuda")
    first = torch.zeros_like(behind)
    for at, m, n in zip(cu.tolist(), old, new):
        (behind if m else first)[at:at + n] = True
    assert bool((out[~first] == 9).all())
    S.check(q, k, v, out, [n if m == 0 else 0 for m, n in zip(old, new)], cu, causal)
    before = out.clone()
    C.P().attention_int4(q, cache, 0, cu, causal, None, out, behind=True)
    assert torch.equal(out[~behind], before[~behind])
    C.check_attention(cache, q, out, old, [n if m else 0 for m, n in zip(old, new)], cu, causal, H ** -0.5)


def test_refused():
    from tpp_pytorch_extension_b200._lib import TpxError
    g = C.gen(102)
    q, k, v = S.inputs(g, 9, 4, 2, 64)
    cu = C.cu_of([5, 4])
    for lengths in (torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(TpxError):
            C.P().attention_packed(q, k, v, cu, lengths=lengths)


class Watch:
    """What a layer's attention is made of, and what goes into its output projection."""

    def __init__(self, monkeypatch):
        from tpp_pytorch_extension_b200._C import _fused_llm_infer as F
        from tpp_pytorch_extension_b200._C import _packed_attn as P
        self.qkv, self.q, self.k, self.ctx, self.ops = [], [], [], [], []
        prep, act = P.qk_norm_rope, F.fc_plain_act

        def qk_norm_rope(*a, **kw):
            q, k = prep(*a, **kw)
            self.qkv.append(a[0]), self.q.append(q), self.k.append(k)
            return q, k

        def fc_plain_act(x, *a, **kw):
            if len(self.ctx) < len(self.q):
                self.ctx.append(x.clone())
            return act(x, *a, **kw)

        monkeypatch.setattr(P, "qk_norm_rope", qk_norm_rope)
        monkeypatch.setattr(F, "fc_plain_act", fc_plain_act)
        for name in ("attention_packed", "attention_int4"):
            monkeypatch.setattr(P, name, self.count(name, getattr(P, name)))

    def count(self, name, op):
        def call(*a, **kw):
            self.ops.append(name)
            return op(*a, **kw)
        return call


def check_layer(w, i, cache, old, new, cu, Nq, Nkv, H):
    """The context of call i against what every sequence has to see."""
    q, ctx = w.q[i], w.ctx[i].view(-1, Nq, H)
    v = w.qkv[i].view(-1, Nq + 2 * Nkv, H)[:, Nq + Nkv:]
    S.check(q, w.k[i], v, ctx, [n if m == 0 else 0 for m, n in zip(old, new)], cu)
    C.check_attention(cache, q, ctx, old, [n if m else 0 for m, n in zip(old, new)], cu, True, H ** -0.5)


TURNS = [[40, 3, 0, 64], [5, 0, 70, 33], [1, 1, 1, 1], [0, 2, 0, 5], [31, 0, 1, 0]]


@pytest.mark.parametrize("Nq,Nkv,H", [(4, 2, 64), (4, 1, 128)])
def test_turns_through_a_layer(cuda, monkeypatch, Nq, Nkv, H):
    """Prompts, later turns beside a new prompt, single tokens, drafts beside sequences that rest."""
    model = M.runner(cuda, heads=Nq, kv_heads=Nkv, H=H, layers=1)
    layer, w, g = model.layers[0], Watch(monkeypatch), C.gen(103, H)
    cache = C.P().Int4Cache(1, 40, Nkv, H, 4, 8)
    cache.add_pages(160)
    old = [0] * 4
    for i, new in enumerate(TURNS):
        cu = C.cu_of(new)
        layer.forward_packed(C.rand(g, sum(new), 256).bfloat16(), cache, cu)
        check_layer(w, i, cache, old, new, cu, Nq, Nkv, H)
        cache.advance(cu)
        old = [a + b for a, b in zip(old, new)]
    assert w.ops == ["attention_packed"] + ["attention_packed", "attention_int4"] * 4  # nothing is cached before the first, and the host knows
    assert_no_kernel_error()


def test_a_recorded_call_goes_by_the_lengths_of_its_replay(cuda, monkeypatch):
    """Recorded while nothing is cached, replayed behind cached tokens and for a new prompt."""
    Nq, Nkv, H = 4, 2, 64
    model = M.runner(cuda, heads=Nq, kv_heads=Nkv, H=H, layers=1)
    layer, w, g = model.layers[0], Watch(monkeypatch), C.gen(104)
    cache = C.P().Int4Cache(1, 40, Nkv, H, 2, 8)
    cache.add_pages(160)
    cu, hs = C.cu_of([30, 10]), C.rand(g, 40, 256).bfloat16()
    layer.forward_packed(hs.clone(), cache, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward_packed(hs, cache, cu)
    old = [0, 0]
    for new in ([30, 10], [25, 15], [0, 40]):
        if new == [0, 40]:
            cache.release(1)
            cache.add_pages([160, 160])
            old[1] = 0
        cu.copy_(C.cu_of(new))
        hs.copy_(C.rand(g, 40, 256))
        graph.replay()
        check_layer(w, 1, cache, old, new, cu, Nq, Nkv, H)
        cache.advance(cu)
        old = [a + b for a, b in zip(old, new)]
    assert_no_kernel_error()
