"""The packed layer on two gloo ranks against one: which heads a rank has, the share of the residual, the sums over ranks, and what goes into and
comes out of the cache. Linears and attention are plain ones in 64 bits here; what is under test is the layer's host side."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

D, NQ, NKV, H, FF = 128, 4, 2, 64, 192
CALLS = [[3, 0, 5], [2, 4, 0], None, None]  # new tokens of three sequences, or one of each


def _fakes(F, P, _lib):
    from tests import packed_util as U
    norm = lambda x, g, eps: x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * g.double()  # noqa: E731
    _lib.require_cuda = lambda *a: None
    F.fc_plain_norm = lambda x, g, eps, w, b=None: norm(x, g, eps) @ w.double().T
    F.fc_plain_act = lambda x, w, b=None, act=None, mul_in=None, res=None, res_scale=1.0: x @ w.double().T + res * res_scale
    F.fc_gate_up = lambda x, wg, wu, act, norm=None: (lambda y: torch.nn.functional.silu(y @ wg.double().T) * (y @ wu.double().T))(_norm_of(x, norm))
    _norm_of = lambda x, n: norm(x, *n)  # noqa: E731
    kept = {}  # sequence: keys and values

    def qk_norm_rope(qkv, nq, nkv, h, ep=None, positions=None, cu_seqlens=None, cache=None, layer=0, want_k=True):
        x = qkv.view(qkv.shape[0], -1, h)
        cu = range(cache.B + 1) if cu_seqlens is None else cu_seqlens.tolist()
        for b in range(cache.B):
            kept.setdefault(b, []).extend(x[cu[b]:cu[b + 1], nq:])
        return x[:, :nq], x[:, nq:nq + nkv] if want_k else None

    def attend(q, b, before):
        kv = torch.stack(kept[b])
        n = kv.shape[1] // 2
        return U.attention(q, kv[:, :n], kv[:, n:], before, True, h_scale)[0]

    h_scale = H ** -0.5

    def packed(q, k, v, cu, lengths=None):
        out = torch.full_like(q, float("nan"))
        c = cu.tolist()
        for b in range(len(c) - 1):
            if c[b] < c[b + 1] and (lengths is None or lengths[b] == 0):
                assert lengths is not None or len(kept[b]) == c[b + 1] - c[b]
                out[c[b]:c[b + 1]] = U.attention(q[c[b]:c[b + 1]], k[c[b]:c[b + 1]], v[c[b]:c[b + 1]], 0, True, h_scale)[0]
        return out

    def int4(q, cache, layer, cu=None, out=None, behind=False):
        c = list(range(cache.B + 1)) if cu is None else cu.tolist()
        out = torch.full_like(q, float("nan")) if out is None else out
        for b in range(cache.B):
            if c[b] < c[b + 1] and not (behind and cache.lengths[b] == 0):
                out[c[b]:c[b + 1]] = attend(q[c[b]:c[b + 1]], b, int(cache.lengths[b]))
        return out

    P.qk_norm_rope, P.attention_packed, P.attention_int4 = qk_norm_rope, packed, int4


def _run(F, FL, P):
    g = torch.Generator().manual_seed(3)
    sizes = {"q": (NQ * H, D), "k": (NKV * H, D), "v": (NKV * H, D), "o": (D, NQ * H), "gate": (FF, D), "up": (FF, D), "down": (D, FF)}
    w = {k: (torch.randn(s, generator=g) * 0.1).bfloat16() for k, s in sizes.items()}
    ones, grp = torch.ones(D), H * (NQ // NKV)
    plan = {"q": (0, grp), "k": (0, H), "v": (0, H), "o": (1, grp), "gate": (0, 64), "up": (0, 64), "down": (1, 64)}
    w = {k: FL._shard(w[k], d, b) for k, (d, b) in plan.items()}
    layer = F.LlamaDecoderLayer([ones, w["q"], w["k"], w["v"], w["o"], ones, w["gate"], w["up"], w["down"], torch.zeros(2, 32, H)], 0, 1e-5, H, 32, H)
    cache = P.Int4Cache(1, 6, layer.Nkv, H, 3, 2, device="cpu")
    cache.add_pages(40)
    outs = []
    for new in CALLS:
        cu = None if new is None else torch.tensor([0] + new).cumsum(0).to(torch.int32)
        hs = torch.randn(3 if new is None else sum(new), D, generator=g, dtype=torch.float64)
        outs.append(layer.forward_packed(hs, cache, cu).numpy())
        cache.advance(cu)
    return outs, cache.lengths.tolist(), layer.Nq


def _worker(rank, world, port, results):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        from tpp_pytorch_extension_b200 import _lib
        from tpp_pytorch_extension_b200._C import _fused_llm_infer as F
        from tpp_pytorch_extension_b200._C import _packed_attn as P
        from tpp_pytorch_extension_b200.llm import fused_llama_infer as FL
        _fakes(F, P, _lib)
        if world > 1:
            dist.init_process_group("gloo", rank=rank, world_size=world)
            F.set_pg(dist.group.WORLD)
        results.put((rank, world, _run(F, FL, P)))
        if world > 1:
            dist.destroy_process_group()
    except Exception as e:
        results.put((rank, world, repr(e)))


def test_two_ranks_give_what_one_gives():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=a) for a in ((0, 1, port, q), (0, 2, port, q), (1, 2, port, q))]
    for p in procs:
        p.start()
    got = {r[:2]: r[2] for r in (q.get(timeout=120) for _ in procs)}
    for p in procs:
        p.join(timeout=30)
    assert not any(isinstance(r, str) for r in got.values()), got
    outs, lengths, heads = got[0, 1]
    assert lengths == [7, 6, 7] and heads == NQ
    for rank in range(2):
        mine, held, own = got[rank, 2]
        assert held == lengths and own == NQ // 2
        for a, b in zip(map(torch.from_numpy, mine), map(torch.from_numpy, outs)):
            assert torch.allclose(a, b, rtol=1e-10, atol=1e-10) and bool(a.isfinite().all())
