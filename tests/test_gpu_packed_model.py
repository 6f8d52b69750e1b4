"""The Llama layers on prompts laid end to end and a cache held in 4 bits: every operator as the layers call it against its 64-bit form, the
first tokens' logits against the padded path, and generation with and without a recorded step."""
import pytest
import torch

from tests import packed_util as U
from tests import test_gpu_packed_cache as cache_file
from tests import test_gpu_packed_prompts as prompts_file
from tests.gpu_util import assert_no_kernel_error

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8
LENS = [1, 33, 100, 64]


def runner(cuda, weight_dtype="bf16", heads=4, kv_heads=2, H=64, layers=2, bias=False, seed=3):
    from tpp_pytorch_extension_b200._C import _fused_llm_infer as F
    from tpp_pytorch_extension_b200.llm import fused_llama_infer as FL
    shape = FL.LlamaShape(layers, 256, heads, kv_heads, 512, 1024, head_dim=H, max_position_embeddings=256)
    model = FL.build_random_llama(shape, weight_dtype, cuda, seed=seed, std=0.08)
    if bias:
        g = torch.Generator(device=cuda).manual_seed(5)
        for layer in model.layers:
            layer.Bqkv = (torch.randn((heads + 2 * kv_heads) * H, generator=g, device=cuda) * 0.3).bfloat16()
            layer.__class__ = F.Qwen2DecoderLayer
    return model


def prompts(cuda, lens=LENS, vocab=1024):
    g = torch.Generator().manual_seed(11)
    return [torch.randint(0, vocab, (n,), generator=g).to(cuda) for n in lens]


class Recorder:
    """Calls of the operators as the layers make them."""

    def __init__(self, monkeypatch):
        from tpp_pytorch_extension_b200._C import _packed_attn as P
        self.calls = []
        for name in ("qk_norm_rope", "attention_packed", "attention_int4"):
            monkeypatch.setattr(P, name, self.wrap(name, getattr(P, name)))

    def wrap(self, name, op):
        def call(*args, **kw):
            out = op(*args, **kw)
            kw = {k: v.clone() if k == "positions" else v for k, v in kw.items()}  # generate_packed() moves them in place
            cache = kw.get("cache") or (args[1] if name == "attention_int4" else None)
            held = None
            if cache is not None:
                layer = kw["layer"] if "layer" in kw else args[2]
                held = (cache.pools[layer].clone(), cache.table.clone(), cache.lengths.clone())
            self.calls.append((name, args, kw, out, held))
            return out
        return call


def check_calls(calls, lens, steps, Nq, Nkv, H):
    from tpp_pytorch_extension_b200._C._packed_attn import Int4Cache
    assert [c[0] for c in calls] == ["qk_norm_rope", "attention_packed"] * 2 + ["qk_norm_rope", "attention_int4"] * 2 * steps
    for i in range(0, len(calls), 2):
        (_, (qkv, *_), kw, (q, k), held), (name, args, _, out, _) = calls[i], calls[i + 1]
        prompt = name == "attention_packed"
        old, new = held[2].tolist(), lens if prompt else [1] * len(lens)
        assert old == [0 if prompt else n + i // 4 - 1 for n in lens]
        cache = Int4Cache.over([held[0]], held[1], held[2])
        cu = prompts_file.cu_of(new)
        x = qkv.view(qkv.shape[0], -1, H)
        for heads, got in ((slice(0, Nq), q), (slice(Nq, Nq + Nkv), k)):
            if got is not None:
                want, off = U.norm_rope(x[:, heads], None, 1e-6, kw["ep"], kw["positions"])
                cache_file.close_rounded(got, want, off)
        for b, (m, n, at) in enumerate(zip(old, new, cu.tolist())):  # what was appended
            heads = cache_file.sequence_heads(cache, b, m + n)
            for (c, s, z), src in ((heads[3:], x[at:at + n, Nq + Nkv:]), (heads[:3], None if k is None else k[at:at + n])):
                if src is not None:
                    wc, ws, wz = U.quantised(src)
                    c, s, z = (t[m:].unflatten(-1, (-1, 64)) for t in (c, s, z))
                    assert torch.equal(c, wc) and torch.equal(s[..., :1], ws) and torch.equal(z[..., :1], wz)
        if prompt:
            assert args[2].data_ptr() == x[:, Nq + Nkv:].data_ptr()  # the values are read where the linear left them
            prompts_file.check(q, args[1], args[2], out, new, cu)
        else:
            cache_file.check_attention(cache, q, out, old, new, cu, True, H ** -0.5)


@pytest.mark.parametrize("Nq,Nkv,H", [(4, 2, 64), (4, 1, 128), (3, 3, 64)])
def test_the_operators_in_a_run(cuda, monkeypatch, Nq, Nkv, H):
    model = runner(cuda, heads=Nq, kv_heads=Nkv, H=H)
    rec = Recorder(monkeypatch)
    model.generate_packed(prompts(cuda), 4, use_graph=False)
    assert_no_kernel_error()
    check_calls(rec.calls, LENS, 3, Nq, Nkv, H)


@pytest.mark.parametrize("weight_dtype,bias", [("bf16", False), ("bf16", True), ("mxfp4", False)])
def test_first_logits_match_the_padded_path(cuda, weight_dtype, bias, monkeypatch):
    """Prompts see each other's keys nowhere and are not quantized: their logits are those of each prompt alone in the padded path. Both round
    to bf16 seven times in a layer (norm, q/k/v, rotation, weights, context, residual, MLP), two layers, and twice in the head: 16
    roundings of at most 2^-8 each on either side, in the norm of the row."""
    model = runner(cuda, weight_dtype, bias=bias)
    ids = prompts(cuda)
    got = []
    monkeypatch.setattr(model, "_pick", lambda lg: (got.append(lg.clone()), type(model)._pick(model, lg))[1])
    model.generate_packed(ids, 1)
    for p, lg in zip(ids, got[0][:, 0].float()):
        want = model.forward(p.unsqueeze(0))[0][0, -1].float()
        assert float((lg - want).norm()) <= 2 * 16 * BF16 * float(want.norm())


@pytest.mark.parametrize("weight_dtype", ["bf16", "mxfp4"])
def test_recorded_steps_give_the_same_tokens(cuda, weight_dtype):
    model = runner(cuda, weight_dtype, heads=4, kv_heads=2, H=128)
    ids = prompts(cuda, [40, 3, 97])
    eager = model.generate_packed(ids, 40, use_graph=False)
    recorded = model.generate_packed(ids, 40)
    for p, a, b in zip(ids, eager, recorded):
        assert a.shape == (p.numel() + 40,) and torch.equal(a[:p.numel()], p) and torch.equal(a, b)
    assert_no_kernel_error()


def test_refusals(cuda):
    from tpp_pytorch_extension_b200._lib import TpxError
    model = runner(cuda)
    for bad in ([], [torch.zeros(0, dtype=torch.int64, device=cuda)], [torch.zeros((1, 2), dtype=torch.int64, device=cuda)]):
        with pytest.raises(TpxError):
            model.generate_packed(bad, 2)
    p = prompts(cuda, [200])
    with pytest.raises(TpxError):
        model.generate_packed(p, 0)
    with pytest.raises(TpxError):
        model.generate_packed(p, 58)  # 257 tokens, 256 positions
    assert model.generate_packed(p, 57)[0].shape == (257,)
    with pytest.raises(TpxError):
        runner(cuda, H=32).generate_packed(p, 2)  # no 4-bit cache of this head size
