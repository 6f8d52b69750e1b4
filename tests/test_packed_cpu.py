"""What the operators on packed sequences refuse, on the host: nothing is launched."""
import ctypes

import pytest
import torch


def P():
    from tpp_pytorch_extension_b200._C import _packed_attn
    return _packed_attn


def structs():
    from tpp_pytorch_extension_b200 import _lib
    s = _lib._struct
    return (s("Int4CacheStruct", p="pool table lengths", l="pages table_cols B kv_heads H"),
            s("HeadPrepStruct", p="q k v q_norm k_norm ep pos cu_seqlens q_out k_out cache", l="T Nq Nkv H ldq ldk ldv rot max_pos ld_ep", f="eps", i="norm_is_f32"),
            s("Int4AttentionStruct", p="q cache cu_seqlens out scratch", z="scratch_bytes", l="T Nq ldq", f="scale", i="causal"),
            s("PackedAttentionStruct", p="q k v cu_seqlens out", l="T B Nq Nkv H ldq ldk ldv", f="scale", i="causal"))


def lib():
    from tpp_pytorch_extension_b200 import _lib
    return _lib.lib()


A = 1 << 20  # an aligned address that no call gets as far as reading


def cache(**kw):
    f = dict(pool=A, table=A, lengths=A, pages=4, table_cols=2, B=3, kv_heads=2, H=128) | kw
    return structs()[0](**f)


def prep(c=None, **kw):
    f = dict(q=A, k=A, v=A, q_out=A, k_out=A, T=3, Nq=4, Nkv=2, H=128, ldq=1024, ldk=1024, ldv=1024, eps=1e-6) | kw
    if c is not None:
        f["cache"] = ctypes.addressof(c)
    a = structs()[1](**f)
    return lib().tpx_head_prep(ctypes.byref(a), None)


def attend(c, **kw):
    f = dict(q=A, cache=ctypes.addressof(c), out=A, scratch=A, scratch_bytes=1 << 40, T=3, Nq=4, ldq=512, scale=1.0, causal=1) | kw
    a = structs()[2](**f)
    return lib().tpx_int4_attention(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), 1), (dict(k=None), 1), (dict(q_out=None), 1), (dict(k=A + 2), 1), (dict(ldq=1020), 1), (dict(T=-1), 1), (dict(Nq=0, Nkv=0), 1),
    (dict(H=24), 2), (dict(H=272), 2), (dict(H=0), 2), (dict(cu_seqlens=A), 1),
    (dict(ep=A, rot=8, max_pos=4, ld_ep=8), 1), (dict(ep=A, rot=256, max_pos=4, ld_ep=256), 1), (dict(ep=A, rot=128, max_pos=0, ld_ep=128), 1),
    (dict(ep=A, rot=128, max_pos=9, ld_ep=32), 1), (dict(ep=A, rot=40, max_pos=9, ld_ep=40), 1)])
def test_head_prep_refuses(kw, rc):
    assert prep(**kw) == rc and lib().tpx_last_error()


@pytest.mark.parametrize("kw,rc", [(dict(pool=None), 1), (dict(pool=A + 8), 1), (dict(H=96), 2), (dict(B=0), 1), (dict(pages=0), 1), (dict(pages=1 << 31), 1),
                                   (dict(table_cols=0), 1), (dict(table_cols=(1 << 25) + 1), 1), (dict(kv_heads=0), 1)])
def test_caches_are_checked(kw, rc):
    c = cache(**kw)
    assert attend(c) == rc
    assert lib().tpx_int4_read(ctypes.byref(c), None, 3, A, A, None) == rc
    if not kw.get("H"):
        assert prep(c) == rc


def test_calls_on_a_cache_are_checked():
    assert prep(cache(), T=4) == 1 and prep(cache(), Nkv=1) == 1 and prep(cache(H=64)) == 1 and prep(cache(), v=None) == 1
    assert attend(cache(), T=2) == 1 and attend(cache(), Nq=5) == 1 and attend(cache(), Nq=0) == 1 and attend(cache(), q=None) == 1
    assert attend(cache(), ldq=516) == 1 and attend(cache(), out=A + 4) == 1
    assert attend(cache(), scratch=None) == 4 and attend(cache(), scratch_bytes=4096) == 4 and attend(cache(), scratch=A + 128) == 4
    assert lib().tpx_int4_read(None, None, 3, A, A, None) == 1 and lib().tpx_int4_read(ctypes.byref(cache()), None, 4, A, A, None) == 1
    # calls without a token have nothing to do
    assert attend(cache(), T=0, cu_seqlens=A, q=None, out=None, scratch=None) == 0 and prep(cache(), T=0, cu_seqlens=A, q=None, k=None) == 0


def test_python_refusals():
    from tpp_pytorch_extension_b200._lib import TpxError
    m = P()
    x = torch.zeros(3, 8 * 128, dtype=torch.bfloat16)
    with pytest.raises(TpxError, match="CUDA"):
        m.qk_norm_rope(x, 4, 2, 128)
    c = m.Int4Cache(2, 7, 2, 128, 3, 4, device="cpu")
    with pytest.raises(TpxError, match="CUDA"):
        m.attention_int4(x.view(3, 8, 128), c, 0)
    for bad in (dict(head_dim=96), dict(pages=0), dict(columns=0)):
        with pytest.raises(TpxError):
            m.Int4Cache(**(dict(layers=1, pages=4, kv_heads=2, head_dim=64, sequences=2, columns=4, device="cpu") | bad))
    with pytest.raises(TpxError):
        m.Int4Cache.over([torch.zeros(4, 2, 100, dtype=torch.uint8)], c.table, c.lengths)
    with pytest.raises(TpxError):
        m.Int4Cache.over(c.pools, c.table.long(), c.lengths)
    with pytest.raises(TpxError):
        m.Int4Cache.over(c.pools, c.table, c.lengths[:2])


def test_pages_are_handed_out_and_taken_back():
    from tpp_pytorch_extension_b200._lib import TpxError
    c = P().Int4Cache(2, 7, 2, 128, 3, 4, device="cpu")
    assert c.bytes_per_token() == 2 * 2 * 144
    c.add_pages([33, 0, 64])
    assert c.table.tolist() == [[0, 1, -1, -1], [-1] * 4, [2, 3, -1, -1]]
    c.add_pages([33, 1, 65])
    assert c.table.tolist() == [[0, 1, -1, -1], [4, -1, -1, -1], [2, 3, 5, -1]]
    with pytest.raises(TpxError, match="free"):
        c.add_pages(65)
    with pytest.raises(TpxError, match="passes"):
        c.add_pages([33, 1, 129])
    with pytest.raises(TpxError, match="sizes"):
        c.add_pages([1, 2])
    c.lengths.fill_(5)
    c.advance(torch.tensor([0, 2, 2, 7], dtype=torch.int32))
    assert c.lengths.tolist() == [7, 5, 10]
    c.advance()
    assert c.lengths.tolist() == [8, 6, 11]
    c.release(2)
    assert c.lengths.tolist() == [8, 6, 0] and c.table[2].tolist() == [-1] * 4
    c.add_pages([33, 100, 0])
    assert sorted(p for r in c.table.tolist() for p in r if p >= 0) == [0, 1, 2, 3, 4, 5]


def packed(**kw):
    f = dict(q=A, k=A, v=A, cu_seqlens=A, out=A, T=9, B=2, Nq=4, Nkv=2, H=128, ldq=512, ldk=256, ldv=256, scale=1.0, causal=1) | kw
    a = structs()[3](**f)
    return lib().tpx_packed_attention(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,rc", [(dict(q=None), 1), (dict(v=None), 1), (dict(cu_seqlens=None), 1), (dict(out=None), 1), (dict(H=96), 2), (dict(H=256), 2), (dict(Nq=5), 1),
                                   (dict(Nkv=0), 1), (dict(Nq=258), 2), (dict(B=0), 1), (dict(T=-1), 1), (dict(T=1 << 31), 1), (dict(k=A + 8), 1), (dict(ldv=260), 1),
                                   (dict(T=1 << 30, Nkv=4), 1),
                                   (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1)])
def test_packed_attention_refuses(kw, rc):
    assert packed(**kw) == rc and lib().tpx_last_error()
    assert packed(T=0, q=None) == 0


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_attention_over_the_cache_wants_a_finite_scale(scale):
    assert attend(cache(), scale=scale) == 1 and lib().tpx_last_error()


def test_lengths_move_by_the_sequences_of_the_cache():
    from tpp_pytorch_extension_b200._lib import TpxError
    c = P().Int4Cache(1, 3, 1, 64, 3, 1, device="cpu")
    for cu in ([0, 4], [0, 1, 2], [0, 1, 2, 3, 4]):
        with pytest.raises(TpxError, match="sequences"):
            c.advance(torch.tensor(cu, dtype=torch.int32))
    assert c.lengths.tolist() == [0, 0, 0]


def test_models_without_a_packed_form_say_so():
    from tpp_pytorch_extension_b200._lib import TpxError
    from tpp_pytorch_extension_b200.llm.fused_opt_infer import OPTRunner

    class Opt(OPTRunner):
        def __init__(self):
            torch.nn.Module.__init__(self)
            self.layers = [object()]

    with pytest.raises(TpxError, match="packed"):
        Opt().generate_packed([torch.zeros(3, dtype=torch.int64)], 2)
