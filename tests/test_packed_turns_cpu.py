"""Calls for new sequences alone and for sequences with cached tokens alone: refusals, and when the host is certain that nothing is cached."""
import ctypes

import pytest
import torch

from tests import test_packed_cpu as C


def test_the_c_entries_refuse():
    a = C.structs()[3](q=C.A, k=C.A, v=C.A, cu_seqlens=C.A, out=C.A, T=9, B=2, Nq=4, Nkv=2, H=96, ldq=512, ldk=256, ldv=256, scale=1.0, causal=1)
    assert C.lib().tpx_packed_attention_new(ctypes.byref(a), C.A, None) == 2
    a.H = 128
    assert C.lib().tpx_packed_attention_new(ctypes.byref(a), None, None) == 1 and C.lib().tpx_last_error()
    a.T = 0
    assert C.lib().tpx_packed_attention_new(ctypes.byref(a), C.A, None) == 0
    c = C.cache()
    b = C.structs()[2](q=C.A, cache=ctypes.addressof(c), out=C.A, scratch=C.A, scratch_bytes=1 << 40, T=3, Nq=5, ldq=512, scale=1.0, causal=1)
    assert C.lib().tpx_int4_attention_behind(ctypes.byref(b), None) == 1
    b.T, b.cu_seqlens, b.Nq = 0, C.A, 4
    assert C.lib().tpx_int4_attention_behind(ctypes.byref(b), None) == 0


@pytest.mark.parametrize("inference", [False, True])
def test_a_cache_is_new_until_its_lengths_are_written_to(inference):
    from tpp_pytorch_extension_b200._C._packed_attn import Int4Cache
    with torch.inference_mode(inference):
        for change in (lambda c: c.advance(), lambda c: c.advance(torch.tensor([0, 1, 1], dtype=torch.int32)), lambda c: c.lengths.fill_(3),
                       lambda c: c.lengths.copy_(torch.tensor([1, 0])), lambda c: c.lengths[1:].add_(1), lambda c: c.release(0)):
            c = Int4Cache(2, 4, 1, 64, 2, 2, device="cpu")
            c.add_pages([33, 5])
            assert c.is_new() and c.is_new()
            change(c)
            assert not c.is_new()
        c = Int4Cache(1, 4, 1, 64, 2, 2, device="cpu")
        assert not Int4Cache.over(c.pools, c.table, c.lengths).is_new()  # others may have written them
