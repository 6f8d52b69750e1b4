"""Attention over whole prompts laid end to end, against a 64-bit form: lengths from none to long, head groups that do and do not divide a
tile, strided rows, and what must not reach a row."""
import math

import pytest
import torch

from tests import packed_util as U
from tests.gpu_util import assert_no_kernel_error

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8


def P():
    from tpp_pytorch_extension_b200._C import _packed_attn
    return _packed_attn


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def cu_of(lengths, first=0):
    return torch.tensor([first] + list(lengths)).cumsum(0).to(torch.int32).cuda()


def inputs(g, T, Nq, Nkv, H, grow=1.0):
    """q on its own, k and v as views of rows that hold both."""
    q = (rand(g, T, Nq, H) * grow).bfloat16()
    kv = rand(g, T, 2 * Nkv, H).bfloat16()
    return q, kv[:, :Nkv], kv[:, Nkv:]


def check(q, k, v, out, lengths, cu, causal=True, scale=None, rows=None):
    H = q.shape[2]
    R = q.shape[1] // k.shape[1]
    scale = H ** -0.5 if scale is None else scale
    for b, n in enumerate(lengths):
        if n == 0 or (rows is not None and b not in rows):
            continue
        at = int(cu[b])
        x, kk, vv = (t[at:at + n].double() for t in (q, k, v))
        want, w = U.attention(x, kk, vv, 0, causal, scale)
        size = abs(scale) * torch.einsum("nhd,mhd->hnm", x.abs(), kk.abs().repeat_interleave(R, 1)).masked_fill(w == 0, 0).amax(-1)
        plain = torch.einsum("hnm,mhd->nhd", w, vv.abs().repeat_interleave(R, 1))
        # scores: 16 roundings of sums and products; weights: those of both ends, the exponential's 2^-22, one rounding to bf16 each; sums
        # over the keys in fp32; the result is rounded once
        off = (2 * 16 * 2.0 ** -24 * size + 2.0 ** -20 + 2.0 ** -23 * n / 16).T[..., None]
        limit = BF16 * want.abs() + (1.02 * BF16 + 2 * off) * plain
        err = (out[at:at + n].double() - want).abs()
        assert bool((err <= limit).all()), (b, n, float((err - limit).max()), float(err.max()))
    assert_no_kernel_error()


GROUPS = [(1, 1), (4, 1), (8, 2), (32, 8), (7, 1), (5, 5), (12, 1), (3, 1), (33, 1), (128, 1), (10, 2)]


@pytest.mark.parametrize("H", [128, 64])
@pytest.mark.parametrize("Nq,Nkv", GROUPS)
@pytest.mark.parametrize("lengths", [[1], [2, 1, 1], [127, 128, 129], [31, 0, 64, 33, 0], [300, 257]])
def test_lengths_and_groups(Nq, Nkv, H, lengths):
    g = gen(Nq, Nkv, H, *lengths)
    q, k, v = inputs(g, sum(lengths), Nq, Nkv, H)
    cu = cu_of(lengths)
    check(q, k, v, P().attention_packed(q, k, v, cu), lengths, cu)


@pytest.mark.parametrize("H", [128, 64])
@pytest.mark.parametrize("Nq,Nkv,lengths", [(4, 1, [2500]), (2, 2, [1500, 3, 1100]), (7, 1, [1024, 1025]), (16, 1, [0, 1300])])
@pytest.mark.parametrize("causal", [True, False])
def test_long(Nq, Nkv, H, lengths, causal):
    g = gen(Nq, Nkv, H, causal, *lengths)
    q, k, v = inputs(g, sum(lengths), Nq, Nkv, H)
    cu = cu_of(lengths)
    check(q, k, v, P().attention_packed(q, k, v, cu, causal), lengths, cu, causal)


@pytest.mark.parametrize("lengths", [[5, 200, 1], [128, 256], [64, 0, 65]])
def test_both_directions_rows_of_no_sequence_and_a_given_output(lengths):
    g = gen(*lengths)
    T = sum(lengths) + 9
    q, k, v = inputs(g, T, 6, 3, 64)
    cu = cu_of(lengths, 4)
    for causal in (True, False):
        out = torch.full_like(q, 5.0)
        k2, v2 = k.clone(), v.clone()
        for t in (k2, v2):
            t[:4], t[T - 5:] = math.nan, math.inf  # rows of no sequence
        q[:4], q[T - 5:] = math.nan, math.nan
        got = P().attention_packed(q, k2, v2, cu, causal, 0.2, out)
        assert got.data_ptr() == out.data_ptr() and bool((out[:4] == 5).all()) and bool((out[T - 5:] == 5).all())
        check(q, k, v, out, lengths, cu, causal, 0.2)


@pytest.mark.parametrize("H", [64, 128])
@pytest.mark.parametrize("grow", [0.0, 2.0 ** -20, 2.0 ** 5, 2.0 ** 10])
@pytest.mark.parametrize("scale", [None, 2.0 ** -10, 1.0])
def test_scores_of_any_size(H, grow, scale):
    lengths = [400, 130]
    q, k, v = inputs(gen(H, 7), sum(lengths), 4, 2, H, grow)
    cu = cu_of(lengths)
    check(q, k, v, P().attention_packed(q, k, v, cu, True, scale), lengths, cu, True, scale)


def test_scores_that_grow_along_the_sequence():
    """Every tile of keys passes the reference of the one before: O is rescaled each time."""
    H, n = 128, 1500
    g = gen(21)
    q, k, v = inputs(g, n, 4, 1, H)
    k = (k.float() * torch.linspace(0, 40, n, device="cuda")[:, None, None]).bfloat16()
    cu = cu_of([n])
    check(q, k, v, P().attention_packed(q, k, v, cu), [n], cu)


@pytest.mark.parametrize("H", [64, 128])
@pytest.mark.parametrize("Nq", [1, 3, 4])
@pytest.mark.parametrize("key", [0, 5, 100, 127, 128, 290, 400])
def test_infinities_and_nan_stay_with_those_who_see_them(Nq, H, key):
    lengths = [401, 70]
    g = gen(Nq, H, key)
    q, k, v = inputs(g, sum(lengths), Nq, 1, H)
    cu = cu_of(lengths)
    for value in (math.nan, math.inf, -math.inf):
        v2, k2 = v.clone(), k.clone()
        v2[key, 0, 3], k2[key, 0, 9] = value, value
        out = P().attention_packed(q, k, v2, cu)
        check(q, k, v, out[:key] if key else out, [key], cu)
        col = out[key:401, :, 3].float()
        assert bool((col.isnan() if math.isnan(value) else col == value).all())
        clean = v.clone()
        clean[key, 0, 3] = 0
        check(q, k, clean, torch.where(torch.arange(H, device="cuda") == 3, P().attention_packed(q, k, clean, cu), out), lengths, cu)
        out = P().attention_packed(q, k2, v, cu)
        check(q, k, v, out, [key], cu)
        check(q, k, v, out, lengths, cu, rows={1})
        if math.isnan(value):
            assert out[key:401].isnan().all()


@pytest.mark.parametrize("key", range(0, 128, 5))
def test_nan_in_a_key_reaches_every_row_behind_it(key):
    """Whatever way a key's weight is computed, in tiles that all rows of a unit see."""
    n, H = 700, 64
    q, k, v = inputs(gen(key, 3), n, 2, 1, H)
    k = k.clone()
    k[key, 0, 1] = math.nan
    out = P().attention_packed(q, k, v, cu_of([n]))
    assert out[key:].isnan().all() and out[:key].isfinite().all()


def test_many_short_sequences():
    lengths = [(i * 37) % 23 for i in range(1500)]
    g = gen(31)
    q, k, v = inputs(g, sum(lengths), 4, 2, 64)
    cu = cu_of(lengths)
    check(q, k, v, P().attention_packed(q, k, v, cu), lengths, cu, rows=set(range(0, 1500, 41)))


@pytest.mark.parametrize("Nq,Nkv,H", [(8, 4, 64), (4, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("sequences", [32, 33, 127, 128, 129, 200])
def test_units_of_many_sequences(sequences, Nq, Nkv, H):
    """Single tiles, pairs of tiles and empty sequences mixed, dealt by length or in order."""
    lengths = [(i * i * 29 + 7 * i) % 333 if i % 5 else (i % 3) * (i % 17) for i in range(sequences)]
    g = gen(sequences, Nq, H)
    q, k, v = inputs(g, sum(lengths), Nq, Nkv, H)
    cu = cu_of(lengths)
    for causal in (True, False):
        check(q, k, v, P().attention_packed(q, k, v, cu, causal), lengths, cu, causal)


def test_streams_graphs_and_repetition():
    lengths = [[700, 20], [64, 1000]]
    g = gen(41)
    ins = [inputs(g, sum(x), 8, 2, 128) for x in lengths]
    cus = [cu_of(x) for x in lengths]
    want = [P().attention_packed(*i, c) for i, c in zip(ins, cus)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(P().attention_packed(*ins[i], cus[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = P().attention_packed(*ins[0], cus[0])
    cus[0].copy_(torch.tensor([0, 30, 720], dtype=torch.int32))  # the replay reads the lengths that are there then
    graph.replay()
    check(*ins[0], out, [30, 690], cus[0])


def test_empty_call():
    q = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert P().attention_packed(q, q[:, :2], q[:, :2], cu_of([0, 0])).shape == (0, 4, 64)


def test_refused_tensors():
    from tpp_pytorch_extension_b200._lib import TpxError
    q, k, v = inputs(gen(41), 9, 4, 2, 64)
    cu = cu_of([5, 4])
    A = P().attention_packed
    refused = [
        lambda: A(q, k, v, None), lambda: A(q, k, v, cu.long()), lambda: A(q, k, v, cu[:1]), lambda: A(q, k, v, cu.cpu()), lambda: A(q.cpu(), k, v, cu),
        lambda: A(q[:8], k, v, cu), lambda: A(q[:, :3], k, v, cu), lambda: A(q, k, v[:, :1], cu), lambda: A(q, k[..., :32], v[..., :32], cu),
        lambda: A(q[..., :32], k[..., :32], v[..., :32], cu), lambda: A(q.float(), k.float(), v.float(), cu), lambda: A(q.half(), k.half(), v.half(), cu),
        lambda: A(q, k, v, cu, scale=0.0), lambda: A(q, k, v, cu, scale=-1.0), lambda: A(q, k, v, cu, scale=math.nan), lambda: A(q, k, v, cu, scale=math.inf),
        lambda: A(q, k, v, cu, out=q), lambda: A(q, k, v, cu, out=torch.empty_like(k)), lambda: A(q, k, v, cu, out=torch.empty_like(q).float()),
        lambda: A(q, k, v, cu, out=torch.empty(9, 8, 64, device="cuda", dtype=torch.bfloat16)[:, ::2]), lambda: A(q.clone().requires_grad_(), k, v, cu),
        lambda: A(q, k.transpose(0, 1), v.transpose(0, 1), cu), lambda: A(q, k[:1].expand(9, 2, 64), v, cu),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(TpxError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert_no_kernel_error()


def test_a_sequence_does_not_feel_its_neighbours():
    """Rows of other sequences in a tile, whatever their scores are, change no bit."""
    g = gen(43)
    q, k, v = inputs(g, 330, 7, 1, 128)
    cu = cu_of([200, 130])
    plain = P().attention_packed(q, k, v, cu)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    for t, x in ((q2, 2.0 ** 40), (k2, -2.0 ** 40), (v2, math.inf)):
        t[200:] = x
    assert torch.equal(P().attention_packed(q2, k2, v2, cu)[:200], plain[:200])
    assert_no_kernel_error()
