"""Sequences of different lengths laid end to end, without padding, and a KV cache that is held in 4 bits: the pass behind the
q/k/v linear (head norms, rotation, append), attention over whole prompts and attention of a few new tokens over the cache, on the
kernels of include/tpx_packed.h. They stand beside the padded batches and the bf16 pages of _tpp_attn.

Token rows [T, ...] are cut into sequences by cu_seqlens (int32 [B + 1] on the device: sequence b has the rows cu[b] .. cu[b + 1] - 1);
without it row b is the one token of sequence b. Rows outside every sequence are read by nobody, and an output that the caller
passes has theirs left as they were. Nothing here waits for the device, so all of it can be recorded in a CUDA graph."""
import ctypes

import torch

from .. import _lib

S2 = 32       # tokens of a page
GROUP = 64    # values that share a scale and a minimum

_Int4CacheStruct = _lib._struct("Int4CacheStruct", p="pool table lengths", l="pages table_cols B kv_heads H")
_HeadPrepStruct = _lib._struct("HeadPrepStruct", p="q k v q_norm k_norm ep pos cu_seqlens q_out k_out cache", l="T Nq Nkv H ldq ldk ldv rot max_pos ld_ep",
                               f="eps", i="norm_is_f32")
_Int4AttentionStruct = _lib._struct("Int4AttentionStruct", p="q cache cu_seqlens out scratch", z="scratch_bytes", l="T Nq ldq", f="scale", i="causal")

_PackedAttentionStruct = _lib._struct("PackedAttentionStruct", p="q k v cu_seqlens out", l="T B Nq Nkv H ldq ldk ldv", f="scale", i="causal")


def _check(cond, text):
    if not cond:
        raise _lib.TpxError(text)


def _on_device(name, *tensors):
    """Inputs of one call: on the current device, whose stream the kernels run on, and not part of a backward pass, which these
    operators have none of."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.TpxError(f"{name}: tensors must be on a CUDA device (this library has no CPU path)")
        if dev is None:
            dev = t.device
            _check(dev.index == _lib.current_device(), f"{name}: tensors are on {dev}, the current device is cuda:{_lib.current_device()}")
        _check(t.device == dev, f"{name}: tensors are on {dev} and {t.device}")
        _check(not (t.requires_grad and torch.is_grad_enabled()), f"{name} has no backward pass: call it under torch.no_grad()")


def _sequences(name, cu, B, T):
    if cu is None:
        _check(B is None or T == B, f"{name}: {T} tokens without cu_seqlens are not one for each of {B} sequences")
        return None
    _check(cu.dtype == torch.int32 and cu.dim() == 1 and cu.is_contiguous() and (cu.numel() == B + 1 if B is not None else cu.numel() >= 2),
           f"{name}: cu_seqlens must be contiguous int32 with one value more than there are sequences")
    return cu.data_ptr()


def _rows(name, what, t, heads, dim):
    """Elements between the rows of t [T, heads, dim], whose heads lie side by side."""
    _check(t.dtype == torch.bfloat16 and t.dim() == 3 and t.shape[1:] == (heads, dim) and t.stride(2) == 1 and (heads == 1 or t.stride(1) == dim),
           f"{name}: {what} must be bf16 [tokens, {heads}, {dim}] with heads side by side")
    _check(t.shape[0] < 2 or t.stride(0) >= heads * dim, f"{name}: rows of {what} overlap")
    return t.stride(0) if t.shape[0] > 1 else heads * dim


def _output(name, out, shape, device):
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=device)
    _check(out.dtype == torch.bfloat16 and out.shape == shape and out.is_contiguous() and out.device == device,
           f"{name}: the output must be contiguous bf16 {tuple(shape)} on {device}")
    return out


class Int4Cache:
    """Keys and values of many sequences in 4 bits: per layer a pool of pages, uint8 [pages, kv_heads, 36 H] for head size H (64 or
    128), and for all layers one table int32 [B, columns] of the pages of every sequence (32 tokens each; -1: no page) and lengths
    int32 [B], the tokens cached before the next call. 64 values share a scale and a minimum: 4.5 bits per value.

    `pages` pages for every layer; a sequence has room for what add_pages() gave it. Which page belongs to which sequence
    is decided on the host, everything else happens on the device. A page that is written to belongs to one sequence; pages that are only
    read may be shared. The operators do not move lengths: advance() does, once per step, after the last layer."""

    def __init__(self, layers, pages, kv_heads, head_dim, sequences, columns, device="cuda"):
        _check(head_dim in (64, 128), f"Int4Cache: head size {head_dim} is not 64 or 128")
        _check(min(layers, pages, kv_heads, sequences, columns) > 0, "Int4Cache: sizes must be positive")
        self._set([torch.zeros((pages, kv_heads, 36 * head_dim), dtype=torch.uint8, device=device) for _ in range(layers)],
                  torch.full((sequences, columns), -1, dtype=torch.int32, device=device), torch.zeros(sequences, dtype=torch.int32, device=device))
        self._held = [[] for _ in range(sequences)]
        self._free = list(range(pages - 1, -1, -1))

    @classmethod
    def over(cls, pools, table, lengths):
        """A cache on tensors that the caller keeps and pages that the caller hands out (add_pages() then has none)."""
        c = cls.__new__(cls)
        c._set(pools, table, lengths)
        c._held, c._free = None, []
        return c

    def _set(self, pools, table, lengths):
        shape = pools[0].shape
        H = shape[-1] // 36
        _check(len(shape) == 3 and shape[-1] == 36 * H and H in (64, 128) and all(p.dtype == torch.uint8 and p.shape == shape and p.is_contiguous() and
                                                                                 p.device == pools[0].device for p in pools),
               "Int4Cache: pools must be contiguous uint8 [pages, kv_heads, 36 * head size] of one shape, head size 64 or 128")
        _check(table.dtype == torch.int32 and table.dim() == 2 and table.is_contiguous() and table.numel() > 0 and table.device == pools[0].device,
               "Int4Cache: the table must be contiguous int32 [sequences, columns]")
        _check(lengths.dtype == torch.int32 and lengths.shape == table.shape[:1] and lengths.is_contiguous() and lengths.device == pools[0].device,
               "Int4Cache: lengths must be int32 [sequences]")
        self.pools, self.table, self.lengths = pools, table, lengths
        self.pages, self.kv_heads, self.head_dim, self.B = shape[0], shape[1], H, table.shape[0]
        self._structs = {}

    def layer(self, i):
        """The ctypes block of layer i."""
        s = self._structs.get(i)
        if s is None:
            s = self._structs[i] = _Int4CacheStruct(self.pools[i].data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(), self.pages,
                                                    self.table.shape[1], self.B, self.kv_heads, self.head_dim)
        return s

    def add_pages(self, tokens):
        """Room for tokens[b] tokens of sequence b in all (a list, or one number for every sequence): missing pages come from the
        pool. On the host; the table goes to the device in one copy, in the order of the stream."""
        _check(self._held is not None, "Int4Cache: a cache over the caller's tensors has no pages to hand out")
        tokens = [tokens] * self.B if isinstance(tokens, int) else list(tokens)
        _check(len(tokens) == self.B, f"Int4Cache: {len(tokens)} sizes for {self.B} sequences")
        need = [max(-(-n // S2) - len(h), 0) for n, h in zip(tokens, self._held)]
        _check(all(len(h) + k <= self.table.shape[1] for k, h in zip(need, self._held)), f"Int4Cache: a sequence passes {self.table.shape[1]} pages")
        _check(sum(need) <= len(self._free), f"Int4Cache: {sum(need)} pages are needed, {len(self._free)} are free")
        for k, h in zip(need, self._held):
            h.extend(self._free.pop() for _ in range(k))
        if sum(need):
            rows = [h + [-1] * (self.table.shape[1] - len(h)) for h in self._held]
            self.table.copy_(torch.tensor(rows, dtype=torch.int32))

    def release(self, b):
        """Sequence b is over: its pages are free, its length is 0."""
        _check(self._held is not None, "Int4Cache: a cache over the caller's tensors has no pages to take back")
        self._free.extend(reversed(self._held[b]))
        self._held[b] = []
        self.table[b].fill_(-1)
        self.lengths[b].zero_()

    def advance(self, cu_seqlens=None):
        """The tokens of the call are cached: lengths grow by the sequences' tokens (by one without cu_seqlens)."""
        self.lengths.add_(1 if cu_seqlens is None else cu_seqlens[1:] - cu_seqlens[:-1])

    def bytes_per_token(self):
        return len(self.pools) * self.kv_heads * 36 * self.head_dim // S2


def _head_prep(name, q, k, v, T, Nq, Nkv, H, ld, q_norm, k_norm, eps, ep, pos, cache, layer, cu, q_out, k_out):
    rot = max_pos = ld_ep = norm_f32 = 0
    for w in (q_norm, k_norm):
        if w is not None:
            _check(w.numel() == H and w.is_contiguous() and w.dtype in (torch.bfloat16, torch.float32), f"{name}: norm weights must be bf16 or fp32 [{H}]")
            norm_f32 = int(w.dtype == torch.float32)
    _check(q_norm is None or k_norm is None or q_norm.dtype == k_norm.dtype, f"{name}: both norm weights must have one type")
    if ep is not None:
        _check(ep.dtype == torch.float32 and ep.dim() == 3 and ep.shape[0] == 2 and ep.is_contiguous(),
               f"{name}: the rotation table must be contiguous fp32 [2, positions, rotated values]")
        max_pos, rot = ep.shape[1], ep.shape[2]
        ld_ep = rot
        _check(pos is not None or cache is not None, f"{name}: positions are needed to rotate without a cache")
    if pos is not None:
        _check(pos.dtype == torch.int64 and pos.is_contiguous() and pos.numel() == T, f"{name}: positions must be contiguous int64, one per token")
    _check(cu is None or cache is not None, f"{name}: cu_seqlens cuts the tokens of a cache")
    st, cptr, cup = None, None, None
    if cache is not None:
        st = cache.layer(layer)
        cptr = ctypes.addressof(st)
        cup = _sequences(name, cu, cache.B, T)
    a = _HeadPrepStruct(q, k, v, _lib.ptr(q_norm), _lib.ptr(k_norm), _lib.ptr(ep), _lib.ptr(pos), cup, q_out, k_out, cptr, T, Nq, Nkv, H, ld[0], ld[1], ld[2],
                        rot, max_pos, ld_ep, eps, norm_f32)
    _lib.check(_lib.lib().tpx_head_prep(ctypes.byref(a), _lib.stream()))


def qk_norm_rope(qkv, heads, kv_heads, head_dim, q_norm=None, k_norm=None, eps=1e-6, ep=None, positions=None, cu_seqlens=None, cache=None, layer=0,
                 want_k=True, q_out=None, k_out=None):
    """The pass behind a q/k/v linear. qkv bf16 [T, (heads + 2 kv_heads) * head_dim], query heads first, then keys, then values; rows may be
    strided. Every query and key head is divided by its root mean square (sqrt(mean(x^2) + eps)) and multiplied by q_norm / k_norm
    [head_dim] (bf16 or fp32; None: no norm), then its first rot values rotate in pairs (i, i + rot / 2) by the row `position` of
    ep fp32 [2, positions, rot] (cosines, sines; None: no rotation; positions outside the table leave a head unrotated). Returns
    q [T, heads, head_dim] and k [T, kv_heads, head_dim], bf16 (k None with want_k=False).

    With a cache, k and the values also go to layer `layer` of it in 4 bits, behind the tokens that are cached (`lengths` stays:
    cache.advance() after the last layer), and `positions` defaults to the tokens' places in the cache."""
    name = "qk_norm_rope"
    _on_device(name, qkv, q_norm, k_norm, ep, positions, cu_seqlens, q_out, k_out, cache.table if cache is not None else None)
    width = (heads + 2 * kv_heads) * head_dim
    _check(qkv.dtype == torch.bfloat16 and qkv.dim() == 2 and qkv.shape[1] == width and qkv.stride(1) == 1 and (qkv.shape[0] < 2 or qkv.stride(0) >= width),
           f"{name}: qkv must be bf16 [tokens, {width}]")
    T = qkv.shape[0]
    ld = qkv.stride(0) if T > 1 else width
    q = _output(name, q_out, (T, heads, head_dim), qkv.device)
    k = _output(name, k_out, (T, kv_heads, head_dim), qkv.device) if want_k or k_out is not None else None
    base = qkv.data_ptr()
    _head_prep(name, base, base + 2 * heads * head_dim, base + 2 * (heads + kv_heads) * head_dim, T, heads, kv_heads, head_dim, (ld, ld, ld), q_norm, k_norm, eps,
               ep, positions, cache, layer, cu_seqlens, q.data_ptr(), None if k is None else k.data_ptr())
    return q, k


def append_int4(k, v, cache, layer, cu_seqlens=None):
    """Keys and values bf16 [T, kv_heads, head_dim] (rows may be strided), ready as they are, into layer `layer` of the cache."""
    name = "append_int4"
    _on_device(name, k, v, cu_seqlens, cache.table)
    ldk, ldv = (_rows(name, n, t, cache.kv_heads, cache.head_dim) for n, t in (("k", k), ("v", v)))
    _check(k.shape == v.shape, f"{name}: k and v differ in shape")
    _head_prep(name, None, k.data_ptr(), v.data_ptr(), k.shape[0], 0, cache.kv_heads, cache.head_dim, (0, ldk, ldv), None, None, 0.0, None, None, cache, layer,
               cu_seqlens, None, None)


def read_int4(cache, layer, tokens, cu_seqlens=None, lengths=None):
    """The values that layer `layer` holds of `tokens` tokens, bf16 (k, v) [tokens, kv_heads, head_dim]: row i of sequence b is its token
    lengths[b] + i (lengths: the cache's, or another int32 [B]). With lengths of zero and cu_seqlens over the cached lengths this is the whole history."""
    name = "read_int4"
    _on_device(name, cache.table, cu_seqlens, lengths)
    st = cache.layer(layer)
    if lengths is not None:
        _check(lengths.dtype == torch.int32 and lengths.shape == cache.lengths.shape and lengths.is_contiguous(), f"{name}: lengths must be int32 [{cache.B}]")
        st = _Int4CacheStruct(st.pool, st.table, lengths.data_ptr(), st.pages, st.table_cols, st.B, st.kv_heads, st.H)
    cup = _sequences(name, cu_seqlens, cache.B, tokens)
    k, v = (torch.empty((tokens, cache.kv_heads, cache.head_dim), dtype=torch.bfloat16, device=cache.table.device) for _ in range(2))
    _lib.check(_lib.lib().tpx_int4_read(ctypes.byref(st), cup, tokens, k.data_ptr(), v.data_ptr(), _lib.stream()))
    return k, v


def attention_int4(q, cache, layer, cu_seqlens=None, causal=True, scale=None, out=None):
    """Attention of the call's tokens q bf16 [T, heads, head_dim] over their sequences in layer `layer` of the cache, the call's own
    keys and values (appended before) included: softmax(q k^T scale) v, bf16 like q. Token i of sequence b sees the tokens up to
    its own place lengths[b] + i, or, with causal=False, all of its sequence. A token that sees none (no page) gives zeros."""
    name = "attention_int4"
    _on_device(name, q, cu_seqlens, out, cache.table)
    _check(q.dim() == 3 and q.shape[1] > 0 and q.shape[1] % cache.kv_heads == 0, f"{name}: q must be bf16 [tokens, heads, {cache.head_dim}], heads a multiple of {cache.kv_heads}")
    T, Nq, H = q.shape
    ldq = _rows(name, "q", q, Nq, cache.head_dim)
    cup = _sequences(name, cu_seqlens, cache.B, T)
    o = _output(name, out, (T, Nq, H), q.device)
    L = _lib.lib()
    nb = L.tpx_int4_attention_scratch_bytes(T, cache.B, Nq, cache.kv_heads, H)
    sc = torch.empty(nb, dtype=torch.uint8, device=q.device)  # of this call alone: calls on two streams, and two graphs, share nothing
    a = _Int4AttentionStruct(q.data_ptr(), ctypes.addressof(cache.layer(layer)), cup, o.data_ptr(), sc.data_ptr(), nb, T, Nq, ldq,
                             H ** -0.5 if scale is None else scale, int(causal))
    _lib.check(L.tpx_int4_attention(ctypes.byref(a), _lib.stream()))
    return o


def attention_packed(q, k, v, cu_seqlens, causal=True, scale=None, out=None):
    """Attention over whole prompts laid end to end: q bf16 [T, heads, H], k and v [T, kv_heads, H] (rows may be strided, as views of a
    q/k/v linear's output are; H 64 or 128; up to 128 heads per key head): softmax(q k^T scale) v within each sequence, where token i
    sees the tokens 0 .. i, or with causal=False all of them. bf16 [T, heads, H]; rows of no sequence are not written."""
    name = "attention_packed"
    _on_device(name, q, k, v, cu_seqlens, out)
    _check(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and k.shape[0] == q.shape[0] and k.shape[1] > 0 and q.shape[1] % k.shape[1] == 0,
           f"{name}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    T, Nq, H = q.shape
    Nkv = k.shape[1]
    ld = _rows(name, "q", q, Nq, H), _rows(name, "k", k, Nkv, H), _rows(name, "v", v, Nkv, H)
    _check(cu_seqlens is not None, f"{name}: cu_seqlens is needed")
    cup = _sequences(name, cu_seqlens, None, T)
    o = _output(name, out, (T, Nq, H), q.device)
    a = _PackedAttentionStruct(q.data_ptr(), k.data_ptr(), v.data_ptr(), cup, o.data_ptr(), T, cu_seqlens.numel() - 1, Nq, Nkv, H, *ld,
                               H ** -0.5 if scale is None else scale, int(causal))
    _lib.check(_lib.lib().tpx_packed_attention(ctypes.byref(a), _lib.stream()))
    return o
