"""Sequences of different lengths laid end to end, without padding, and a KV cache that is held in 4 bits: the pass behind the
q/k/v linear (head norms, rotation, append), attention over whole prompts and attention of a few new tokens over the cache, on the
kernels of include/tpx_packed.h. They stand beside the padded batches and the bf16 pages of _tpp_attn.

Token rows [T, ...] are cut into sequences by cu_seqlens (int32 [B + 1] on the device, not falling: sequence b has the rows cu[b] .. cu[b + 1] - 1);
without it row b is the one token of sequence b. Rows outside every sequence are read by nobody, and an output that the caller
passes has theirs left as they were. Nothing here waits for the device, so all of it can be recorded in a CUDA graph."""
import torch

from .. import _lib

S2 = 32       # tokens of a page


def _check(cond, text):
    if not cond:
        raise _lib.TpxError(text)


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
        with torch.inference_mode(False):  # whose tensors would not count their changes
            lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._set([torch.zeros((pages, kv_heads, 36 * head_dim), dtype=torch.uint8, device=device) for _ in range(layers)],
                  torch.full((sequences, columns), -1, dtype=torch.int32, device=device), lengths)
        self._new = lengths._version
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
        self._pools, self._table, self._lengths = tuple(pools), table, lengths
        self.B = table.shape[0]
        self._layers = {}
        self._new = None
        self.layer(0)

    # changed in place only: the operators keep their addresses
    pools = property(lambda self: self._pools)
    table = property(lambda self: self._table)
    lengths = property(lambda self: self._lengths)

    def layer(self, i):
        """What the operators take for layer i: its addresses and sizes, checked once (the tensors are this object's)."""
        s = self._layers.get(i)
        if s is None:
            s = self._layers[i] = _lib.torch_ops().cache_bytes(self._pools[i], self._table, self._lengths)
        return s

    def is_new(self):
        """Whether it is certain, without a look at the device, that nothing is cached: lengths that this object has made and that nobody has written
        to since. Not while a CUDA graph is recorded, which may be replayed later."""
        return self._new is not None and self.lengths._version == self._new and not (self.lengths.is_cuda and torch.cuda.is_current_stream_capturing())

    @property
    def pages(self):
        return self.pools[0].shape[0]

    @property
    def kv_heads(self):
        return self.pools[0].shape[1]

    @property
    def head_dim(self):
        return self.pools[0].shape[2] // 36

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
        """The tokens of the call are cached: lengths grow by the sequences' tokens. Without cu_seqlens by one, where a sequence has a page:
        a slot that was released, or that holds nothing yet, stays at 0 while the others decode."""
        _check(cu_seqlens is None or cu_seqlens.shape == (self.B + 1,), f"Int4Cache: cu_seqlens is not that of {self.B} sequences")
        self.lengths.add_(self.table.amax(1) >= 0 if cu_seqlens is None else cu_seqlens[1:] - cu_seqlens[:-1])

    def bytes_per_token(self):
        return len(self.pools) * self.kv_heads * 36 * self.head_dim // S2


def qk_norm_rope(qkv, heads, kv_heads, head_dim, q_norm=None, k_norm=None, eps=1e-6, ep=None, positions=None, cu_seqlens=None, cache=None, layer=0,
                 want_k=True, q_out=None, k_out=None):
    """The pass behind a q/k/v linear. qkv bf16 [T, (heads + 2 kv_heads) * head_dim], query heads first, then keys, then values; rows may be
    strided. Every query and key head is divided by its root mean square (sqrt(mean(x^2) + eps)) and multiplied by q_norm / k_norm
    [head_dim] (bf16 or fp32; None: no norm), then its first rot values rotate in pairs (i, i + rot / 2) by the row `position` of
    ep fp32 [2, positions, rot] (cosines, sines; None: no rotation; positions outside the table leave a head unrotated). Returns
    q [T, heads, head_dim] and k [T, kv_heads, head_dim], bf16 (k None with want_k=False).

    With a cache, k and the values also go to layer `layer` of it in 4 bits, behind the tokens that are cached (`lengths` stays:
    cache.advance() after the last layer), and `positions` defaults to the tokens' places in the cache."""
    return _lib.torch_ops().head_prep(qkv, heads, kv_heads, head_dim, q_norm, k_norm, eps, ep, positions, cu_seqlens, cache and cache.layer(layer),
                                      want_k, q_out, k_out)


def append_int4(k, v, cache, layer, cu_seqlens=None):
    """Keys and values bf16 [T, kv_heads, head_dim] (rows may be strided), ready as they are, into layer `layer` of the cache."""
    _lib.torch_ops().append(k, v, cache.layer(layer), cu_seqlens)


def read_int4(cache, layer, tokens, cu_seqlens=None, lengths=None):
    """The values that layer `layer` holds of `tokens` tokens, bf16 (k, v) [tokens, kv_heads, head_dim]: row i of sequence b is its token
    lengths[b] + i (lengths: the cache's, or another int32 [B]). With lengths of zero and cu_seqlens over the cached lengths this is the whole history."""
    return _lib.torch_ops().read(cache.layer(layer), tokens, cu_seqlens, lengths)


def attention_int4(q, cache, layer, cu_seqlens=None, causal=True, scale=None, out=None, behind=False):
    """Attention of the call's tokens q bf16 [T, heads, head_dim] over their sequences in layer `layer` of the cache, the call's own
    keys and values (appended before) included: softmax(q k^T scale) v, bf16 like q. Token i of sequence b sees the tokens up to
    its own place lengths[b] + i, or, with causal=False, all of its sequence. A token that sees none (no page) gives zeros.
    behind=True: for the sequences alone that have tokens cached before the call; rows of the others are not written."""
    return _lib.torch_ops().int4_attention(q, cache.layer(layer), cu_seqlens, causal, scale, out, behind)


def attention_packed(q, k, v, cu_seqlens, causal=True, scale=None, out=None, lengths=None):
    """Attention over whole prompts laid end to end: q bf16 [T, heads, H], k and v [T, kv_heads, H] (rows may be strided, as views of a
    q/k/v linear's output are; H 64 or 128; up to 128 heads per key head; scale > 0, H^-1/2 by default): softmax(q k^T scale) v within each sequence, where token i
    sees the tokens 0 .. i, or with causal=False all of them. bf16 [T, heads, H]; rows of no sequence are not written. With lengths
    (int32 [B], the tokens cached before the call) only for the sequences that have none; rows of the others are not written: they are
    attention_int4(..., behind=True)'s."""
    return _lib.torch_ops().packed_attention(q, k, v, cu_seqlens, causal, scale, out, lengths)
