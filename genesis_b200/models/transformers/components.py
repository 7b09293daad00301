"""Rotary embedding helpers. Parity: reference `genesis/models/transformers/components.py:30-179`.

`RotaryEmbedding` keeps `[max_pos, dim]` cos/sin caches (halves duplicated, i.e.
`cat(freqs, freqs)`), registered as non-persistent buffers, extended on demand.
`apply_rotary_pos_emb` keeps the reference signature on `[B, H, S, D]` tensors;
`apply_rope` is the fused path on `[B, S, H, D]` (one kernel per tensor instead of ~14).
"""
import numpy as np
import torch

from ...tensor import Tensor, tensor
from ... import nn
from ...nn import functional as F

# The reference selects a PyTorch re-implementation of these classes with NANOCHAT_BACKEND=torch; here there is one
# implementation, and the name stays for code that reads it.
BACKEND = "genesis"



def find_multiple(n, k):
    return n if n % k == 0 else n + k - (n % k)


def rotate_half(x):
    d = x.shape[-1] // 2
    return F.cat((-x[..., d:], x[..., :d]), dim=-1)


class _Unseen:
    """Pairs of tables that are none of a module's buffers.  A module looks for those in lists, tuples and dicts too, and saves,
    converts and moves what it finds; it does not look in here."""
    __slots__ = ("_pairs",)

    def __init__(self):
        self._pairs = []

    def __len__(self):
        return len(self._pairs)

    def __getitem__(self, i):
        return self._pairs[i]

    def append(self, pair):
        self._pairs.append(pair)


class RotaryEmbedding(nn.Module):
    def __init__(self, dim, max_position_embeddings=2048, base=10000.0, device=None):
        super().__init__()
        self.dim, self.base = dim, float(base)
        self.max_position_embeddings = max_position_embeddings
        self._device = device
        self._outgrown = _Unseen()      # what larger tables have replaced: captured steps go on reading it
        self._exact = _Unseen()         # tables in 32 bits of a module that was converted to 16
        self._build(max_position_embeddings)

    def _values(self, seq_len, dev):
        """(inverse frequencies, cos, sin) in 32 bits."""
        inv = 1.0 / (self.base ** (np.arange(0, self.dim, 2, dtype=np.float64) / self.dim))
        t = np.arange(seq_len, dtype=np.float64)
        freqs = np.outer(t, inv)
        emb = np.concatenate([freqs, freqs], axis=-1)
        return [tensor(x.astype(np.float32), device=dev) for x in (inv, np.cos(emb), np.sin(emb))]

    def _build(self, seq_len):
        dev = self._device
        old = self.__dict__.get("cos_cached")
        if old is not None:
            dev = old.device
        values = self._values(seq_len, dev)      # (nothing changes where this fails, as it does while a stream is captured)
        if old is not None:
            self.__dict__.setdefault("_outgrown", _Unseen()).append((old, self.sin_cached))     # (a module that was pickled without)
        self.max_seq_len_cached = seq_len
        for name, t in zip(("inv_freq", "cos_cached", "sin_cached"), values):
            self.register_buffer(name, t, persistent=False)

    def reserve(self, seq_len):
        """Makes the tables reach so many positions.  They at least double, so that all outgrown ones together are no larger."""
        if seq_len > self.max_seq_len_cached:
            self._build(max(seq_len, 2 * self.max_seq_len_cached))

    def tables32(self):
        """(cos, sin) in 32 bits, which the paged operators take, also where the module was converted to 16 (in bfloat16 a cosine
        is up to 2^-9 off, at every position)."""
        cos = self.cos_cached
        if cos._t.dtype is torch.float32:
            return cos, self.sin_cached
        kept = self.__dict__.setdefault("_exact", _Unseen())
        if not len(kept) or kept[-1][0].shape != cos.shape or kept[-1][0].device != cos.device:
            kept.append(tuple(self._values(cos.shape[0], cos.device)[1:]))
        return kept[-1]

    def forward(self, x=None, seq_len=None):
        if seq_len is not None:
            self.reserve(seq_len)
        if seq_len is None:
            return self.cos_cached, self.sin_cached
        return self.cos_cached[:seq_len], self.sin_cached[:seq_len]


def apply_rotary_pos_emb(q, k, cos, sin, position_ids=None):
    """q, k: [B, H, S, D]; cos, sin: [S or max_pos, D]; position_ids: [B, S] or None."""
    if position_ids is not None:
        cos = F.unsqueeze(cos[position_ids], 1)
        sin = F.unsqueeze(sin[position_ids], 1)
    else:
        S = q.shape[-2]
        cos = F.reshape(cos[:S], (1, 1, S, cos.shape[-1]))
        sin = F.reshape(sin[:S], (1, 1, S, sin.shape[-1]))
    q_embed = q * cos + rotate_half(q) * sin
    k_embed = k * cos + rotate_half(k) * sin
    return q_embed, k_embed


def apply_rope(x, rotary, position_ids=None):
    """Fused rotate-half RoPE on x [B, S, H, D]."""
    S = x.shape[1]
    rotary.reserve(S)
    pos = None if position_ids is None else position_ids
    return F.rope(x, rotary.cos_cached, rotary.sin_cached, pos)


def paged_self_attention(y, rotary, num_heads, cache, page_table, lengths, counts=None, prompt=False):
    """Self-attention of a fused projection's y [B, S, (num_heads + 2 Hkv) D] through one layer of a paged cache -> [B, S,
    num_heads * D].  The tokens' keys and values are put into the cache; with `prompt` the sequences have no others and the real
    tokens stand first in each row (`prompt_first`), and the flash attention over the call's own keys takes the place of reading
    them back."""
    B, S, _ = y.shape
    rotary.reserve(max(S, page_table.shape[1] * cache.page_size))
    cos, sin = rotary.tables32()
    if prompt:
        q, k, v = F.qkv_rope(y, cos, sin, None, num_heads, cache.num_kv_heads, cache.head_dim)
        F.paged_kv_write(k, v, cache, page_table, lengths, counts)
        o = F.flash_attention(q, k, v, causal=True)
    else:
        q = F.paged_qkv_rope(y, cos, sin, cache, page_table, lengths, num_heads, counts)
        o = F.paged_attention(q, cache, page_table, lengths, counts)
    return F.reshape(o, (B, S, num_heads * cache.head_dim))


def prompt_first(idx, lengths):
    """Prompts [B, S] whose real tokens are each row's last lengths[b] -> (idx with them first, how many they are [B], and for
    `in_places` where each place's token went [B, S]).  Nothing waits for the device."""
    t = lengths._t if isinstance(lengths, Tensor) else None
    if t is None or t.shape != idx.shape[:1] or t.device != idx._t.device:
        return idx, None, None                   # (the operators say what is wrong with them)
    S = idx.shape[1]
    n, step = t.clamp(0, S), torch.arange(S, device=t.device)
    pad = (S - n).long()[:, None]
    idx = Tensor._wrap(torch.gather(idx._t, 1, (step + pad) % max(S, 1)))
    return idx, Tensor._wrap(n), Tensor._wrap((step - pad) % max(S, 1))


def last_tokens(x, counts=None):
    """[B, S, H] -> [B, 1, H]: each sequence's last real token (its last, without `counts`)."""
    if counts is None or x.shape[1] == 1:
        return x[:, x.shape[1] - 1:]
    at = (counts._t.long() - 1).clamp(0, x.shape[1] - 1)
    return F.unsqueeze(x[Tensor._wrap(torch.arange(x.shape[0], device=at.device)), Tensor._wrap(at)], 1)


def in_places(x, places=None):
    """x [B, S, H] of the tokens that `prompt_first` gave, in the order that it took them from."""
    if places is None:
        return x
    return x[Tensor._wrap(torch.arange(x.shape[0], device=places._t.device).unsqueeze(1)), places]
