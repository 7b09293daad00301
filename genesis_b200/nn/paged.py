"""Paged key / value caches: the memory that a decoder answers from.

Keys and values live in pages of `page_size` tokens; a page table says which pages hold a sequence, so sequences of any
lengths share one pool, grow page by page, and may share the pages of a common beginning.  The reference keeps no such cache
(its MoE attention concatenates the past, `models/transformers/moe.py:504-530`; its dense model encodes its prompt anew for
every token).  The operators on a layer are `nn.functional.paged_kv_write`, `paged_qkv_rope`, `paged_kv_read` and
`paged_attention`."""
import ctypes

import torch

from ..device import as_torch_device
from ..dtypes import DType
from ..ops.paged import CACHE_TYPES, E4M3, pools_of
from ..tensor import Tensor

__all__ = ["PagedKVCache", "PagedKVLayer"]


def _cache_dtype(dtype):
    names = {str(t).replace("torch.", ""): t for t in CACHE_TYPES}
    if isinstance(dtype, DType):
        dtype = dtype.name
    t = names.get(dtype) if isinstance(dtype, str) else dtype
    if t not in CACHE_TYPES:
        raise ValueError(f"a cache holds one of {', '.join(names)}, got {dtype!r}")
    return t


def _positive(name, x):
    if isinstance(x, bool) or not isinstance(x, int) or not 0 < x < 2 ** 31:
        raise ValueError(f"PagedKVCache: {name} must be a positive 32-bit int, got {x!r}")
    return x


class PagedKVLayer:
    """The pools of one decoder layer: raw k, v [pages, KV heads, page size, head dim], and in 8 bits k_scale, v_scale
    [pages, KV heads, page size] (uint8; a row stands for its e4m3 numbers times 2^(scale - 127)), else None."""
    __slots__ = ("_k", "_v", "_k_scale", "_v_scale", "_pools", "_call")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if k.dim() != 4 or v.shape != k.shape or k.dtype not in CACHE_TYPES or v.dtype != k.dtype or k.shape[2] % 16 or 0 in k.shape:
            raise ValueError(f"PagedKVLayer: k and v must be pools [pages, KV heads, page size, head dim] of one type, the page size "
                             f"a multiple of 16, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        scales = [t for t in (k_scale, v_scale) if t is not None]
        if len(scales) != (2 if k.dtype == E4M3 else 0) or any(t.shape != k.shape[:3] or t.dtype != torch.uint8 for t in scales):
            raise ValueError("PagedKVLayer: pools of 8 bits, and no others, have scales [pages, KV heads, page size] of uint8")
        for t in (k, v, *scales):
            if not t.is_contiguous() or t.data_ptr() % 16 or t.device != k.device:
                raise ValueError("PagedKVLayer: pools and scales must be contiguous, start on 16 bytes and be on one device")
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        # what every call passes on (so the pools cannot be exchanged): device, the kernels' description, sizes, type
        self._pools = pools_of(k, v, k_scale, v_scale)
        self._call = (k.get_device(), ctypes.addressof(self._pools), tuple(k.shape), CACHE_TYPES[k.dtype])

    def __reduce__(self):              # (torch does not pickle e4m3)
        raw = [t.view(torch.uint8) if t.dtype == E4M3 else t for t in (self._k, self._v)]
        return _layer_of, (*raw, self._k_scale, self._v_scale)

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)

    @property
    def num_pages(self):
        return self.k.shape[0]

    @property
    def num_kv_heads(self):
        return self.k.shape[1]

    @property
    def page_size(self):
        return self.k.shape[2]

    @property
    def head_dim(self):
        return self.k.shape[3]

    def __repr__(self):
        return (f"PagedKVLayer({self.num_pages} pages of {self.page_size} tokens, {self.num_kv_heads} x {self.head_dim}, "
                f"{str(self.k.dtype).replace('torch.', '')}, {self.k.device})")


def _layer_of(k, v, k_scale, v_scale):
    return PagedKVLayer(*((k, v) if k_scale is None else (k.view(E4M3), v.view(E4M3))), k_scale, v_scale)


class PagedKVCache:
    """Pages for the keys and values of all layers of a decoder, and which of them are free.

    `dtype`: float32, float16, bfloat16 or float8_e4m3fn (8 bits, with a power of two for every token and head).
    `page_size` is a multiple of 16.  `cache[i]` is layer i, what the operators take; all layers use the same page numbers.

        pages = cache.allocate([len_a + room, len_b + room])     # page numbers of each sequence
        table = cache.page_table(pages)                          # int32 Tensor [2, most pages], -1 where there is none
        ...
        cache.release(pages)

    A table may name a page for several sequences (a common beginning), for reading; whose page it is remains the caller's to know.
    Like any tensor's, the pools' memory is to be waited for by another stream that reads or writes it; page numbers are handed out
    on the host and nothing here waits for the device."""

    def __init__(self, num_pages, num_kv_heads, head_dim, page_size=64, num_layers=1, dtype="bfloat16", device=None):
        P, H, D, page, L = (_positive(n, x) for n, x in (("num_pages", num_pages), ("num_kv_heads", num_kv_heads),
                                                         ("head_dim", head_dim), ("page_size", page_size),
                                                         ("num_layers", num_layers)))
        if page % 16:
            raise ValueError(f"PagedKVCache: page_size must be a multiple of 16, got {page}")
        self.dtype, self.page_size, self.num_pages = _cache_dtype(dtype), page, P
        dev = as_torch_device(device)
        raw = torch.uint8 if self.dtype == E4M3 else self.dtype

        def pool():
            return torch.zeros(P, H, page, D, dtype=raw, device=dev).view(self.dtype)

        def scales():
            return torch.zeros(P, H, page, dtype=torch.uint8, device=dev) if self.dtype == E4M3 else None

        self.layers = [PagedKVLayer(pool(), pool(), scales(), scales()) for _ in range(L)]
        self._free = list(range(P - 1, -1, -1))
        self._taken = set()

    @property
    def device(self):
        return self.layers[0].k.device

    @property
    def free_pages(self):
        return len(self._free)

    def __len__(self):
        return len(self.layers)

    def __getitem__(self, i):
        return self.layers[i]

    def pages_for(self, tokens):
        """Pages that hold so many tokens."""
        if isinstance(tokens, bool) or not isinstance(tokens, int) or tokens < 0:
            raise ValueError(f"PagedKVCache: tokens must be a non-negative int, got {tokens!r}")
        return -(-tokens // self.page_size)

    def allocate(self, tokens):
        """Lists of page numbers, one with room for each of the counts of tokens."""
        pages = [[] for _ in tokens]
        self.extend(pages, tokens)
        return pages

    def extend(self, pages, tokens):
        """Adds pages to the lists until sequence i has room for tokens[i]; none is added if the cache has too few."""
        if len(pages) != len(tokens):
            raise ValueError(f"PagedKVCache: {len(pages)} sequences, {len(tokens)} counts of tokens")
        more = [max(0, self.pages_for(n) - len(p)) for p, n in zip(pages, tokens)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(more)} pages asked for, {len(self._free)} of {self.num_pages} free")
        for p, n in zip(pages, more):
            for _ in range(n):
                p.append(self._free.pop())
                self._taken.add(p[-1])

    def release(self, pages):
        """Gives the pages of finished sequences back and empties their lists."""
        every = [i for p in pages for i in p]
        if len(set(every)) != len(every) or not self._taken.issuperset(every):
            raise ValueError("PagedKVCache: a page that is not in use, or is listed twice, cannot be released")
        self._taken.difference_update(every)
        self._free.extend(reversed(every))
        for p in pages:
            p.clear()

    def page_table(self, pages, width=None):
        """The lists as an int32 Tensor [sequences, width] on the cache's device, -1 behind each list's end.  A wider table
        than the longest list leaves room for pages that follow without a table of another shape."""
        width = max([len(p) for p in pages], default=0) if width is None else width
        if any(len(p) > width for p in pages):
            raise ValueError(f"PagedKVCache: a sequence has more than {width} pages")
        rows = [list(p) + [-1] * (width - len(p)) for p in pages]
        return Tensor._wrap(torch.tensor(rows, dtype=torch.int32).reshape(len(pages), width).to(self.device))

    def __repr__(self):
        return f"PagedKVCache({len(self.layers)} layers, {self.free_pages} pages free, {self.layers[0]!r})"
