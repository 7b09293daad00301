"""Paged key / value caches on raw torch tensors: kernels of `csrc/paged_kv.cu` and `csrc/paged_attention.cu` on CUDA, torch
on the CPU (which is what the tests compare with).

A layer's pools are k, v [pages, Hkv, page, D] and, for 8 bits, scales [pages, Hkv, page] of uint8: a row stands for its e4m3
numbers times 2^(scale - 127).  `table` [B, per], `lengths` [B] and `counts` [B] (or None) are int32; token s of sequence b stands
at position lengths[b] - counts[b] + s, for s < counts[b] (clipped to 0 .. S) and positions from 0 on."""
import ctypes
import functools

import torch

from . import native as N

E4M3 = torch.float8_e4m3fn
CACHE_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, E4M3: 8}


# ------------------------------------------------------------------------------------------------
# the CPU's form
# ------------------------------------------------------------------------------------------------
def power_of_two(e):
    """2^e of int32 numbers from -127 (taken as 0) to 127."""
    return ((e + 127) << 23).view(torch.float32)


def quantise(x):
    """float32 x [..., D] -> (e4m3 [..., D], uint8 [...]): the smallest e >= -126 with the largest finite |x| <= 448 * 2^e,
    stored as e + 127; infinities and NaN become NaN."""
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1).view(torch.int32)
    e = ((top >> 23) - 135 + ((top & 0x7fffff) > 0x600000).int()).clamp(min=-126)
    y = torch.where(fine, x * power_of_two(-e).unsqueeze(-1), torch.full_like(x, float("nan")))
    return y.to(E4M3), (e + 127).to(torch.uint8)


def _counts(counts, B, S):
    return torch.full((B,), S) if counts is None else counts.long().clamp(0, S)


def _slots(layer, table, b, pos):
    """(pages, places) of the positions `pos` of the sequences `b`."""
    page, per = layer.page_size, table.shape[1]
    if pos.numel() and int(pos.max()) >= per * page:
        raise IndexError(f"position {int(pos.max())} of a sequence whose page table has room for {per * page} tokens")
    i = torch.div(pos, page, rounding_mode="floor")
    pages = table[b, i].long()
    bad = (pages < 0) | (pages >= layer.k.shape[0])
    if bool(bad.any()):
        raise IndexError(f"page {int(pages[bad][0])} of a cache of {layer.k.shape[0]} pages")
    return pages, pos - i * page


def _new_tokens(lengths, counts, B, S):
    """(sequence, token of the call, position) of the tokens that are real."""
    n = _counts(counts, B, S)
    s = torch.arange(S)
    pos = lengths.long().clamp(min=0)[:, None] - n[:, None] + s
    b, s = torch.nonzero((s < n[:, None]) & (pos >= 0), as_tuple=True)
    return b, s, pos[b, s]


def _store(layer, pages, places, k, v):
    heads = torch.arange(k.shape[1])
    at = (pages[:, None], heads, places[:, None])
    for pool, scales, x in ((layer.k, layer.k_scale, k), (layer.v, layer.v_scale, v)):
        if scales is None:
            pool[at] = x.to(pool.dtype)
        else:
            x, e = quantise(x.float())
            pool.view(torch.uint8)[at] = x.view(torch.uint8)
            scales[at] = e


def _rows(pool, scales, pages, places):
    """[n, Hkv, D] float32 rows of a pool."""
    if scales is None:
        return pool[pages, :, places].float()
    x = pool.view(torch.uint8)[pages, :, places].view(E4M3).float()
    return x * power_of_two(scales[pages, :, places].int() - 127).unsqueeze(-1)


def _put_cpu(q, k, v, tables, layer, table, lengths, counts):
    B, S = k.shape[:2]
    b, s, pos = _new_tokens(lengths, counts, B, S)
    if tables is not None and pos.numel() and int(pos.max()) >= tables[0].shape[0]:
        raise IndexError(f"position {int(pos.max())} behind rotation tables of {tables[0].shape[0]} positions")
    pages, places = _slots(layer, table, b, pos)
    if tables is None:
        _store(layer, pages, places, k[b, s], v[b, s])
        return None
    cos, sin = (t[pos].float().unsqueeze(1) for t in tables)
    half = k.shape[-1] // 2

    def rotated(x):
        x = x.float()
        return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin

    out = torch.zeros(q.shape, dtype=q.dtype)
    out[b, s] = rotated(q[b, s]).to(q.dtype)
    _store(layer, pages, places, rotated(k[b, s]), v[b, s])
    return out


def _read_cpu(layer, table, lengths, L, dtype):
    B = table.shape[0]
    at = torch.arange(L)
    b, pos = torch.nonzero(at < lengths.long()[:, None], as_tuple=True)
    pages, places = _slots(layer, table, b, pos)
    outs = []
    for pool, scales in ((layer.k, layer.k_scale), (layer.v, layer.v_scale)):
        out = torch.zeros(B, L, pool.shape[1], pool.shape[3], dtype=dtype)
        out[b, pos] = _rows(pool, scales, pages, places).to(dtype)
        outs.append(out)
    return outs


def _attention_cpu(q, layer, table, lengths, counts, scale):
    B, S, Hq, D = q.shape
    Hkv, n = layer.k.shape[1], _counts(counts, B, S)
    out = torch.zeros(B, S, Hq, D)
    for b in range(B):
        start = max(int(lengths[b]), 0) - int(n[b])
        end = start + int(n[b])
        if n[b] == 0 or end <= 0:
            continue
        at = torch.arange(end)
        pages, places = _slots(layer, table, torch.full_like(at, b), at)
        k, v = (_rows(pool, sc, pages, places).transpose(0, 1) for pool, sc in ((layer.k, layer.k_scale), (layer.v, layer.v_scale)))
        rows = int(n[b])
        x = q[b, :rows].float().reshape(rows, Hkv, Hq // Hkv, D).permute(1, 0, 2, 3)
        z = torch.einsum("hsgd,hnd->hsgn", x, k) * scale
        seen = at <= start + torch.arange(rows)[:, None]
        z = z.masked_fill(~seen[None, :, None], float("-inf"))
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(top == float("-inf"), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        # (a key that a row does not see is no part of its sum, whatever its value holds)
        vs = torch.where(seen[:, :, None], v[:, None], torch.zeros_like(v[:, None]))
        o = torch.einsum("hsgn,hsnd->hsgd", p, vs)
        o = torch.where(total == 0, torch.zeros_like(o), o / total)
        out[b, :rows] = o.permute(1, 0, 2, 3).reshape(rows, Hq, D)
    return out.to(q.dtype)


# ------------------------------------------------------------------------------------------------
# the kernels
# ------------------------------------------------------------------------------------------------
class Pools(ctypes.Structure):
    """One layer's pools as the kernels' entry points take them (`PagedPools` in csrc/paged_common.cuh)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + \
               [(n, ctypes.c_int) for n in ("pages", "kv_heads", "page", "head_dim", "type")]


def pools_of(k, v, k_scale, v_scale):
    return Pools(k.data_ptr(), v.data_ptr(), N._ptr(k_scale), N._ptr(v_scale), *k.shape, CACHE_TYPES[k.dtype])


def _dense_last(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _launch(what, index, dev, fn, *args):
    """Calls an entry point that ends in (status, stream) with `dev` as the current device."""
    if index == torch.cuda.current_device():
        N._chk(fn(*args, N.status_tensor(dev).data_ptr(), N._st()), what)
    else:
        with torch.cuda.device(index):
            N._chk(fn(*args, N.status_tensor(dev).data_ptr(), N._st()), what)


def write(k, v, layer, table, lengths, counts):
    """Keys and values [B, S, Hkv, D] into their pages."""
    index, pools, _, _ = layer._call
    if index < 0:
        _put_cpu(None, k, v, None, layer, table, lengths, counts)
        return
    k, v = _dense_last(k), _dense_last(v)
    (kb, ks, kh, _), (vb, vs, vh, _) = k.stride(), v.stride()
    _launch("paged_write", index, k.device, N.lib().gb_paged_write, pools, k.data_ptr(), kb, ks, kh, v.data_ptr(), vb, vs, vh,
            table.data_ptr(), lengths.data_ptr(), N._ptr(counts), k.shape[0], k.shape[1], table.shape[1], N._DT[k.dtype])


def rope_write(y, tables, Hq, layer, table, lengths, counts):
    """Rotated queries [B, S, Hq, D] from y [B, S, (Hq + 2 Hkv) D], with the rotated keys and the values put into their pages;
    zeros for tokens that are none.  `tables`: cos, sin [positions, D] float32."""
    index, pools, (_, Hkv, _, D), _ = layer._call
    if index < 0:
        x = y.unflatten(-1, (Hq + 2 * Hkv, D))
        return _put_cpu(x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], tables, layer, table, lengths, counts)
    y = _dense_last(y)
    B, S, _ = y.shape
    sb, ss, _ = y.stride()
    cos, sin = tables
    out = torch.empty(B, S, Hq, D, dtype=y.dtype, device=y.device)
    _launch("paged_qkv_rope", index, y.device, N.lib().gb_paged_qkv_rope, pools, y.data_ptr(), sb, ss, out.data_ptr(), cos.data_ptr(),
            sin.data_ptr(), cos.shape[0], table.data_ptr(), lengths.data_ptr(), N._ptr(counts), B, S, Hq, table.shape[1],
            N._DT[y.dtype])
    return out


def read(layer, table, lengths, L, dtype):
    """(k, v) [B, L, Hkv, D] of `dtype`, zeros behind each sequence's end."""
    index, pools, (_, Hkv, _, D), _ = layer._call
    if index < 0:
        return _read_cpu(layer, table, lengths, L, dtype)
    B, per = table.shape
    dev = table.device
    k = torch.empty(B, L, Hkv, D, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _launch("paged_read", index, dev, N.lib().gb_paged_read, pools, k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(),
            B, L, per, N._DT[dtype])
    return k, v


@functools.lru_cache(maxsize=256)
def _workspace(device_index, *sizes):
    with torch.cuda.device(device_index):
        return N.lib().gb_paged_attention_workspace(*sizes)


def attention(q, layer, table, lengths, counts, scale):
    """softmax(scale q k^T) v of the tokens q [B, S, Hq, D] over the pages of their sequences -> [B, S, Hq, D]."""
    index, at, (pages, Hkv, page, D), cdt = layer._call
    if index < 0:
        return _attention_cpu(q, layer, table, lengths, counts, scale)
    B, S, Hq, _ = q.shape
    dev, per, dt = q.device, table.shape[1], N._DT[q.dtype]
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(q)
    words = _workspace(index, B, S, Hq, Hkv, D, page, pages, per, dt, cdt)
    work = torch.empty(words, dtype=torch.float32, device=dev) if words else None
    _launch("paged_attention", index, dev, N.lib().gb_paged_attention, at, q.data_ptr(), out.data_ptr(), table.data_ptr(),
            lengths.data_ptr(), N._ptr(counts), B, S, Hq, per, scale, dt, N._ptr(work))
    return out
