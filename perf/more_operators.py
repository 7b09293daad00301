"""A paged key-value cache and what reads it, as cases that can be measured.

Four operators of decoding, next to the flash attention and the rotary kernels that the framework has had before.  Keys and
values live in pages [pages, KV heads, page size, head dim] of one pool; a page table [B, pages of a sequence] says which pages
hold a sequence, in order (-1: none).  `lengths` [B] are the tokens of each sequence once this call's are in, `counts` [B] how many
of the call's S tokens are real (all, unless given): token s of sequence b stands at position lengths[b] - counts[b] + s.

* `paged_kv_write`: puts keys and values [B, S, KV heads, D] into their pages, in the cache's type;
* `paged_qkv_rope`: from a fused q | k | v projection's output, rotated queries, with the rotated keys and the values put into
  their pages by the same kernel;
* `paged_kv_read`: the sequences back as dense [B, longest, KV heads, D], zeros behind each sequence's end;
* `paged_attention`: attention of the newest tokens over the pages.

A cache in 8 bits holds e4m3 numbers and, for every token and KV head, the exponent e of a power of two, stored as e + 127: a row's
largest finite magnitude is at most 448 * 2^e and no smaller e has that property (-126 is the smallest).

`run` computes each case in plain torch, or with `own` through the framework; `exact` restates it in 64 bits.  Heads are those of
this repository's configurations: 14 / 2 of 64, 12 / 2 of 128, 32 / 4 of 128, 12 / 12 of 64.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
THETA = 1e6
HEADS = [(14, 2, 64), (12, 2, 128), (32, 4, 128), (12, 12, 64)]
LARGEST = 2 * 8 * 32768 * 4 * 129          # bytes of the largest listed cache


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def _case(kind, B, S, T, heads, dtype, cache, page, ragged=True, **more):
    """S new tokens (at most) of B sequences of up to T; `cache`: the type that keys and values are held in."""
    return dict(kind=kind, B=B, S=S, T=T, Hq=heads[0], Hkv=heads[1], D=heads[2], dtype=dtype, cache=cache, page=page, ragged=ragged, **more)


def listed():
    return [
        # one decoding step of a batch of 16: its queries, keys and values leave the projection for attention and the cache
        dict(_case("rope", 16, 1, 1000, HEADS[0], "bf16", "bf16", 16), name="rope_step"),
        # the prompts of a batch, as long as the training sequences
        dict(_case("rope", 8, 2048, 2048, HEADS[0], "bf16", "bf16", 64, ragged=False), name="rope_prompt"),
        # a piece of each of four prompts, some nearly at their end, into a cache of 8 bits, read back for attention over all of it
        dict(_case("rope", 4, 511, 4000, HEADS[2], "fp16", "e4m3", 64), name="rope_piece_8bit"),
        # prompts whose keys the flash attention needed too, kept in 8 bits and read back when the chat goes on
        dict(_case("write", 8, 4096, 4096, HEADS[2], "bf16", "e4m3", 64, ragged=False), name="write_prompt_8bit"),
        # three short odd sequences of a model in fp32
        dict(_case("write", 3, 77, 130, HEADS[3], "fp32", "fp32", 16), name="write_odd"),
        # a common long prefix brought back for the next piece of its prompt
        dict(_case("read", 2, 0, 32768, HEADS[0], "bf16", "bf16", 64), name="read_long"),
        # a ragged batch, held in 8 bits
        dict(_case("read", 8, 0, 5000, HEADS[2], "bf16", "e4m3", 32), name="read_8bit"),
        # one chat: a single token over 8192 keys, all latency
        dict(_case("attend", 1, 1, 8192, HEADS[0], "bf16", "bf16", 64, ragged=False), name="attend_one"),
        # a full batch of sequences of all lengths
        dict(_case("attend", 64, 1, 4096, HEADS[2], "bf16", "bf16", 64), name="attend_batch"),
        # long documents in a cache of 8 bits, the largest of all
        dict(_case("attend", 8, 1, 32768, HEADS[2], "bf16", "e4m3", 64, ragged=False), name="attend_long_8bit"),
        # five drafted tokens of four sequences, checked at once; odd lengths
        dict(_case("attend", 4, 5, 2001, HEADS[1], "fp16", "fp16", 16), name="attend_draft"),
        # a small model in fp32 with as many KV heads as query heads
        dict(_case("attend", 3, 1, 700, HEADS[3], "fp32", "fp32", 16), name="attend_fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "attend", "attend", "attend"])
    heads = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    cache = "e4m3" if dtype != "fp32" and rng.random() < 0.4 else dtype
    B, page, ragged = _log(rng, 1, 64), rng.choice([16, 32, 64, 128]), rng.random() < 0.7
    if kind in ("rope", "write"):
        S = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        T = S + _log(rng, 1, 4096)
    else:
        S = 0 if kind == "read" else rng.choice([1, 1, 1, rng.randint(2, 8)])
        T = _log(rng, 8 + S, 32768)
    while True:
        case = _case(kind, B, S, T, heads, dtype, cache, page, ragged)
        if work(case)["bytes"] <= LARGEST:
            return case
        B, S, T = (B // 2, S, T) if B > 1 else (B, (S + 1) // 2, (T + 1) // 2)


def _lengths(case):
    """(tokens of each sequence, how many of them are new)."""
    B, S, T = case["B"], case["S"], case["T"]
    lengths, counts = [], []
    for i in range(B):
        cut = (i * 2654435761 + 12345) % 1000 / 1000 if case["ragged"] and i else 0.0
        lengths.append(max(S, 1, round(T * (1 - 0.95 * cut))))
        counts.append(max(1, S - i % 3) if case["ragged"] and S > 1 and case["kind"] != "attend" else S)
    return lengths, counts


def _pages(case):
    """Pages that a sequence may have, and pages of the pool: those in use and a few of others'."""
    used = [-(-n // case["page"]) for n in _lengths(case)[0]]
    return max(used), sum(used) + 3


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _power(e):
    """2^e of whole numbers from -126 to 127, as floats of 32 bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantised(x):
    """x [..., D] in 32 bits as e4m3 bytes and exponents [...]."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = e - 9 + (m > 0.875).to(e.dtype)          # m 2^e <= 448 2^(e - 9) for m up to 448 / 512
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(min=-126)
    y = x * _power(-e).unsqueeze(-1)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, S, Hq, Hkv, D, page = (case[n] for n in ("B", "S", "Hq", "Hkv", "D", "page"))
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    lengths, counts = _lengths(case)
    per, total = _pages(case)
    order = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    table = torch.full((B, per), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(lengths):
        used = -(-n // page)
        table[b, :used] = order[at:at + used]
        at += used
    d = dict(table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV))
    if case["S"] and counts != [S] * B:
        d["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    # keys have a few strong channels, as trained models' have
    gain = 1 + 2 * (torch.rand(Hkv, 1, D, device=DEV, generator=g) > 0.97).float()
    for n in "kv":
        pool = torch.empty(total, Hkv, page, D, dtype=torch.uint8 if case["cache"] == "e4m3" else dt, device=DEV)
        if case["cache"] == "e4m3":
            d[n + "_scale"] = torch.empty(total, Hkv, page, dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // (Hkv * page * D))
        for a in range(0, total, step):
            x = normal(min(step, total - a), Hkv, page, D)
            x = x * gain if n == "k" else x
            if case["cache"] == "e4m3":
                pool[a:a + step], d[n + "_scale"][a:a + step] = _quantised(x)
            else:
                pool[a:a + step] = x
        d[n] = pool
    if case["kind"] == "rope":
        d["y"] = normal(B, S, (Hq + 2 * Hkv) * D).to(dt)
        w = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
        a = torch.arange(max(lengths), dtype=torch.float64, device=DEV)[:, None] * torch.cat([w, w])
        d["cos"], d["sin"] = a.cos().float(), a.sin().float()
    elif case["kind"] == "write":
        d["new_k"], d["new_v"] = (normal(B, S, Hkv, D) * gain.view(Hkv, D)).to(dt), normal(B, S, Hkv, D).to(dt)
    elif case["kind"] == "attend":
        d["q"] = normal(B, S, Hq, D).to(dt)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    s = dict(d, case=case, longest=max(_lengths(case)[0]))
    if not own:
        # where the new tokens go: rows of the call (b S + s) that are real, their pages and places in them
        if case["kind"] in ("rope", "write"):
            n, c = _lengths(case)
            rows = [(b * case["S"] + i, b, n[b] - c[b] + i) for b in range(case["B"]) for i in range(c[b])]
            r, b, at = torch.tensor(rows, device=DEV).unbind(1)
            s["rows"], s["at"], s["slot"] = r, at, (d["table"][b, at // case["page"]].long(), at % case["page"])
        return s
    import os
    # torch's own memory statistics, which a timing program may ask for, exist only with torch's own allocator
    os.environ.setdefault("GENESIS_B200_POOL", "0")
    import genesis_b200 as genesis
    cache = genesis.nn.PagedKVCache(d["k"].shape[0], case["Hkv"], case["D"], page_size=case["page"],
                                    dtype="float8_e4m3fn" if case["cache"] == "e4m3" else d["k"].dtype, device=DEV)[0]
    for n in ("k", "v", "k_scale", "v_scale"):
        if n in d:
            pool = getattr(cache, n)
            pool.copy_(s.pop(n).view(pool.dtype))
    s["layer"] = cache
    for n in ("table", "lengths", "counts", "y", "cos", "sin", "new_k", "new_v", "q"):
        if n in d:
            s[n] = genesis.Tensor(d[n])
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _put(s, n, x):
    """Rows x [new tokens, KV heads, D] in 32 bits into the pool `n`."""
    pages, places = s["slot"]
    heads = torch.arange(x.shape[1], device=DEV)
    if n + "_scale" in s:
        x, e = _quantised(x)
        s[n + "_scale"][pages[:, None], heads, places[:, None]] = e
    s[n][pages[:, None], heads, places[:, None]] = x.to(s[n].dtype)


def _dense(s, n):
    """The pool `n` as [B, KV heads, longest, D] in 32 bits, zeros behind each sequence."""
    case, pages = s["case"], s["table"].clamp(min=0).long()
    x = s[n][pages]
    if n + "_scale" in s:
        x = x.view(torch.float8_e4m3fn).float() * _power(s[n + "_scale"][pages].int() - 127).unsqueeze(-1)
    x = x.float().transpose(1, 2).reshape(case["B"], case["Hkv"], -1, case["D"])[:, :, :s["longest"]]
    there = torch.arange(s["longest"], device=DEV) < s["lengths"][:, None]
    return torch.where(there[:, None, :, None], x, torch.zeros_like(x))


def _read(s):
    return [_dense(s, n).transpose(1, 2).to(TYPES[s["case"]["dtype"]]).contiguous() for n in "kv"]


def _held(s):
    """What the pools hold after a write: themselves, or the values that 8 bits stand for."""
    return _read(s) if "k_scale" in s else [s["k"], s["v"]]


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    B, S, Hq, Hkv, D = (case[n] for n in ("B", "S", "Hq", "Hkv", "D"))
    if case["kind"] == "read":
        return _read(s)
    if case["kind"] == "write":
        _put(s, "k", s["new_k"].view(B * S, Hkv, D)[s["rows"]].float())
        _put(s, "v", s["new_v"].view(B * S, Hkv, D)[s["rows"]].float())
        return _held(s)
    if case["kind"] == "rope":
        x = s["y"].view(B * S, Hq + 2 * Hkv, D)[s["rows"]].float()
        cos, sin = s["cos"][s["at"]].unsqueeze(1), s["sin"][s["at"]].unsqueeze(1)
        half = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
        r = x * cos + half * sin
        q = torch.zeros(B * S, Hq, D, dtype=s["y"].dtype, device=DEV)
        q[s["rows"]] = r[:, :Hq].to(q.dtype)
        _put(s, "k", r[:, Hq:Hq + Hkv])
        _put(s, "v", x[:, Hq + Hkv:])
        return [q.view(B, S, Hq, D)] + _held(s)
    k, v = _dense(s, "k"), _dense(s, "v")
    q = s["q"].float().view(B, S, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    z = (q @ k.transpose(-1, -2)).view(B, Hkv, S, Hq // Hkv, -1) / math.sqrt(D)
    end = s["lengths"][:, None] - S + 1 + torch.arange(S, device=DEV)
    seen = torch.arange(s["longest"], device=DEV) < end[..., None]
    z = torch.where(seen[:, None, :, None], z, torch.full_like(z, -math.inf))
    e = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-3e38))
    o = (e.view(B, Hkv, -1, z.shape[-1]) @ v).view(B, Hkv, S, -1, D) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return [o.permute(0, 2, 1, 3, 4).reshape(B, S, Hq, D).to(s["q"].dtype)]


def _run_own(s, case):
    import genesis_b200 as genesis
    import genesis_b200.nn.functional as F
    layer, table, lengths, counts = s["layer"], s["table"], s["lengths"], s.get("counts")
    with genesis.no_grad():
        if case["kind"] == "attend":
            return [F.paged_attention(s["q"], layer, table, lengths, counts)._t]
        if case["kind"] == "write":
            F.paged_kv_write(s["new_k"], s["new_v"], layer, table, lengths, counts)
            outs = []
        elif case["kind"] == "rope":
            outs = [F.paged_qkv_rope(s["y"], s["cos"], s["sin"], layer, table, lengths, case["Hq"], counts)._t]
        if case["kind"] == "read" or case["cache"] == "e4m3":
            k, v = F.paged_kv_read(layer, table, lengths, s["longest"], dtype=TYPES[case["dtype"]])
            return [k._t, v._t] if case["kind"] == "read" else outs + [k._t, v._t]
        return outs + [layer.k, layer.v]


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    lengths, counts = _lengths(case)
    B, S, Hq, Hkv, D = (case[n] for n in ("B", "S", "Hq", "Hkv", "D"))
    e, c = SIZE[case["dtype"]], SIZE[case["cache"]]
    row = Hkv * (D * c + (1 if case["cache"] == "e4m3" else 0))       # keys or values of one token, as held
    new, held = sum(counts), sum(lengths)
    dense = 2 * B * max(lengths) * Hkv * D * e
    if case["kind"] == "read":
        return dict(bytes=2 * held * row + dense, flops=0)
    if case["kind"] == "attend":
        return dict(bytes=2 * held * row + 2 * B * S * Hq * D * e, flops=4 * S * Hq * D * held)
    back = 2 * held * row + dense if case["cache"] == "e4m3" else 0
    if case["kind"] == "write":
        return dict(bytes=new * 2 * Hkv * D * e + 2 * new * row + back, flops=0)
    tables = 2 * 4 * D // 2 * len({n - c + i for n, c in zip(lengths, counts) for i in range(c)})
    return dict(bytes=new * (2 * Hq + 2 * Hkv) * D * e + 2 * new * row + tables + back, flops=3 * new * (Hq + Hkv) * D)


# ------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def _two_to(e):
    """2^e of whole numbers, as floats of 64 bits with no error (a power function has one here and there)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """x [..., D] in 64 bits -> the values that e4m3 numbers with a power of two for each row stand for."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -126) / 448)).clamp(min=-126)
    for _ in range(2):
        e = torch.where(top > 448 * _two_to(e), e + 1, e)
    y = x / _two_to(e)
    fine = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4
    return torch.round(y / _two_to(fine)) * _two_to(fine) * _two_to(e)


def exact(case, seed):
    d = _inputs(case, seed)
    lengths, counts = _lengths(case)
    B, S, Hq, Hkv, D, page = (case[n] for n in ("B", "S", "Hq", "Hkv", "D", "page"))
    T = max(lengths)
    eight = case["cache"] == "e4m3"

    def sequence(n, b):
        """[tokens, KV heads, D] of sequence b as the pool holds them before the call."""
        at = torch.arange(lengths[b], device=DEV)
        p = d["table"][b].long()[torch.div(at, page, rounding_mode="floor")]
        x = d[n][p, :, at % page]
        if not eight:
            return x.double()
        return x.view(torch.float8_e4m3fn).double() * _two_to(d[n + "_scale"][p, :, at % page].long() - 127)[..., None]

    if case["kind"] == "attend":
        out = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=DEV)
        for b in range(B):
            k, v = sequence("k", b), sequence("v", b)
            for i in range(S):
                n = lengths[b] - S + 1 + i
                q = d["q"][b, i].double().view(Hkv, Hq // Hkv, D)
                p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k[:n]) * D ** -0.5, -1)
                out[b, i] = torch.einsum("hgn,nhd->hgd", p, v[:n]).reshape(Hq, D)
        return [out]
    outs = []
    fresh = {}
    if case["kind"] == "write":
        fresh = {"k": d["new_k"].double(), "v": d["new_v"].double()}
    elif case["kind"] == "rope":
        heads = d["y"].double().view(B, S, Hq + 2 * Hkv, D)
        q = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=DEV)
        k = torch.zeros(B, S, Hkv, D, dtype=torch.float64, device=DEV)
        for b in range(B):
            a = lengths[b] - counts[b]
            c, s = (d[n][a:lengths[b], None, :D // 2].double() for n in ("cos", "sin"))
            z = torch.complex(heads[b, :counts[b], :Hq + Hkv, :D // 2], heads[b, :counts[b], :Hq + Hkv, D // 2:]) * torch.complex(c, s)
            z = torch.cat([z.real, z.imag], -1)
            q[b, :counts[b]], k[b, :counts[b]] = z[:, :Hq], z[:, Hq:]
        outs.append(q)
        fresh = {"k": k, "v": heads[:, :, Hq + Hkv:]}
    for n in "kv":
        if case["kind"] != "read" and not eight:
            pool = d[n].double()
            for b in range(B):
                at = torch.arange(lengths[b] - counts[b], lengths[b], device=DEV)
                pool[d["table"][b].long()[torch.div(at, page, rounding_mode="floor")], :, at % page] = fresh[n][b, :counts[b]]
            outs.append(pool)
            continue
        dense = torch.zeros(B, T, Hkv, D, dtype=torch.float64, device=DEV)
        for b in range(B):
            dense[b, :lengths[b]] = sequence(n, b)
            if n in fresh:
                dense[b, lengths[b] - counts[b]:lengths[b]] = _e4m3(fresh[n][b, :counts[b]])
        outs.append(dense)
    return outs
