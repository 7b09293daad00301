"""Kernels over paged key / value caches against a restatement in 64 bits."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.ops import dispatch as K
from genesis_b200.ops import native as N

import _paged_ref as R

pytestmark = pytest.mark.gpu


def _pools(t):
    return [R.values(p, s) for p, s in ((t.layer.k, t.layer.k_scale), (t.layer.v, t.layer.v_scale))]


def _expect(t, before, lengths, counts, S, rows):
    """The pools after a write of rows (k, v) [B, S, H, D] in 64 bits, as held."""
    for b, n in enumerate(counts):
        for s in range(min(max(n, 0), S)):
            pos = lengths[b] - min(max(n, 0), S) + s
            if pos >= 0:
                for pool, x in zip(before, rows):
                    pool[t.pages[b][pos // t.page], :, pos % t.page] = x[b, s]
    return before


def _same(a, b):
    return torch.equal(a.nan_to_num(7e9, 8e9, 9e9), b.nan_to_num(7e9, 8e9, 9e9))


# ---- writing -------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [128, 64, 80, 7, 256, 32, 16])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("fp16", "e4m3"), ("bf16", "e4m3"), ("fp32", "fp32"), ("fp32", "e4m3"),
                                         ("fp32", "bf16"), ("fp16", "fp16")])
def test_write(D, dtype, cache):
    lengths, counts, S, H = [3, 17, 16, 70, 0, 5, 33], [3, 0, 1, 9, 4, -2, 5], 5, 3
    t = R.Setup(lengths, H, D, cache, 16, "cuda")
    scales = torch.exp2(torch.randint(-20, 20, (7, S, H, 1), generator=t.g).float()) if dtype != "fp16" else 1.0
    k, v = ((t.normal(7, S, H, D, dtype="fp32") * scales).to(R.TYPES[dtype]) for _ in range(2))
    k[0, 0, 0, 0], k[1], v[2, 0, 1], v[3, 1, 0, :2] = math.nan, 0.0, 0.0, torch.tensor([math.inf, -math.inf])
    if cache == "bf16":
        k[3, 2, 0, 0] = -0.0
    want = _expect(t, _pools(t), lengths, counts, S, [R.held(x.double(), R.TYPES[cache]) for x in (k, v)])
    F.paged_kv_write(t.tensor(k), t.tensor(v), t.layer, t.table, t.lens, t.ints(counts))
    for got, w in zip(_pools(t), want):
        assert _same(got, w)


def test_write_takes_views():
    """Heads that are slices of a wider matrix, at odd offsets, transposed, and repeated through a stride of 0."""
    lengths, S, H, D = [9, 25], 4, 2, 64
    for cache in ("bf16", "e4m3"):
        for form in range(5):
            t = R.Setup(lengths, H, D, cache, 16, "cuda", seed=form)
            wide = t.normal(2, S, 6 * D + 8).cuda()
            if form == 0:
                k, v = (wide[..., a:a + H * D].unflatten(-1, (H, D)) for a in (D, 3 * D))
            elif form == 1:
                k, v = (wide[..., a:a + H * D].unflatten(-1, (H, D)) for a in (D + 1, 3 * D + 3))
            elif form == 2:
                k, v = (wide[..., a:a + H * D].reshape(2, S, D, H).transpose(2, 3) for a in (0, D))
            elif form == 3:
                k, v = wide[:, :1, None, :D].expand(2, S, H, D), wide[:1, :, None, D:2 * D].expand(2, S, H, D)
            else:
                k, v = (wide[..., a:a + H * D].reshape(2, H, S, D).transpose(1, 2) for a in (0, D))
            want = _expect(t, _pools(t), lengths, [S, S], S, [R.held(x.cpu().double(), R.TYPES[cache]) for x in (k, v)])
            F.paged_kv_write(genesis.Tensor(k), genesis.Tensor(v), t.layer, t.table, t.lens)
            for got, w in zip(_pools(t), want):
                assert _same(got, w)


@pytest.mark.parametrize("Hq,H,D", [(14, 2, 64), (4, 4, 128), (6, 2, 80), (2, 1, 6), (8, 1, 256)])
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("fp16", "e4m3"), ("bf16", "e4m3"), ("fp32", "fp32"), ("fp32", "e4m3")])
def test_rope_write(Hq, H, D, dtype, cache):
    lengths, counts, S, page = [4, 90, 2, 0, 33], [4, 2, 4, 3, 0], 4, 32
    t = R.Setup(lengths, H, D, cache, page, "cuda")
    y = t.normal(5, S, (Hq + 2 * H) * D, dtype=dtype)
    rot = genesis.models.transformers.components.RotaryEmbedding(D, 90, 1e4)
    cos, sin = rot.cos_cached._t, rot.sin_cached._t
    before = _pools(t)
    q = F.paged_qkv_rope(t.tensor(y), t.tensor(cos), t.tensor(sin), t.layer, t.table, t.lens, Hq, t.ints(counts))._t.cpu()
    x = y.double().view(5, S, Hq + 2 * H, D)
    turned = torch.zeros(5, S, Hq + H, D, dtype=torch.float64)
    live = torch.zeros(5, S, dtype=torch.bool)
    for b in range(5):
        for s in range(counts[b]):
            pos = lengths[b] - counts[b] + s
            if pos >= 0:
                z = x[b, s, :Hq + H]
                turned[b, s] = z * cos[pos].double() + torch.cat((-z[..., D // 2:], z[..., :D // 2]), -1) * sin[pos].double()
                live[b, s] = True
    assert q.dtype == y.dtype and torch.all(q[~live] == 0)
    # two products and a sum in 32 bits (of which one may be fused), then one rounding
    slack = 2.0 ** -23 * (x.abs().amax() * 2)
    assert torch.all((q.double() - turned[:, :, :Hq]).abs() <= R.HALF[y.dtype] * turned[:, :, :Hq].abs() + slack)
    keys, vals = _pools(t)
    want = _expect(t, before, lengths, counts, S, [R.held(turned[:, :, Hq:], R.TYPES[cache]), R.held(x[:, :, Hq + H:], R.TYPES[cache])])
    assert _same(vals, want[1])
    # the 32-bit error may carry a key over a border between two of the cache's numbers, hence a step of its type, and a row's
    # largest over a power of two, which doubles the step of its smallest: 2^-9 of 2^-8 of the largest
    step = {"fp32": 2.0 ** -23, "bf16": 2.0 ** -7, "e4m3": 2.0 ** -3}[cache]
    off = (keys - want[0]).nan_to_num(0).abs()
    assert torch.equal(torch.isnan(keys), torch.isnan(want[0]))
    assert torch.all(off <= step * want[0].nan_to_num(0).abs() + slack + (2.0 ** -16 * want[0].nan_to_num(0).abs().amax(-1, keepdim=True) if cache == "e4m3" else 0))
    assert float((off > slack).double().mean()) < 0.01


# ---- reading -------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [128, 64, 80, 7, 256])
@pytest.mark.parametrize("cache,dtype", [("bf16", "bf16"), ("e4m3", "bf16"), ("e4m3", "fp16"), ("fp32", "fp32"), ("e4m3", "fp32"),
                                         ("bf16", "fp32"), ("fp32", "fp16")])
def test_read(D, cache, dtype):
    lengths, H = [1, 0, 16, 17, 75, -3], 2
    t = R.Setup(lengths, H, D, cache, 16, "cuda", width=6)
    for L in (1, 33, 80):
        outs = F.paged_kv_read(t.layer, t.table, t.lens, L, dtype=str(R.TYPES[dtype]).replace("torch.", ""))
        for i, o in enumerate(outs):
            assert o.shape == (6, L, H, D)
            for b, n in enumerate(lengths):
                n = min(max(n, 0), L)
                assert torch.equal(o._t[b, :n].cpu(), t.kv[b][i][:n].to(R.TYPES[dtype])) and torch.all(o._t[b, n:] == 0)


# ---- attention -----------------------------------------------------------------------------------
def _attend(t, lengths, counts, S, Hq, D, dtype, cache, scale=None, strengths=1.0):
    H = t.layer.num_kv_heads
    B = len(lengths)
    q = (t.normal(B, S, Hq, D, dtype="fp32") * strengths).to(R.TYPES[dtype])
    c = None if counts is None else t.ints(counts)
    o = F.paged_attention(t.tensor(q), t.layer, t.table, t.ints(lengths), c, scale=scale)._t
    n = [S] * B if counts is None else [min(max(x, 0), S) for x in counts]
    want, size, reach = R.attention(q, t.kv, [max(a, 0) - b for a, b in zip(lengths, n)], n, D ** -0.5 if scale is None else scale)
    off = (o.cpu().double() - want).abs()
    bound = R.tolerance(q, want, size, reach, max(lengths, default=0), cache)
    assert o.dtype == q.dtype and torch.all(off <= bound), f"{float((off / bound.clamp(min=1e-300)).max())} of the bound"
    assert o.shape == (B, S, Hq, D) and H
    return q, o


TYPES = [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3"), ("fp32", "fp32")]


@pytest.mark.parametrize("Hq,H,D", [(14, 2, 64), (12, 2, 128), (32, 4, 128), (12, 12, 64), (6, 2, 80), (3, 1, 7), (16, 1, 64), (40, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_attention_of_single_tokens(Hq, H, D, dtype, cache):
    lengths = [1, 0, 2, 15, 16, 17, 31, 33, 100, 257, 600, -5]
    for width in (50, 10000):
        t = R.Setup(lengths, H, D, cache, 16, "cuda", width=width)
        _attend(t, lengths, None, 1, Hq, D, dtype, cache)


@pytest.mark.parametrize("Hq,H,D", [(14, 2, 64), (32, 4, 128), (12, 12, 64), (6, 2, 80), (8, 8, 128)])
@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("S", [2, 5, 19])
@pytest.mark.parametrize("width", [0, 4000])         # the rows of an item go by what the table has room for
def test_attention_of_several_tokens(Hq, H, D, dtype, cache, S, width):
    lengths, counts = [1, 0, 2, 16, 40, 100, 333, 70], [1, 3, 2, S, S, 1, S, 0]
    t = R.Setup(lengths, H, D, cache, 32, "cuda", width=width)
    _attend(t, lengths, counts, S, Hq, D, dtype, cache)
    _attend(t, lengths, None, S, Hq, D, dtype, cache)         # sequences shorter than the call: rows that see nothing


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,D", [(14, 2, 64), (32, 4, 128)])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_attention_over_long_sequences(dtype, cache, Hq, H, D, page):
    lengths = [9000, 4097, 63, 1]
    t = R.Setup(lengths, H, D, cache, page, "cuda")
    _attend(t, lengths, None, 1, Hq, D, dtype, cache)
    _attend(t, lengths, None, 1, Hq, D, dtype, cache, scale=0.31, strengths=3.0)
    t = R.Setup(lengths, H, D, cache, page, "cuda", width=60000 // page * 16)
    _attend(t, lengths, None, 3, Hq, D, dtype, cache)


@pytest.mark.parametrize("dtype,cache,Hq,H,D", [("fp32", "e4m3", 14, 2, 64), ("bf16", "fp32", 4, 4, 128), ("fp16", "bf16", 6, 2, 64),
                                               ("fp32", "bf16", 8, 1, 256), ("bf16", "bf16", 6, 3, 80), ("fp16", "e4m3", 2, 2, 96),
                                               ("bf16", "e4m3", 4, 1, 1), ("fp32", "fp32", 3, 3, 200)])
@pytest.mark.parametrize("S", [1, 3])
def test_attention_of_any_type_and_head(dtype, cache, Hq, H, D, S):
    lengths = [3000, 1, 0, 64, 65, 700]
    t = R.Setup(lengths, H, D, cache, 16, "cuda", width=200)
    _attend(t, lengths, None, S, Hq, D, dtype, cache)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_scales_of_either_sign_and_none(dtype, cache):
    t = R.Setup([300, 17], 2, 64, cache, 16, "cuda")
    for scale in (-0.2, 0.0, 1e-3):
        _attend(t, [300, 17], None, 1, 14, 64, dtype, cache, scale=scale)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_attention_of_many_sequences(dtype, cache):
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 200, (300,), generator=g).tolist()
    t = R.Setup(lengths, 2, 64, cache, 16, "cuda", width=40)
    _attend(t, lengths, None, 1, 14, 64, dtype, cache)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_scores_far_apart_and_one_sided(dtype, cache):
    """A key that outweighs all others, keys of one sign, and values of very different sizes."""
    lengths, Hq, H, D = [700, 50, 3], 4, 2, 64
    t = R.Setup(lengths, H, D, cache, 16, "cuda", value_scale=0.05)
    q = t.normal(3, 1, Hq, D, dtype=dtype)
    for b, n in enumerate(lengths):
        k, v = t.kv[b]
        k.add_(0.5)
        k[n // 2] = q[b, 0, :H].double() * 2
        v[n // 2] *= 2.0 ** -8
        v[n // 3] *= 2.0 ** 6
        k.copy_(R.held(k, R.TYPES[cache]))
        v.copy_(R.held(v, R.TYPES[cache]))
        at = torch.arange(n)
        for x, pool, sc in ((k, t.layer.k, t.layer.k_scale), (v, t.layer.v, t.layer.v_scale)):
            t._place(pool, sc, torch.tensor(t.pages[b])[at // 16], at % 16, x)
    o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens, scale=1.0)._t.cpu()
    want, size, reach = R.attention(q, t.kv, [n - 1 for n in lengths], [1] * 3, 1.0)
    assert torch.all((o.double() - want).abs() <= R.tolerance(q, want, size, reach, 700, cache))


def test_what_is_not_finite_stays_with_its_rows():
    for dtype, cache in TYPES:
        t = R.Setup([40, 40, 40], 2, 64, cache, 16, "cuda")
        q = t.normal(3, 1, 4, 64, dtype=dtype)
        clean = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.clone()
        bad = q.clone()
        bad[1, 0, 1, 5] = math.nan
        o = F.paged_attention(t.tensor(bad), t.layer, t.table, t.lens)._t
        assert torch.all(torch.isnan(o[1, 0, 1]))
        keep = torch.ones(3, 4, dtype=torch.bool)
        keep[1, 1] = False
        assert torch.equal(o[:, 0][keep], clean[:, 0][keep])
        # a NaN among the values of a key that is seen reaches that column of all rows of its head, and no other
        p, at = t.pages[2][1], 3
        if cache == "e4m3":
            t.layer.v.view(torch.uint8)[p, 1, at, 7] = 0x7f
        else:
            t.layer.v[p, 1, at, 7] = math.nan
        o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t
        assert torch.all(torch.isnan(o[2, 0, 2:, 7])) and int(torch.isnan(o).sum()) == 2
        # queries of +-inf scores: -inf throughout gives zeros
        if cache != "e4m3":
            t.layer.k[torch.tensor(t.pages[0], device="cuda")] = -math.inf
            o = F.paged_attention(t.tensor(q.abs() + 0.1), t.layer, t.table, t.lens)._t
            assert torch.all(o[0] == 0)


@pytest.mark.parametrize("S", [3, 9])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_tokens_that_come_later_do_not_reach_back(dtype, cache, S):
    """Infinities and NaN in the newest token's keys and values belong to the rows that see it."""
    for D, width in ((64, 0), (128, 0), (48, 0), (64, 20000), (128, 20000)):
        lengths = [33, 7, 200]
        t = R.Setup(lengths, 2, D, cache, 16, "cuda", width=width)
        q = t.normal(3, S, 8, D, dtype=dtype)
        clean = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.clone()
        for b, n in enumerate(lengths):
            if n < S:
                continue
            p, at = t.pages[b][(n - 1) // 16], (n - 1) % 16
            for pool in (t.layer.k, t.layer.v):
                if cache == "e4m3":
                    pool.view(torch.uint8)[p, 1, at, 3:9] = 0x7f
                else:
                    pool[p, 1, at, 3:6], pool[p, 1, at, 6:9] = math.nan, math.inf
        o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t
        assert torch.equal(o[:, :S - 1], clean[:, :S - 1]) and torch.equal(o[:, S - 1, :4], clean[:, S - 1, :4])
        hit = [n >= S for n in lengths]
        assert torch.all(torch.isnan(o[hit][:, S - 1, 4:, 3:6]))


def test_the_same_call_gives_the_same_bits():
    for dtype, cache in TYPES:
        t = R.Setup([5000, 1200, 3], 2, 64, cache, 16, "cuda")
        q = t.tensor(t.normal(3, 1, 14, 64, dtype=dtype))
        first = F.paged_attention(q, t.layer, t.table, t.lens)._t.clone()
        for _ in range(5):
            assert torch.equal(F.paged_attention(q, t.layer, t.table, t.lens)._t, first)


def test_queries_that_are_views():
    t = R.Setup([70, 20], 2, 64, "bf16", 16, "cuda")
    q = t.normal(2, 1, 4, 64).cuda()
    want = F.paged_attention(genesis.Tensor(q), t.layer, t.table, t.lens)._t
    wide = torch.zeros(2, 1, 4, 129, dtype=torch.bfloat16, device="cuda")
    wide[..., 1:65] = q
    flat = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = q.reshape(-1)
    for x in (wide[..., 1:65], q.transpose(1, 2).contiguous().transpose(1, 2), flat[1:].view(2, 1, 4, 64)):
        assert torch.equal(F.paged_attention(genesis.Tensor(x), t.layer, t.table, t.lens)._t, want)


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("bf16", "e4m3")])
def test_thousands_of_sequences(dtype, cache):
    """More sequences than a warp has lanes, a hundred times over; every seventh rests."""
    g = torch.Generator().manual_seed(8)
    lengths = torch.randint(1, 60, (3300,), generator=g)
    lengths[::7] = 0
    lengths[1234] = 5000
    t = R.Setup(lengths.tolist(), 1, 64, cache, 16, "cuda")
    _attend(t, lengths.tolist(), None, 1, 4, 64, dtype, cache)


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("fp16", "e4m3")])
def test_one_head_and_many_rows(dtype, cache):
    """64 query heads on one KV head, four tokens: sixteen tiles of rows that read the same keys."""
    for width in (0, 30000):
        t = R.Setup([130, 77], 1, 128, cache, 16, "cuda", width=width)
        _attend(t, [130, 77], None, 4, 64, 128, dtype, cache)


# ---- bad pages, far pages ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,cache,D", [("bf16", "bf16", 64), ("fp16", "e4m3", 128), ("fp32", "fp32", 16)])
def test_bad_pages_are_skipped_and_raised(dtype, cache, D):
    t = R.Setup([40, 20], 2, D, cache, 16, "cuda")
    q, kv = t.tensor(t.normal(2, 1, 4, D, dtype=dtype)), t.tensor(t.normal(2, 1, 2, D, dtype=dtype))
    y = t.tensor(t.normal(2, 1, 8 * D, dtype=dtype))
    tables = [t.tensor(torch.ones(48, D)) for _ in range(2)]
    for page in (-1, t.layer.num_pages, -2 ** 31, 2 ** 31 - 1):
        clean = F.paged_attention(q, t.layer, t.table, t.lens)._t.clone()       # (the writes below change the cache)
        dense = F.paged_kv_read(t.layer, t.table, t.lens, 40)[0]._t.clone()
        N.check_status()
        bad = t.table._t.clone()
        bad[0, 2] = page
        bad = genesis.Tensor(bad)
        calls = [lambda: F.paged_attention(q, t.layer, bad, t.lens), lambda: F.paged_kv_read(t.layer, bad, t.lens, 40)[0],
                 lambda: F.paged_kv_write(kv, kv, t.layer, bad, t.lens), lambda: F.paged_qkv_rope(y, *tables, t.layer, bad, t.lens, 4)]
        for i, call in enumerate(calls):
            before = _pools(t)
            o = call()
            with pytest.raises(IndexError, match="site=8"):
                N.check_status()
            if i == 0:
                assert torch.equal(o._t[1], clean[1]) and torch.all(torch.isfinite(o._t[0]))
            elif i == 1:
                assert torch.equal(o._t[1], dense[1]) and torch.equal(o._t[0, :32], dense[0, :32]) and torch.all(o._t[0, 32:] == 0)
            else:      # sequence 0's token went nowhere, sequence 1's to its place
                p = t.pages[1][1]
                for old, new in zip(before, _pools(t)):
                    old[p, :, 3] = new[p, :, 3]
                    assert _same(old, new)
    # longer than the table
    far = t.ints([49, 20])
    for call in (lambda: F.paged_attention(q, t.layer, t.table, far), lambda: F.paged_kv_read(t.layer, t.table, far, 60)[0],
                 lambda: F.paged_kv_write(kv, kv, t.layer, t.table, far), lambda: F.paged_qkv_rope(y, *tables, t.layer, t.table, far, 4)):
        call()
        with pytest.raises(IndexError, match="site=9"):
            N.check_status()
    short = [t.tensor(torch.ones(39, D)) for _ in range(2)]
    F.paged_qkv_rope(y, *short, t.layer, t.table, t.lens, 4)
    with pytest.raises(IndexError, match="site=9"):
        N.check_status()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_pages_beyond_31_bits(cache):
    """A pool of more than 2^31 numbers (2^32 bytes in 16 bits), with a sequence in its last pages."""
    H, D, page = 2, 128, 64
    P = 2 ** 31 // (H * D * page) + 40
    layer = genesis.nn.PagedKVCache(P, H, D, page_size=page, dtype="bfloat16" if cache == "bf16" else "float8_e4m3fn", device="cuda")[0]
    assert layer.k.numel() > 2 ** 31
    table = genesis.Tensor(torch.tensor([[P - 1, 0, P - 7], [P - 2, P - 3, 1]], dtype=torch.int32, device="cuda"))
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(2, 150, H, D, generator=g).bfloat16() for _ in range(2))
    n = genesis.Tensor(torch.tensor([150, 150], dtype=torch.int32, device="cuda"))
    F.paged_kv_write(genesis.Tensor(k.cuda()), genesis.Tensor(v.cuda()), layer, table, n)
    held = [R.held(x.double(), R.TYPES[cache]) for x in (k, v)]
    for o, w in zip(F.paged_kv_read(layer, table, n, 150), held):
        assert torch.equal(o._t.cpu().double(), w)
    q = torch.randn(2, 1, 8, D, generator=g).bfloat16()
    o = F.paged_attention(genesis.Tensor(q.cuda()), layer, table, n)._t.cpu()
    want, size, reach = R.attention(q, [(held[0][b], held[1][b]) for b in range(2)], [149] * 2, [1] * 2, D ** -0.5)
    assert torch.all((o.double() - want).abs() <= R.tolerance(q, want, size, reach, 150, cache))


# ---- streams and graphs --------------------------------------------------------------------------
def test_on_another_stream():
    t = R.Setup([3000, 100], 2, 64, "e4m3", 16, "cuda")
    q = t.tensor(t.normal(2, 1, 14, 64))
    want = F.paged_attention(q, t.layer, t.table, t.lens)._t
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(10):
        for s in side:
            with torch.cuda.stream(s):
                outs.append(F.paged_attention(q, t.layer, t.table, t.lens)._t)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_captured_steps_go_on(cache):
    """A step captured once (rotation, write, attention, length + 1) and replayed gives what eager steps give, for two caches
    whose graphs run side by side."""
    Hq, H, D, page, steps = 14, 2, 64, 16, 40
    rot = genesis.models.transformers.components.RotaryEmbedding(D, 128, 1e4)
    tables = [genesis.Tensor(x._t.cuda()) for x in (rot.cos_cached, rot.sin_cached)]
    g = torch.Generator().manual_seed(9)
    ys = torch.randn(steps, 2, 3, 1, (Hq + 2 * H) * D, generator=g).bfloat16().cuda()
    start = [7, 0, 30]

    def fresh(which):
        t = R.Setup(start, H, D, cache, page, "cuda", seed=which, width=5, spare=8)
        spare = [i for i in range(t.layer.num_pages) if i not in sum(t.pages, [])]
        table = t.table._t
        for b in range(3):
            for i in range(len(t.pages[b]), -(-(start[b] + steps) // page)):
                if spare:
                    table[b, i] = spare.pop()
        assert int((table[torch.arange(3), torch.tensor([2, 2, 4])] >= 0).sum()) == 3
        return t, genesis.Tensor(torch.empty_like(ys[0, 0]))

    def step(t, y):
        t.lens._t.add_(1)
        q = F.paged_qkv_rope(y, *tables, t.layer, t.table, t.lens, Hq)
        return F.paged_attention(q, t.layer, t.table, t.lens)

    want = []
    for which in range(2):
        t, y = fresh(which)
        outs = []
        for i in range(steps):
            y._t.copy_(ys[i, which])
            outs.append(step(t, y)._t.clone())
        want.append(outs)
    graphs = []
    for which in range(2):
        t, y = fresh(which)
        kept = t.lens._t.clone()
        y._t.copy_(ys[0, which])
        step(t, y)                                  # warm up on a copy of the lengths' state
        t.lens._t.copy_(kept)
        torch.cuda.synchronize()
        graph = genesis.cuda.CUDAGraph()
        with genesis.cuda.graph(graph):
            o = step(t, y)
        t.lens._t.copy_(kept)
        graphs.append((graph, t, y, o, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps):
        for which, (graph, t, y, o, stream) in enumerate(graphs):
            with torch.cuda.stream(stream):
                y._t.copy_(ys[i, which])
                graph.replay()
                got[which].append(o._t.clone())
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_no_library_call():
    t = R.Setup([300, 20], 2, 64, "e4m3", 16, "cuda")
    K.reset_fallbacks()
    with K.strict_native():
        y = t.tensor(t.normal(2, 1, 18 * 64))
        tables = [t.tensor(torch.ones(512, 64)) for _ in range(2)]
        q = F.paged_qkv_rope(y, *tables, t.layer, t.table, t.lens, 14)
        F.paged_attention(q, t.layer, t.table, t.lens)
        F.paged_kv_read(t.layer, t.table, t.lens, 300)
    assert K.fallback_counts() == {}
