"""Paged key / value caches on the CPU: values, refusals, bookkeeping of pages."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.nn.paged import PagedKVCache
from genesis_b200.ops.paged import quantise

import _paged_ref as R


def _i(*xs):
    return genesis.Tensor(torch.tensor(xs, dtype=torch.int32))


# ---- pages ---------------------------------------------------------------------------------------
def test_pages_are_handed_out_and_come_back():
    c = PagedKVCache(6, 2, 8, page_size=16, num_layers=3, dtype="float16")
    assert len(c) == 3 and c.free_pages == 6 and c[2].k.shape == (6, 2, 16, 8) and c[0].k_scale is None
    pages = c.allocate([1, 0, 33])
    assert [len(p) for p in pages] == [1, 0, 3] and c.free_pages == 2 and len({i for p in pages for i in p}) == 4
    c.extend(pages, [16, 17, 10])                       # enough, two more, and more than enough
    assert [len(p) for p in pages] == [1, 2, 3] and c.free_pages == 0
    with pytest.raises(RuntimeError, match="1 pages asked for, 0 of 6 free"):
        c.extend(pages, [17, 17, 33])
    assert [len(p) for p in pages] == [1, 2, 3]
    table = c.page_table(pages)
    assert table._t.dtype == torch.int32 and table.shape == (3, 3) and table._t[1].tolist() == pages[1] + [-1]
    assert c.page_table(pages, width=5).shape == (3, 5) and c.page_table([]).shape == (0, 0)
    with pytest.raises(ValueError, match="more than 2"):
        c.page_table(pages, width=2)
    gone = [list(pages[0])]
    c.release(pages[:1])
    assert c.free_pages == 1 and pages[0] == []
    for wrong in (gone, [pages[1], list(pages[1])], [[99]]):
        with pytest.raises(ValueError, match="released"):
            c.release(wrong)
    c.release(pages)
    assert sorted(c._free) == list(range(6))


def test_caches_that_are_refused():
    for kw in (dict(page_size=24), dict(page_size=0), dict(dtype="int8"), dict(dtype=torch.float64), dict(num_layers=0),
               dict(head_dim=True), dict(num_pages=2 ** 31), dict(num_kv_heads=1.0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(num_pages=2, num_kv_heads=1, head_dim=8), **kw})
    k = torch.zeros(2, 1, 16, 8)
    e = torch.zeros(2, 1, 16, 8, dtype=torch.uint8).view(torch.float8_e4m3fn)
    u = torch.zeros(2, 1, 16, dtype=torch.uint8)
    genesis.nn.PagedKVLayer(k, k), genesis.nn.PagedKVLayer(e, e, u, u)
    for wrong in ((k, k[:1]), (k, k.half()), (k.double(), k.double()), (k[:, :, :15], k[:, :, :15]), (k[0], k[0]), (k[:0], k[:0]),
                  (torch.zeros(2, 1, 8, 16).transpose(2, 3), k), (e, e), (k, k, u, u), (e, e, u, None), (e, e, u[:1], u), (e, e, u.int(), u),
                  (torch.zeros(257)[1:].view(2, 1, 16, 8), k)):
        with pytest.raises(ValueError, match="PagedKVLayer"):
            genesis.nn.PagedKVLayer(*wrong)
    assert PagedKVCache(1, 1, 8, dtype=genesis.bfloat16)[0].k.dtype == torch.bfloat16
    assert PagedKVCache(1, 1, 8, dtype=torch.float8_e4m3fn)[0].k_scale.dtype == torch.uint8


def test_copies_have_pools_of_their_own():
    import copy
    import pickle
    c = PagedKVCache(2, 1, 8, page_size=16, dtype="float8_e4m3fn")
    pages = c.allocate([20])
    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert d[0].k.data_ptr() != c[0].k.data_ptr() and d.free_pages == 0 and d.dtype == c.dtype
        F.paged_kv_write(*(genesis.Tensor(torch.ones(1, 20, 1, 8)) for _ in range(2)), d[0], d.page_table(pages), _i(20))
        assert torch.all(c[0].k.view(torch.uint8) == 0) and int((d[0].k.view(torch.uint8) != 0).sum()) == 160
    with pytest.raises(AttributeError):
        c[0].k = torch.zeros(1)


# ---- 8 bits --------------------------------------------------------------------------------------
def test_rows_of_8_bits_are_rounded_once():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(500, 12, generator=g) * torch.exp2(torch.randint(-40, 40, (500, 1), generator=g).float())
    x[0], x[1, 0], x[2, 0], x[3] = 0.0, math.nan, -math.inf, 1e-42
    x[4, :4], x[5, :2] = torch.tensor([448.0, 16.0, 17.0, 18.0]), torch.tensor([math.nextafter(448.0, 1e3) + 1e-4, 1.0])
    x[4, 4:], x[5, 2:], x[6] = 0.1, 0.1, 3.4e38
    y, e = quantise(x)
    v = torch.ldexp(y.double(), (e.int() - 127).unsqueeze(-1).double())
    w = R.e4m3_values(x.double())
    assert torch.equal(torch.isnan(v), torch.isnan(w)) and torch.equal(v.nan_to_num(), w.nan_to_num())
    assert int(e[4]) == 127 and int(e[5]) == 128 and int(e[0]) == 1
    assert y[4].double()[:4].tolist() == [448.0, 16.0, 16.0, 18.0]           # 17 stands halfway: to the even one


# ---- values --------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["fp32", "fp16", "bf16", "e4m3"])
@pytest.mark.parametrize("counts", [None, [3, 0, 1, 9, -2]])
def test_write_puts_rows_where_they_belong(cache, counts):
    B, S, H, D, page = 5, 3, 2, 6, 16
    lengths = [3, 17, 16, 40, 0] if counts is None else [20, 17, 16, 40, 0]
    t = R.Setup(lengths, H, D, cache, page)
    k, v = t.normal(B, S, H, D, dtype="fp32"), t.normal(B, S, H, D, dtype="fp32")
    before = [R.values(p, s) for p, s in ((t.layer.k, t.layer.k_scale), (t.layer.v, t.layer.v_scale))]
    F.paged_kv_write(t.tensor(k), t.tensor(v), t.layer, t.table, t.lens, None if counts is None else t.ints(counts))
    for pool, scale, x, old in ((t.layer.k, t.layer.k_scale, k, before[0]), (t.layer.v, t.layer.v_scale, v, before[1])):
        for b in range(B):
            n = min(max(S if counts is None else counts[b], 0), S)
            for s in range(n):
                pos = lengths[b] - n + s
                if pos >= 0:
                    old[t.pages[b][pos // page], :, pos % page] = R.held(x[b, s].double(), R.TYPES[cache])
        new = R.values(pool, scale)
        assert torch.equal(new.nan_to_num(7e9), old.nan_to_num(7e9))          # every other place as it was


@pytest.mark.parametrize("cache,dtype", [("fp32", "fp32"), ("e4m3", "fp16"), ("bf16", "bf16")])
def test_rope_write_and_read(cache, dtype):
    B, S, Hq, H, D, page = 3, 4, 4, 2, 8, 16
    lengths, counts = [4, 21, 2], [4, 2, 4]
    t = R.Setup(lengths, H, D, cache, page)
    y = t.normal(B, S, (Hq + 2 * H) * D, dtype=dtype)
    rot = genesis.models.transformers.components.RotaryEmbedding(D, 32, 1e4)
    q = F.paged_qkv_rope(t.tensor(y), rot.cos_cached, rot.sin_cached, t.layer, t.table, t.lens, Hq, t.ints(counts))
    assert q.shape == (B, S, Hq, D)
    k, v = F.paged_kv_read(t.layer, t.table, t.lens, 25, dtype="float32")
    assert k.shape == (B, 25, H, D) and torch.all(k._t[2, 2:] == 0)
    x = y.double().view(B, S, Hq + 2 * H, D)
    half = R.HALF[R.TYPES[dtype]]
    for b in range(B):
        for s in range(S):
            pos = lengths[b] - counts[b] + s
            if s >= counts[b] or pos < 0:
                assert torch.all(q._t[b, s] == 0)
                continue
            c, sn = rot.cos_cached._t[pos].double(), rot.sin_cached._t[pos].double()
            turned = x[b, s] * c + torch.cat((-x[b, s, :, D // 2:], x[b, s, :, :D // 2]), -1) * sn
            # two products and a sum in 32 bits, then one rounding to the output's type
            slack = 3 * 2.0 ** -24 * (x[b, s].abs().max() * 2)
            assert torch.all((q._t[b, s].double() - turned[:Hq]).abs() <= half * turned[:Hq].abs() + slack)
            # (a 32-bit rounding may carry a key over a border of its 8 bits: then it is off by a step of 2^-3 at most)
            want, step = R.held(turned[Hq:Hq + H], R.TYPES[cache]), {"fp32": 0.0, "bf16": 2.0 ** -7, "e4m3": 2.0 ** -3}[cache]
            assert torch.all((k._t[b, pos].double() - want).abs() <= step * want.abs() + slack)
            assert torch.equal(v._t[b, pos].double(), R.held(x[b, s, Hq + H:], R.TYPES[cache]))
    half_read = F.paged_kv_read(t.layer, t.table, t.lens, 3)[0]
    assert half_read.shape == (B, 3, H, D) and half_read._t.dtype == (torch.bfloat16 if cache == "e4m3" else R.TYPES[cache])


@pytest.mark.parametrize("cache,dtype", [("fp32", "fp32"), ("bf16", "bf16"), ("e4m3", "bf16"), ("e4m3", "fp16")])
def test_attention(cache, dtype):
    lengths, counts, S = [1, 16, 50, 0, 3, 5], [1, 3, 2, 3, 3, 9], 3
    t = R.Setup(lengths, 2, 8, cache)
    q = t.normal(6, S, 6, 8, dtype=dtype)
    o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens, t.ints(counts))
    n = [min(c, S) for c in counts]
    want, size, reach = R.attention(q, t.kv, [a - b for a, b in zip(lengths, n)], n, 8 ** -0.5)
    assert o._t.dtype == q.dtype
    assert torch.all((o._t.double() - want).abs() <= R.tolerance(q, want, size, reach, 50, cache))
    assert torch.all(o._t[0, 1:] == 0) and torch.all(o._t[3] == 0)
    # a length of 2 with three new tokens: the first is none
    short = F.paged_attention(t.tensor(q), t.layer, t.table, t.ints([1, 2, 2, 0, 2, 2]))._t
    assert torch.all(short[:, 0] == 0) and torch.all(short[3] == 0) and not torch.any(torch.all(short[[1, 2], 1] == 0, -1))


def test_tokens_that_come_later_do_not_reach_back():
    t = R.Setup([20], 2, 8, "bf16")
    q = t.normal(1, 3, 4, 8)
    clean = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.clone()
    t.layer.k[t.pages[0][1], :, 3], t.layer.v[t.pages[0][1], :, 3] = math.nan, math.inf
    o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t
    assert torch.equal(o[:, :2], clean[:, :2]) and not torch.any(torch.isfinite(o[:, 2]))


def test_a_prompt_and_single_tokens_give_what_flash_attention_gives():
    B, T, Hq, H, D = 2, 37, 4, 2, 16
    genesis.manual_seed(1)
    y = torch.randn(B, T, (Hq + 2 * H) * D)
    rot = genesis.models.transformers.components.RotaryEmbedding(D, 64, 1e4)
    tables = rot.cos_cached, rot.sin_cached
    with genesis.no_grad():
        want = F.flash_attention(*F.qkv_rope(genesis.Tensor(y), *tables, None, Hq, H, D), causal=True)._t
    cache = PagedKVCache(8, H, D, page_size=16, dtype="float32")
    pages = cache.allocate([T, T])
    table, got = cache.page_table(pages), []
    for a, b in ((0, 30), (30, 31), (31, 32), (32, 37)):
        n = _i(b, b)
        q = F.paged_qkv_rope(genesis.Tensor(y[:, a:b]), *tables, cache[0], table, n, Hq)
        got.append(F.paged_attention(q, cache[0], table, n)._t)
    assert torch.allclose(torch.cat(got, 1), want, atol=2e-6)


# ---- refusals ------------------------------------------------------------------------------------
def _call(op, t, **kw):
    B, S, Hq, H, D = 2, 2, 4, 2, 8
    a = dict(cache=t.layer, page_table=t.table, lengths=t.lens, counts=None, k=t.tensor(torch.zeros(B, S, H, D)),
             v=t.tensor(torch.zeros(B, S, H, D)), q=t.tensor(torch.zeros(B, S, Hq, D)), y=t.tensor(torch.zeros(B, S, 8 * D)),
             cos=t.tensor(torch.zeros(64, D)), sin=t.tensor(torch.zeros(64, D)), num_heads=Hq, max_length=3, dtype=None, scale=None)
    a.update(kw)
    if op == "write":
        return F.paged_kv_write(a["k"], a["v"], a["cache"], a["page_table"], a["lengths"], a["counts"])
    if op == "rope":
        return F.paged_qkv_rope(a["y"], a["cos"], a["sin"], a["cache"], a["page_table"], a["lengths"], a["num_heads"], a["counts"])
    if op == "read":
        return F.paged_kv_read(a["cache"], a["page_table"], a["lengths"], a["max_length"], a["dtype"])
    return F.paged_attention(a["q"], a["cache"], a["page_table"], a["lengths"], a["counts"], a["scale"])


REFUSED = [
    ("write rope read attend", dict(cache=None), TypeError),
    ("write rope read attend", dict(page_table=torch.zeros(2, 2, dtype=torch.int32)), TypeError),
    ("write rope read attend", dict(page_table=genesis.Tensor(torch.zeros(2, 2, dtype=torch.int64))), TypeError),
    ("write rope attend", dict(page_table=genesis.Tensor(torch.zeros(3, 2, dtype=torch.int32))), ValueError),
    ("write rope read attend", dict(lengths=_i(1, 2, 3)), ValueError),
    ("write rope read attend", dict(lengths=genesis.Tensor(torch.zeros(2))), TypeError),
    ("write rope read attend", dict(lengths=None), TypeError),
    ("write rope attend", dict(counts=_i(1)), ValueError),
    ("write", dict(k=genesis.Tensor(torch.zeros(2, 2, 2, 4))), ValueError),
    ("write", dict(v=genesis.Tensor(torch.zeros(2, 1, 2, 8))), ValueError),
    ("write", dict(v=genesis.Tensor(torch.zeros(2, 2, 2, 8).half())), TypeError),
    ("write", dict(k=genesis.Tensor(torch.zeros(2, 2, 2, 8).double())), TypeError),
    ("write", dict(k=genesis.Tensor(torch.zeros(2, 2, 2, 8), requires_grad=True)), RuntimeError),
    ("rope", dict(y=genesis.Tensor(torch.zeros(2, 2, 64), requires_grad=True)), RuntimeError),
    ("rope", dict(y=genesis.Tensor(torch.zeros(2, 2, 56))), ValueError),
    ("rope", dict(num_heads=3), ValueError),
    ("rope", dict(num_heads=True), ValueError),
    ("rope", dict(cos=genesis.Tensor(torch.zeros(64, 8).double())), TypeError),
    ("rope", dict(cos=genesis.Tensor(torch.zeros(64, 4))), ValueError),
    ("rope", dict(sin=genesis.Tensor(torch.zeros(32, 8))), ValueError),
    ("read", dict(max_length=-1), ValueError),
    ("read", dict(max_length=2.0), ValueError),
    ("read", dict(dtype="int32"), TypeError),
    ("attend", dict(q=genesis.Tensor(torch.zeros(2, 2, 3, 8))), ValueError),
    ("attend", dict(q=genesis.Tensor(torch.zeros(2, 2, 4, 16))), ValueError),
    ("attend", dict(q=genesis.Tensor(torch.zeros(2, 4, 8))), ValueError),
    ("attend", dict(q=genesis.Tensor(torch.zeros(2, 2, 4, 8), requires_grad=True)), RuntimeError),
    ("attend", dict(scale=math.nan), ValueError),
    ("attend", dict(scale="1"), ValueError),
]


@pytest.mark.parametrize("ops,change,error", REFUSED)
def test_refused(ops, change, error):
    t = R.Setup([20, 3], 2, 8, "fp32")
    for op in ops.split():
        with pytest.raises(error):
            _call(op, t, **change)
        with genesis.no_grad():
            if error is not RuntimeError:
                with pytest.raises(error):
                    _call(op, t, **change)
            else:
                _call(op, t, **change)


def test_bad_pages_and_positions():
    t = R.Setup([20, 3], 2, 8, "fp32")
    for op in ("write", "rope", "read", "attend"):
        long = dict(max_length=40)
        with pytest.raises(IndexError, match="room for 32"):
            _call(op, t, lengths=t.ints([33, 3]), **long)
        bad = t.table._t.clone()
        bad[0, 1] = 99
        with pytest.raises(IndexError, match="page 99"):
            _call(op, t, page_table=genesis.Tensor(bad), **long)
        bad[0, 1] = -1
        with pytest.raises(IndexError, match="page -1"):
            _call(op, t, page_table=genesis.Tensor(bad), **long)
        # a page that the call has no token in may be anything
        _call(op, t, page_table=genesis.Tensor(bad), lengths=t.ints([16, 3]), **long)
    with pytest.raises(IndexError, match="rotation tables"):
        _call("rope", t, cos=t.tensor(torch.zeros(19, 8)), sin=t.tensor(torch.zeros(19, 8)))


def test_empty_calls():
    t = R.Setup([], 2, 8, "fp32")
    assert F.paged_attention(t.tensor(torch.zeros(0, 1, 4, 8)), t.layer, t.table, t.ints([])).shape == (0, 1, 4, 8)
    assert F.paged_kv_read(t.layer, t.table, t.ints([]), 5)[1].shape == (0, 5, 2, 8)
    t = R.Setup([0, 0], 2, 8, "e4m3")
    assert t.table.shape == (2, 0)
    assert torch.all(F.paged_attention(t.tensor(torch.ones(2, 3, 4, 8)), t.layer, t.table, t.lens)._t == 0)
    F.paged_kv_write(t.tensor(torch.ones(2, 3, 2, 8)), t.tensor(torch.ones(2, 3, 2, 8)), t.layer, t.table, t.lens)
    assert torch.all(t.layer.k.view(torch.uint8) == 0x7f)
    assert F.paged_kv_read(t.layer, t.table, t.lens, 0)[0].shape == (2, 0, 2, 8)
    F.paged_kv_write(t.tensor(torch.ones(2, 0, 2, 8)), t.tensor(torch.ones(2, 0, 2, 8)), t.layer, t.table, t.lens)
