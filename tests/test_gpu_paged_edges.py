"""Calls on a paged cache at the edges of what their documentation allows, on the GPU."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.models.transformers import MoEConfig, MoEForCausalLM, QwenForCausalLM, TransformerConfig
from genesis_b200.nn import PagedKVCache
from genesis_b200.ops import native as N

import _paged_ref as R

pytestmark = pytest.mark.gpu


def _ints(*xs):
    return genesis.Tensor(torch.tensor(xs, dtype=torch.int32, device="cuda"))


def _bits(t):
    return [x.clone().view(torch.uint8) for x in (t.layer.k, t.layer.v)]


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 6])           # a row a group of lanes, and a row a warp
def test_rotation_tables_without_a_position(D, cache):
    """Tables of no rows have no address; a call with them still rotates, finds no position, and writes nothing."""
    t = R.Setup([20, 0, 33], 2, D, cache, 16, "cuda")
    y, none = t.tensor(t.normal(3, 2, 8 * D)), t.tensor(torch.zeros(0, D))
    before = _bits(t)
    N.check_status()
    q = F.paged_qkv_rope(y, none, none, t.layer, t.table, t.lens, 4)
    with pytest.raises(IndexError, match="site=9"):
        N.check_status()
    assert torch.all(q._t == 0) and all(torch.equal(a, b) for a, b in zip(_bits(t), before))
    q = F.paged_qkv_rope(y, none, none, t.layer, t.table, t.ints([0, 0, 0]), 4)
    N.check_status()
    assert torch.all(q._t == 0) and all(torch.equal(a, b) for a, b in zip(_bits(t), before))


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 6])
def test_a_token_behind_the_rotation_tables_is_put_nowhere(D, cache):
    """Neither its key nor its value; the tokens before it are put as ever."""
    t = R.Setup([20, 4], 2, D, cache, 16, "cuda")
    y, table = t.tensor(t.normal(2, 3, 8 * D)), t.tensor(torch.ones(18, D))
    before = _bits(t)
    F.paged_qkv_rope(y, table, table, t.layer, t.table, t.lens, 4)
    with pytest.raises(IndexError, match="site=9"):
        N.check_status()
    for old, new in zip(before, _bits(t)):
        same = (old == new).flatten(3).all(-1).all(1).cpu()             # [pages, places]
        want = torch.ones_like(same)
        want[t.pages[0][1], 1] = want[t.pages[1][0], 1] = want[t.pages[1][0], 2] = want[t.pages[1][0], 3] = False
        assert torch.equal(same, want)


def test_positions_next_to_31_bits():
    """One page of 2^20 tokens that a table names 2048 times.  Keys are counted in 31 bits, so the last 256 positions are behind
    the table; up to them, keys seen over and over weigh what they weigh once."""
    D, page = 64, 2 ** 20
    layer = genesis.nn.PagedKVCache(1, 1, D, page_size=page, dtype="float16", device="cuda")[0]
    g = torch.Generator("cuda").manual_seed(6)
    layer.k.copy_(torch.randn(1, 1, page, D, device="cuda", generator=g))
    layer.v.fill_(1)
    layer.v[:, :, ::3, 1::2] = 0
    table = genesis.Tensor(torch.zeros(1, 2048, dtype=torch.int32, device="cuda"))
    q = genesis.Tensor(torch.randn(1, 1, 1, D, device="cuda", generator=g).half())
    once = F.paged_attention(q, layer, genesis.Tensor(table._t[:, :1].contiguous()), _ints(page))._t.float()
    N.check_status()
    assert torch.all((once[..., ::2] - 1).abs() <= 2.0 ** -10) and torch.all((once[..., 1::2] - 2 / 3).abs() <= 0.05)
    for n in (2 ** 31 - 256, 2 ** 31 - 255, 2 ** 31 - 1):
        o = F.paged_attention(q, layer, table, _ints(n))._t.float()
        if n > 2 ** 31 - 256:
            with pytest.raises(IndexError, match="site=9"):
                N.check_status()
        N.check_status()
        # a warp adds up 2^26 / 2368 chunks, each addition off by 2^-24 of the sum at most, in the sums and in the normaliser: 2^-8.2;
        # two results are rounded to 11 bits
        assert torch.all((o - once).abs() <= 2.0 ** -8.2 + 2.0 ** -10)
    x = genesis.Tensor(torch.full((1, 1, 1, D), 3.0, device="cuda").half())
    before = layer.k.clone()
    F.paged_kv_write(x, x, layer, table, _ints(2 ** 31 - 1))
    with pytest.raises(IndexError, match="site=9"):
        N.check_status()
    assert torch.equal(layer.k, before)
    F.paged_kv_write(x, x, layer, table, _ints(2 ** 31 - 256))             # position 2^31 - 257 = 257 before the page's end
    N.check_status()
    assert torch.all(layer.k[0, 0, page - 257] == 3) and torch.equal(layer.k[0, 0, :page - 257], before[0, 0, :page - 257])


# ---- infinities and NaN --------------------------------------------------------------------------
FAST = [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32")]                 # (8 bits hold no infinities)
OTHER = [("bf16", "fp32"), ("fp32", "bf16"), ("fp16", "bf16")]                # number by number
KINDS = [(a, b, D, w) for a, b in FAST for D in (64, 128, 48) for w in (0, 20000)] + [(a, b, 64, 0) for a, b in OTHER]


def _put(t, pool, b, pos, head, columns, x):
    pool[t.pages[b][pos // t.page], head, pos % t.page, columns] = x


def _pair(lengths, D, cache, width, seed=0):
    return [R.Setup(lengths, 2, D, cache, 16, dev, seed=seed, width=width if dev == "cuda" else 0) for dev in ("cpu", "cuda")]


def _kinds(x):
    """What an element is: 0 finite, 1, -1 an infinity, 2 NaN."""
    x = x.cpu().double()
    return torch.where(torch.isnan(x), 2.0, torch.where(torch.isinf(x), x.sign(), torch.zeros_like(x)))


@pytest.mark.parametrize("dtype,cache,D,width", KINDS)
@pytest.mark.parametrize("S", [1, 3, 9])
def test_infinities_among_the_values(dtype, cache, D, width, S):
    """A column of a row that sees an infinity is that infinity, one that sees both signs or a NaN is NaN, and all others are
    what they were, bit by bit; on the CPU alike.  First, middle and last keys, and ones that only later tokens see."""
    lengths = [1, 40, 700, 17]
    pair = _pair(lengths, D, cache, width)
    q = pair[0].normal(4, S, 8, D, dtype=dtype)
    clean = F.paged_attention(pair[1].tensor(q), pair[1].layer, pair[1].table, pair[1].lens)._t.clone()
    for t in pair:
        for b, pos, head, column, x in ((0, 0, 0, 3, math.inf), (0, 0, 1, 4, -math.inf), (0, 0, 1, 5, math.nan),
                                        (1, 0, 0, 0, math.inf), (1, 39, 0, 1, -math.inf), (1, 0, 0, 2, math.inf), (1, 39, 0, 2, -math.inf),
                                        (1, 20, 1, 7, math.inf), (1, 38, 1, 8, math.nan), (1, 5, 1, D - 1, -math.inf),
                                        (2, 0, 0, 6, -math.inf), (2, 699, 0, 9, math.inf), (2, 350, 0, 11, math.inf), (2, 351, 0, 11, math.inf),
                                        (2, 352, 0, 12, math.inf), (2, 698, 0, 12, -math.inf), (2, 3, 1, 13, math.nan), (2, 4, 1, 13, math.inf)):
            _put(t, t.layer.v, b, pos, head, column, x)
    cpu, gpu = (F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.cpu() for t in pair)
    assert torch.equal(_kinds(gpu), _kinds(cpu)) and int((_kinds(cpu) == 1).sum()) >= 8 and int((_kinds(cpu) == -1).sum()) >= 8
    fine = _kinds(cpu) == 0
    assert torch.equal(gpu[fine], clean.cpu()[fine])


@pytest.mark.parametrize("dtype,cache,D,width", KINDS)
@pytest.mark.parametrize("S", [1, 4])
def test_infinities_among_the_keys(dtype, cache, D, width, S):
    """Scores of -inf weigh nothing: the rows are those without the key.  Queries of 11 bits and less, and of more."""
    lengths, drop = [40, 700, 33], [7, 350, 0]
    pair = _pair(lengths, D, cache, width, seed=2)
    q = pair[0].normal(3, S, 8, D, dtype=dtype)
    q[..., 0] = torch.tensor([1.0, 0.5, 3.0, 1 / 3, 2.0 ** -10, 1.0, 1.5, 0.1]).to(q.dtype)
    for t in pair:
        for b, pos in enumerate(drop):
            for head in range(2):
                _put(t, t.layer.k, b, pos, head, 0, -math.inf)
    kv = [[torch.cat((x[:pos], x[pos + 1:])) for x in pair[0].kv[b]] for b, pos in enumerate(drop)]
    want, size, reach = R.attention(q, kv, [n - 1 - S for n in lengths], [S] * 3, D ** -0.5)
    bound = R.tolerance(q, want, size, reach, 700, cache)
    for t in pair:
        o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.cpu()
        assert torch.all((o.double() - want).abs() <= bound)
    # with an infinity among its values too, such a key gives NaN there: 0 times an infinity
    for t in pair:
        for b, pos in enumerate(drop):
            _put(t, t.layer.v, b, pos, 1, 2, math.inf)
    cpu, gpu = (F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.cpu() for t in pair)
    assert torch.all(torch.isnan(cpu[:, :, 4:, 2])) and torch.equal(_kinds(gpu), _kinds(cpu))


@pytest.mark.parametrize("dtype,cache,D,width", KINDS)
@pytest.mark.parametrize("S", [1, 4])
def test_rows_whose_scores_are_minus_infinity_throughout(dtype, cache, D, width, S):
    """Zeros, whether keys or the query are infinite, and whatever the values hold."""
    lengths = [40, 700, 5]
    pair = _pair(lengths, D, cache, width, seed=3)
    q = pair[0].normal(3, S, 8, D, dtype=dtype)
    q[..., 0] = 1.0
    q[1, :, 0, 0] = -math.inf                # its keys are positive there
    for t in pair:
        for b, n in enumerate(lengths):
            for pos in range(n):
                if b != 1:
                    _put(t, t.layer.k, b, pos, 1, 0, -math.inf)
                else:
                    _put(t, t.layer.k, b, pos, 0, 0, 1.0 + pos % 3)
            _put(t, t.layer.v, b, n - 1, 1 if b != 1 else 0, 2, math.inf)
            _put(t, t.layer.v, b, 0, 1 if b != 1 else 0, 3, -math.inf)
    cpu, gpu = (F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.cpu() for t in pair)
    for o in (cpu, gpu):
        assert torch.all(o[[0, 2]][:, :, 4:] == 0) and torch.all(o[1, :, 0] == 0)
    assert torch.equal(_kinds(gpu), _kinds(cpu))


@pytest.mark.parametrize("dtype,cache", FAST)
def test_infinities_of_keys_with_little_weight(dtype, cache):
    """A weight that is no number of fp16 any more is still one; in another part of the sequence, too."""
    lengths = [600]
    pair = _pair(lengths, 64, cache, 0, seed=4)
    q = torch.zeros(1, 1, 2, 64).to(R.TYPES[dtype])
    q[..., 0] = 8.0
    for t in pair:
        for pos in range(600):
            _put(t, t.layer.k, 0, pos, slice(None), 0, 4.0 if pos == 300 else 0.0)      # weights of e^-32 next to one of 1
        for i, pos in enumerate((0, 299, 301, 599)):
            _put(t, t.layer.v, 0, pos, slice(None), i, math.inf)
    cpu, gpu = (F.paged_attention(t.tensor(q), t.layer, t.table, t.lens, scale=1.0)._t.cpu() for t in pair)
    assert torch.all(cpu[..., :4] == math.inf) and torch.equal(_kinds(gpu), _kinds(cpu))


# ---- digits of 32-bit attention over long sequences ----------------------------------------------
@pytest.mark.parametrize("Hq,H,D", [(14, 2, 64), (32, 4, 128), (12, 12, 64), (6, 2, 80)])
@pytest.mark.parametrize("S,width", [(1, 0), (3, 0), (3, 20000)])
def test_long_sequences_in_32_bits_keep_their_digits(Hq, H, D, S, width):
    """The error of a whole output, not of single numbers at their worst: weights that miss their low parts would show."""
    lengths = [9000, 4097, 700]
    t = R.Setup(lengths, H, D, "fp32", 16, "cuda", seed=9, width=width)
    q = t.normal(3, S, Hq, D, dtype="fp32") * 3
    o = F.paged_attention(t.tensor(q), t.layer, t.table, t.lens)._t.cpu().double()
    want, size, _ = R.attention(q, t.kv, [n - S for n in lengths], [S] * 3, D ** -0.5)

    def rms(x):
        return float(x.square().mean().sqrt())

    # A score is the sum of D products of 22 bits each, 3 D^-1/2 in size on average: 2^-22 of 3 together, and as much again from sums
    # that are cut off at 2^-24 in each of D / 8 steps; the exponent's own rounding is 2^-24 of scores of up to 16, 2^-20.  Products
    # of weights and values and their sums add 2^-22 each.  In all below 2^-19 of the magnitudes that are added up.
    bound = 2.0 ** -19 * rms(size)
    assert rms(o - want) <= bound
    # what the bound is for: the same with weights of 11 bits
    cut = torch.zeros_like(want)
    for b, n in enumerate(lengths):
        for s in range(S):
            k, v = (x[:n - S + s + 1].repeat_interleave(Hq // H, 1) for x in t.kv[b])
            z = torch.einsum("hd,nhd->hn", q[b, s].double(), k) * D ** -0.5
            p = torch.exp(z - z.amax(-1, keepdim=True))
            step = torch.ldexp(torch.ones_like(p), torch.frexp(p)[1] - 11)
            cut[b, s] = torch.einsum("hn,nhd->hd", torch.round(p / step) * step, v) / p.sum(-1)[:, None]
    assert rms(cut - want) > 2 * bound


# ---- 8 bits --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,S", [("bf16", 1), ("bf16", 3), ("fp32", 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [-126, -121, -119, -110, 100])
def test_values_of_the_smallest_and_large_powers_of_two(dtype, S, D, power):
    """Rows whose power of two is next to the smallest, whose unit is no normal number of 32 bits any more."""
    t = R.Setup([40, 700], 2, D, "e4m3", 16, "cuda", seed=7)
    q = t.normal(2, S, 8, D, dtype=dtype)
    small = R.Setup([40, 700], 2, D, "e4m3", 16, "cuda", seed=7)
    for x in (t, small):
        x.layer.v_scale.fill_(127)
    small.layer.v_scale.fill_(127 + power)
    one, tiny = (F.paged_attention(x.tensor(q), x.layer, x.table, x.lens)._t.cpu().double() for x in (t, small))
    want = one * 2.0 ** power
    # the same numbers under another power of two: equal but for what falls below the smallest subnormal number of the output, or
    # of 32 bits before the last division (2^-149, once a warp and once a join: a handful), and a rounding that this tips over
    # (number by number, a weight is multiplied by the power first: 2^-150 off below 2^-126, times a value of up to 448, for each key)
    step = 2.0 ** -133 if dtype == "bf16" else 2.0 ** -149 + 700 * 448 * 2.0 ** -150
    assert torch.all((tiny - want).abs() <= step + 16 * 2.0 ** -149 + want.abs() * R.HALF[R.TYPES[dtype]] * 2) and torch.any(tiny != 0)


# ---- models --------------------------------------------------------------------------------------
def _model(kind, positions=256, head_dim=64):
    genesis.manual_seed(11)
    base = dict(vocab_size=512, hidden_size=4 * head_dim, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=positions, rope_theta=1e4)
    if kind == "dense":
        return QwenForCausalLM(TransformerConfig(**base)).eval().cuda()
    return MoEForCausalLM(MoEConfig(**base, num_experts_per_tok=2, num_local_experts=4, moe_intermediate_size=256)).eval().cuda()


def _tokens(*shape, seed=3):
    return torch.randint(0, 512, shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def _prompted(m, start, room, dtype="bfloat16", layers=2, head_dim=64):
    """A cache with prompts of the given lengths -> (cache, table, lengths)."""
    cache = PagedKVCache(sum(-(-(n + room) // 16) for n in start), 2, head_dim, page_size=16, num_layers=layers, dtype=dtype, device="cuda")
    table, lengths = cache.page_table(cache.allocate([n + room for n in start])), _ints(*start)
    m.forward_paged(genesis.Tensor(_tokens(len(start), max(start), seed=5)), cache, table, lengths, _ints(*start), prompt=True)
    return cache, table, lengths


def _captured(step, lengths, keep):
    """`step` warmed up and captured -> (graph, output); lengths as they were."""
    step()
    lengths._t.copy_(keep)
    torch.cuda.synchronize()
    graph = genesis.cuda.CUDAGraph()
    with genesis.cuda.graph(graph):
        out = step()
    lengths._t.copy_(keep)
    return graph, out


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_a_captured_step_after_a_plain_call_outgrows_the_tables(kind):
    m = _model(kind)
    start = (5, 40, 17)
    toks = _tokens(3, 1, seed=4)
    with genesis.no_grad(), genesis.amp.autocast(dtype=genesis.bfloat16):
        cache, table, lengths = _prompted(m, start, 20)
        keep = lengths._t.clone()

        def step():
            lengths._t += 1
            return m.forward_paged(genesis.Tensor(toks), cache, table, lengths)

        want = step()._t.clone()
        lengths._t.copy_(keep)
        graph, out = _captured(step, lengths, keep)
        graph.replay()
        assert torch.equal(out._t, want)
        m(genesis.Tensor(_tokens(1, 300)))                       # outgrows the tables
        assert m.model.layers[0].self_attn.rotary_emb.max_seq_len_cached >= 300
        rubbish = [torch.full((256, 64), 1e4, device="cuda") for _ in range(64)]      # over whatever has become free
        lengths._t.copy_(keep)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out._t, want) and rubbish


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("half,cache_dtype", [("bfloat16", "bfloat16"), ("half", "float16"), ("bfloat16", "float8_e4m3fn")])
def test_models_converted_to_16_bits(kind, half, cache_dtype):
    """Generation and a captured step of a model in 16 bits; its answers are those of the same model with tables in 32."""
    answers = []
    for rebuilt in (False, True):
        m = getattr(_model(kind), half)()
        if rebuilt:
            for layer in m.model.layers:
                layer.self_attn.rotary_emb._build(256)
        with genesis.no_grad():
            cache, table, lengths = _prompted(m, (5, 40), 20, cache_dtype)
            keep, toks = lengths._t.clone(), genesis.Tensor(_tokens(2, 1, seed=4))

            def step():
                lengths._t += 1
                return m.forward_paged(toks, cache, table, lengths)

            want = step()._t.clone()
            lengths._t.copy_(keep)
            graph, out = _captured(step, lengths, keep)
            graph.replay()
            assert torch.equal(out._t, want)
            answers.append(want)
        prompt = genesis.Tensor(_tokens(2, 9))
        assert m.generate(prompt, max_new_tokens=4, temperature=0.0, cache_dtype=cache_dtype).shape == (2, 13)
        del graph
    assert torch.equal(*answers)


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_prompts_padded_in_front_and_behind(kind):
    """The same bits, whichever side the padding is on."""
    m = _model(kind)
    toks, have, S = _tokens(3, 40), (40, 7, 23), 40
    rows = torch.zeros(2, 3, S, dtype=torch.int64, device="cuda")
    for b, n in enumerate(have):
        rows[0, b, :n] = rows[1, b, S - n:] = toks[b, :n]
    rows[1, 1, :S - 7] = 5
    for last in (True, False):
        outs = []
        for idx, counts in ((rows[0], _ints(*have)), (rows[1], None)):
            cache = PagedKVCache(12, 2, 64, page_size=16, num_layers=2, dtype="bfloat16", device="cuda")
            table = cache.page_table(cache.allocate([41, 41, 41]))
            with genesis.no_grad(), genesis.amp.autocast(dtype=genesis.bfloat16):
                out = m.forward_paged(genesis.Tensor(idx), cache, table, _ints(*have), counts, prompt=True, last=last)._t
                nxt = m.forward_paged(genesis.Tensor(toks[:, :1]), cache, table, _ints(*(n + 1 for n in have)))._t
            outs.append((out, nxt))
        (a, x), (b, y) = outs
        assert torch.equal(x, y)
        if last:
            assert torch.equal(a, b)
        else:
            assert all(torch.equal(a[i, :n], b[i, S - n:]) for i, n in enumerate(have))


def test_slots_that_rest_in_a_captured_step():
    """A slot out of use and one that comes to rest, through replays: no error is recorded, the lengths and pages of both stay, and
    the others go on as without them."""
    m = _model("dense")
    toks = _tokens(6, 3, 1, seed=8)
    with genesis.no_grad(), genesis.amp.autocast(dtype=genesis.bfloat16):
        cache = PagedKVCache(12, 2, 64, page_size=16, num_layers=2, dtype="bfloat16", device="cuda")
        table, lengths, active = cache.page_table(cache.allocate([60, 0, 60])), _ints(5, 0, 40), _ints(1, 0, 1)
        m.forward_paged(genesis.Tensor(_tokens(3, 40, seed=5)), cache, table, lengths, lengths, prompt=True)
        state = [x.clone() for layer in cache.layers for x in (layer.k, layer.v)]
        idx = genesis.Tensor(toks[0].clone())

        def step():
            lengths._t += active._t
            return m.forward_paged(idx, cache, table, lengths, active)

        graph, out = _captured(step, lengths, lengths._t.clone())
        N.check_status()
        for i in range(6):
            active._t[2] = int(i < 3)
            idx._t.copy_(toks[i])
            graph.replay()
            if i == 2:
                kept = [x.clone() for layer in cache.layers for x in (layer.k, layer.v)]
        N.check_status()
        assert lengths._t.tolist() == [11, 0, 43]
        mine = [p for p in range(12) if p in table._t[2].tolist()]
        assert all(torch.equal(a[mine], b[mine]) for a, b in zip(kept, [x for layer in cache.layers for x in (layer.k, layer.v)]))
        got = out._t[0].clone()
        # the first sequence alone
        for x, y in zip([x for layer in cache.layers for x in (layer.k, layer.v)], state):
            x.copy_(y)
        one, alone = _ints(5), None
        for i in range(6):
            one._t += 1
            alone = m.forward_paged(genesis.Tensor(toks[i, :1]), cache, genesis.Tensor(table._t[:1].contiguous()), one)._t
        q = genesis.Tensor(torch.randn(3, 1, 4, 64, device="cuda").bfloat16())
        assert torch.all(F.paged_attention(q, cache[0], table, lengths, active)._t[1:] == 0)
        # (products over other numbers of rows may be split otherwise: a dozen roundings to bf16 in each of two layers, 2^-9 on average)
        assert float((got.float() - alone[0].float()).norm() / alone[0].float().norm()) < 2 * 12 * 2.0 ** -9
    N.check_status()


def _sharp(kind, head_dim):
    """A model whose scores matter: queries and keys of several times the usual size."""
    m = _model(kind, head_dim=head_dim)
    for layer in m.model.layers:
        for w in (layer.self_attn.q_proj.weight, layer.self_attn.k_proj.weight):
            w._t.mul_(5.0)
    return m


def _decoded(m, tokens, head_dim, dtype, ahead=0):
    """Logits of the tokens 99 .. 111 of 120 over a paged cache: a prompt, single tokens, a piece.  `ahead`: what single tokens'
    lengths are off by."""
    cache = PagedKVCache(10, 2, head_dim, page_size=32, num_layers=2, dtype=dtype, device="cuda")
    table = cache.page_table(cache.allocate([130, 130]))
    got = [m.forward_paged(genesis.Tensor(tokens[:, :100]), cache, table, _ints(100, 100), prompt=True)._t]
    for n in range(101, 106):
        got.append(m.forward_paged(genesis.Tensor(tokens[:, n - 1:n]), cache, table, _ints(n + ahead, n + ahead))._t)
    got.append(m.forward_paged(genesis.Tensor(tokens[:, 105:112]), cache, table, _ints(112 + ahead, 112 + ahead), last=False)._t)
    return torch.cat(got, 1).float()


def _off(got, want):
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_decoding_against_encoding_everything_in_32_bits(kind, head_dim):
    """Both models, in 32 bits throughout, and what a position that is off by one would do."""
    m, tokens = _sharp(kind, head_dim), _tokens(2, 112)
    with genesis.no_grad():
        want = m(genesis.Tensor(tokens))._t[:, 99:112].float()
        # matrix products round their operands to 11 bits.  Operands that differ by 2^-20 round apart one time in 2^9, by 2^-11: 2^-15.5 of
        # each of 14 products' results in two layers and the head, on either side, were they all of one sign: below 2^-10
        assert _off(_decoded(m, tokens, head_dim, "float32"), want) < 2.0 ** -10
        assert _off(_decoded(m, tokens, head_dim, "float32", ahead=1), want) > 2.0 ** -8


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("cache_dtype,slack", [("bfloat16", 0.0), ("float16", 0.0), ("float8_e4m3fn", 2.0 ** -4)])
def test_decoding_in_mixed_types_over_caches_of_all_types(kind, head_dim, cache_dtype, slack):
    """Queries in 32 bits over 16- and 8-bit caches, which a model outside autocast asks for; against a cache in 32 bits."""
    m, tokens = _sharp(kind, head_dim), _tokens(2, 112)
    with genesis.no_grad():
        want = _decoded(m, tokens, head_dim, "float32")
        # keys and values lose 2^-9 (fp16: 2^-12; 8 bits: 2^-5 each on average, 2^-4 in all) in two layers; scores of up to 16 carry that on
        bound = 2 * 2.0 ** -9 * 4 + slack * 4
        assert _off(_decoded(m, tokens, head_dim, cache_dtype), want) < bound


@pytest.mark.parametrize("head_dim", [64, 128])
def test_decoding_in_bf16_against_encoding_everything(head_dim):
    """Under autocast; a position that is off by one is further off than the roundings allow."""
    m, tokens = _sharp("dense", head_dim), _tokens(2, 112)
    with genesis.no_grad(), genesis.amp.autocast(dtype=genesis.bfloat16):
        want = m(genesis.Tensor(tokens))._t[:, 99:112].float()
        # a dozen roundings to bf16 a layer, 2^-9 / 3^1/2 of a number each and independent of one another, on either side, carried on
        # by scores of several times the usual size
        bound = 4 * (2 * 2 * 12) ** 0.5 * 2.0 ** -9 / 3 ** 0.5
        assert _off(_decoded(m, tokens, head_dim, "bfloat16"), want) < bound
        assert _off(_decoded(m, tokens, head_dim, "bfloat16", ahead=1), want) > 2 * bound
