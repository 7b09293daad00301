"""Calls on a paged cache at the edges of what their documentation allows, on the GPU."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.models.transformers import MoEConfig, MoEForCausalLM, QwenForCausalLM, TransformerConfig
from genesis_b200.nn import PagedKVCache
from genesis_b200.ops import native as N

import _paged_ref as R

pytestmark = pytest.mark.gpu


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


# ---- models --------------------------------------------------------------------------------------
def _model(kind, positions=256, head_dim=64):
    genesis.manual_seed(11)
    base = dict(vocab_size=512, hidden_size=4 * head_dim, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=positions, rope_theta=1e4)
    if kind == "dense":
        return QwenForCausalLM(TransformerConfig(**base)).eval().cuda()
    return MoEForCausalLM(MoEConfig(**base, num_experts_per_tok=2, num_local_experts=4, moe_intermediate_size=256)).eval().cuda()


def _ints(*xs):
    return genesis.Tensor(torch.tensor(xs, dtype=torch.int32, device="cuda"))


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
