"""Decoders over a paged cache on the GPU."""
import pytest
import torch

import genesis_b200 as genesis
from genesis_b200.models.transformers import MoEConfig, MoEForCausalLM, QwenForCausalLM, TransformerConfig
from genesis_b200.nn import PagedKVCache
from genesis_b200.ops import dispatch as K

pytestmark = pytest.mark.gpu


def _model(kind, head_dim=64):
    genesis.manual_seed(11)
    base = dict(vocab_size=512, hidden_size=4 * head_dim, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=256, rope_theta=1e4)
    if kind == "dense":
        return QwenForCausalLM(TransformerConfig(**base)).eval().cuda()
    return MoEForCausalLM(MoEConfig(**base, num_experts_per_tok=2, num_local_experts=4, moe_intermediate_size=256)).eval().cuda()


def _ints(*xs):
    return genesis.Tensor(torch.tensor(xs, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("cache_dtype", ["bfloat16", "float8_e4m3fn"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_single_tokens_against_encoding_everything(head_dim, cache_dtype):
    m = _model("dense", head_dim)
    tokens = torch.randint(0, 512, (2, 120), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    with genesis.no_grad(), genesis.amp.autocast(dtype=genesis.bfloat16):
        full = m(genesis.Tensor(tokens))._t.float()
        cache = PagedKVCache(8, 2, head_dim, page_size=32, num_layers=2, dtype=cache_dtype, device="cuda")
        table = cache.page_table(cache.allocate([120, 120]))
        K.reset_fallbacks()
        got = [m.forward_paged(genesis.Tensor(tokens[:, :100]), cache, table, _ints(100, 100), prompt=True)._t[:, 0]]
        for n in range(101, 111):
            got.append(m.forward_paged(genesis.Tensor(tokens[:, n - 1:n]), cache, table, _ints(n, n))._t[:, 0])
        got.append(m.forward_paged(genesis.Tensor(tokens[:, 110:120]), cache, table, _ints(120, 120))._t[:, 0])
        assert K.fallback_counts() == {}
    want = full[:, list(range(99, 110)) + [119]]
    off = (torch.stack(got, 1).float() - want).norm() / want.norm()
    # a dozen roundings to bf16 a layer, each off by at most 2^-8 of what it rounds, on either side; keys and values in 8 bits add 2^-4
    # at most of the attention's part
    assert float(off) < 2 * 2 * 12 * 2.0 ** -8 + (0.125 if cache_dtype != "bfloat16" else 0.0)


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_generate_with_a_cache(kind):
    m = _model(kind)
    prompt = genesis.Tensor(torch.randint(0, 512, (3, 17), device="cuda"))
    with genesis.amp.autocast(dtype=genesis.bfloat16):
        for dt in ("bfloat16", "float16", "float8_e4m3fn"):
            out = m.generate(prompt, max_new_tokens=5, temperature=0.0, cache_dtype=dt)
            assert out.shape == (3, 22) and torch.equal(out._t[:, :17], prompt._t)
            assert torch.equal(out._t, m.generate(prompt, max_new_tokens=5, temperature=0.0, cache_dtype=dt)._t)
    out = m.generate(prompt, max_new_tokens=3, temperature=0.7, top_k=8, cache_dtype="float32")      # a model in 32 bits
    assert out.shape == (3, 20)


def test_a_captured_step_replays_as_the_sequences_grow():
    m = _model("dense")
    B, start, steps = 3, (5, 40, 17), 30
    toks = torch.randint(0, 512, (steps, B, 1), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    prompt = torch.randint(0, 512, (B, 40), device="cuda", generator=torch.Generator("cuda").manual_seed(5))

    def fresh():
        cache = PagedKVCache(16, 2, 64, page_size=16, num_layers=2, dtype="float8_e4m3fn", device="cuda")
        table, lengths = cache.page_table(cache.allocate([n + steps for n in start])), _ints(*start)
        m.forward_paged(genesis.Tensor(prompt), cache, table, lengths, _ints(*start), prompt=True)
        return cache, table, lengths

    with genesis.no_grad(), genesis.amp.autocast(dtype=genesis.bfloat16):
        cache, table, lengths = fresh()
        want = []
        for i in range(steps):
            lengths._t += 1
            want.append(m.forward_paged(genesis.Tensor(toks[i]), cache, table, lengths)._t.clone())
        cache, table, lengths = fresh()
        idx = genesis.Tensor(toks[0].clone())

        def step():
            lengths._t += 1
            return m.forward_paged(idx, cache, table, lengths)

        keep = lengths._t.clone()
        step()
        lengths._t.copy_(keep)
        torch.cuda.synchronize()
        graph = genesis.cuda.CUDAGraph()
        with genesis.cuda.graph(graph):
            out = step()
        lengths._t.copy_(keep)
        for i in range(steps):
            idx._t.copy_(toks[i])
            graph.replay()
            assert torch.equal(out._t, want[i])
