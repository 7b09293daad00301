"""Decoders over a paged cache on the CPU: what they answer is what encoding everything anew answers."""
import pytest
import torch

import genesis_b200 as genesis
from genesis_b200.models.transformers import MoEConfig, MoEForCausalLM, QwenForCausalLM, TransformerConfig
from genesis_b200.nn import PagedKVCache


def _model(kind):
    genesis.manual_seed(11)
    base = dict(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, head_dim=16, max_position_embeddings=64, rope_theta=1e4)
    if kind == "dense":
        return QwenForCausalLM(TransformerConfig(**base)).eval()
    return MoEForCausalLM(MoEConfig(**base, num_experts_per_tok=2, num_local_experts=4, moe_intermediate_size=48)).eval()


def _ints(*xs):
    return genesis.Tensor(torch.tensor(xs, dtype=torch.int32))


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_greedy_tokens_are_the_same(kind):
    m = _model(kind)
    prompt = genesis.Tensor(torch.randint(0, 97, (3, 9), generator=torch.Generator().manual_seed(1)))
    want = m.generate(prompt, max_new_tokens=12, temperature=0.0)
    got = m.generate(prompt, max_new_tokens=12, temperature=0.0, cache_dtype="float32")
    assert got.shape == (3, 21) and torch.equal(got._t, want._t)
    assert torch.equal(m.generate(prompt, max_new_tokens=0, cache_dtype="float32")._t, prompt._t)
    short = m.generate(prompt, max_new_tokens=3, temperature=0.8, top_k=5, cache_dtype="float8_e4m3fn")
    assert short.shape == (3, 12) and torch.equal(short._t[:, :9], prompt._t) and int(short._t.max()) < 97
    with pytest.raises(ValueError, match="a cache holds one of"):
        m.generate(prompt, max_new_tokens=1, cache_dtype="int8")


def test_training_mode_is_given_back():
    m = _model("dense").train()
    m.generate(genesis.Tensor(torch.zeros(1, 2, dtype=torch.int64)), max_new_tokens=2, cache_dtype="float32")
    assert m.training


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_ragged_prompts_pieces_and_single_tokens(kind):
    """Prompts of different lengths, padded to one call; then pieces, single tokens, and a sequence that rests."""
    m = _model(kind)
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 97, (3, 40), generator=g)
    with genesis.no_grad():
        full = [m(genesis.Tensor(tokens[b:b + 1]))._t[0] for b in range(3)]
        cache = PagedKVCache(12, 2, 16, page_size=16, num_layers=2, dtype="float32")
        table = cache.page_table(cache.allocate([40, 40, 40]))
        have = [7, 20, 1]
        idx = torch.zeros(3, 20, dtype=torch.int64)
        for b, n in enumerate(have):
            idx[b, :n] = tokens[b, :n]
        out = m.forward_paged(genesis.Tensor(idx), cache, table, _ints(*have), _ints(*have), prompt=True)
        assert out.shape == (3, 1, 97)
        for b, n in enumerate(have):
            assert torch.allclose(out._t[b, 0], full[b][n - 1], atol=1e-4)
        for counts in ([5, 1, 8], [1, 1, 1], [1, 0, 1], [3, 2, 29]):
            S = max(counts)
            idx = torch.zeros(3, S, dtype=torch.int64)
            for b, n in enumerate(counts):
                idx[b, :n] = tokens[b, have[b]:have[b] + n]
            have = [a + n for a, n in zip(have, counts)]
            out = m.forward_paged(genesis.Tensor(idx), cache, table, _ints(*have), _ints(*counts), last=False)._t
            for b, n in enumerate(counts):
                for s in range(n):
                    assert torch.allclose(out[b, s], full[b][have[b] - n + s], atol=1e-4)
    assert have[2] == 40


def test_positions_behind_the_rotation_tables():
    """A page table with more room than the tables: they grow, and the old ones stay for whoever reads them."""
    m = _model("dense")
    rot = m.model.layers[0].self_attn.rotary_emb
    old = rot.cos_cached
    tokens = torch.randint(0, 97, (1, 70), generator=torch.Generator().manual_seed(3))
    with genesis.no_grad():
        cache = PagedKVCache(6, 2, 16, page_size=16, num_layers=2, dtype="float32")
        table = cache.page_table(cache.allocate([96]))
        m.forward_paged(genesis.Tensor(tokens[:, :69]), cache, table, _ints(69), prompt=True)
        out = m.forward_paged(genesis.Tensor(tokens[:, 69:]), cache, table, _ints(70))
        assert rot.max_seq_len_cached >= 96 and rot._outgrown[0][0] is old
        assert torch.allclose(out._t[0, 0], m(genesis.Tensor(tokens))._t[0, 69], atol=1e-4)
        # padding behind the prompt may be longer than the table has room for
        cache = PagedKVCache(1, 2, 16, page_size=16, num_layers=2, dtype="float32")
        table = cache.page_table(cache.allocate([5]))
        short = m.forward_paged(genesis.Tensor(tokens[:, :40]), cache, table, _ints(5), _ints(5), prompt=True)
        assert torch.allclose(short._t[0, 0], m(genesis.Tensor(tokens[:, :5]))._t[0, 4], atol=1e-4)
