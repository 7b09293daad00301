"""Calls on a paged cache at the edges of what their documentation allows, on the CPU."""
import copy
import gc
import weakref

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.models.transformers import MoEConfig, MoEForCausalLM, QwenForCausalLM, TransformerConfig
from genesis_b200.models.transformers.components import RotaryEmbedding, apply_rope
from genesis_b200.nn import PagedKVCache

import _paged_ref as R


def test_rotation_tables_without_a_position():
    t = R.Setup([20, 0], 2, 8, "fp32")
    y, none = t.tensor(torch.ones(2, 1, 8 * 8)), t.tensor(torch.zeros(0, 8))
    before = R.values(t.layer.k, None)
    with pytest.raises(IndexError, match="rotation tables of 0 positions"):
        F.paged_qkv_rope(y, none, none, t.layer, t.table, t.lens, 4)
    assert torch.equal(R.values(t.layer.k, None).nan_to_num(7e9), before.nan_to_num(7e9))
    q = F.paged_qkv_rope(y, none, none, t.layer, t.table, t.ints([0, 0]), 4)      # no token: nothing to rotate
    assert torch.all(q._t == 0)


# ---- rotation tables of a model ------------------------------------------------------------------
def _model(kind, positions=64, seed=11):
    genesis.manual_seed(seed)
    base = dict(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, head_dim=16, max_position_embeddings=positions, rope_theta=1e4)
    if kind == "dense":
        return QwenForCausalLM(TransformerConfig(**base)).eval()
    return MoEForCausalLM(MoEConfig(**base, num_experts_per_tok=2, num_local_experts=4, moe_intermediate_size=48)).eval()


def _ints(*xs):
    return genesis.Tensor(torch.tensor(xs, dtype=torch.int32))


def _rotaries(m):
    return [layer.self_attn.rotary_emb for layer in m.model.layers]


def _tokens(*shape, seed=3):
    return genesis.Tensor(torch.randint(0, 97, shape, generator=torch.Generator().manual_seed(seed)))


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_outgrown_tables_are_no_part_of_a_checkpoint(kind):
    m = _model(kind)
    keys, buffers = list(m.state_dict()), [n for n, _ in m.named_buffers()]
    m.generate(_tokens(2, 5), max_new_tokens=70, temperature=0.0, cache_dtype="float32")
    assert _rotaries(m)[0].max_seq_len_cached > 64
    assert list(m.state_dict()) == keys and [n for n, _ in m.named_buffers()] == buffers
    fresh = _model(kind, seed=12)
    assert fresh.load_state_dict(m.state_dict()) == ([], []) and m.load_state_dict(fresh.state_dict()) == ([], [])
    twin = copy.deepcopy(m)
    assert list(twin.state_dict()) == keys
    # what a captured step reads is neither converted nor moved
    kept = [(t, t._t) for pair in _rotaries(m)[0]._outgrown for t in pair]
    m.bfloat16()
    assert kept and all(t._t is raw for t, raw in kept)


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("grow", ["forward", "forward_paged", "rotary", "apply_rope"])
def test_outgrown_tables_stay_whoever_outgrows_them(kind, grow):
    """A captured step reads the tables it was captured with, whichever call replaces them."""
    m = _model(kind)
    cache = PagedKVCache(8, 2, 16, page_size=16, num_layers=2, dtype="float32")
    with genesis.no_grad():
        m.forward_paged(_tokens(1, 5), cache, cache.page_table(cache.allocate([64])), _ints(5), prompt=True)
        old = [weakref.ref(t._t) for rot in _rotaries(m) for t in (rot.cos_cached, rot.sin_cached)]
        if grow == "forward":
            m(_tokens(1, 65))
        elif grow == "forward_paged":
            m.forward_paged(_tokens(1, 70), cache, cache.page_table(cache.allocate([5])), _ints(5), _ints(5), prompt=True)
        else:
            for rot in _rotaries(m):
                rot(seq_len=65) if grow == "rotary" else apply_rope(genesis.Tensor(torch.zeros(1, 65, 2, 16)), rot)
    assert all(rot.max_seq_len_cached >= 65 for rot in _rotaries(m))
    gc.collect()
    assert all(r() is not None for r in old)


def test_what_is_kept_of_outgrown_tables_is_bounded():
    """A table of pages that widens page by page: a few pairs, which together are no larger than the present ones."""
    m = _model("dense", positions=32)
    cache = PagedKVCache(40, 2, 16, page_size=16, num_layers=2, dtype="float32")
    pages = cache.allocate([5])
    with genesis.no_grad():
        m.forward_paged(_tokens(1, 5), cache, cache.page_table(pages), _ints(5), prompt=True)
        for n in range(6, 500):
            cache.extend(pages, [n])
            if n % 16 == 1:
                m.forward_paged(_tokens(1, 1), cache, cache.page_table(pages), _ints(n))
    for rot in _rotaries(m):
        assert 497 <= rot.max_seq_len_cached <= 1024 and 1 <= len(rot._outgrown) <= 5
        assert sum(cos.shape[0] for cos, _ in rot._outgrown) <= rot.max_seq_len_cached
    plain = _model("dense", positions=32)
    with genesis.no_grad():
        for n in range(33, 200, 7):
            plain(_tokens(1, n))
    assert all(len(rot._outgrown) <= 3 and rot.max_seq_len_cached == 256 for rot in _rotaries(plain))


@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("half", ["bfloat16", "half"])
def test_models_converted_to_16_bits(kind, half):
    """forward_paged rotates by tables in 32 bits, whatever the module's buffers were converted to."""
    answers = []
    for rebuilt in (False, True):
        m = getattr(_model(kind), half)()
        assert _rotaries(m)[0].cos_cached._t.dtype != torch.float32
        keys = list(m.state_dict())
        if rebuilt:                                     # the same model with its buffers in 32 bits
            for rot in _rotaries(m):
                rot._build(64)
        cache = PagedKVCache(8, 2, 16, page_size=16, num_layers=2, dtype="float16")
        table, tokens = cache.page_table(cache.allocate([60, 60])), _tokens(2, 34)
        with genesis.no_grad():
            got = [m.forward_paged(tokens[:, :30], cache, table, _ints(30, 30), prompt=True)._t]
            got += [m.forward_paged(tokens[:, n - 1:n], cache, table, _ints(n, n))._t for n in (31, 32, 33, 34)]
        answers.append(torch.cat(got, 1))
        assert list(m.state_dict()) == keys
        assert all(len(rot._exact) == (0 if rebuilt else 1) for rot in _rotaries(m))
        out = m.generate(_tokens(2, 5), max_new_tokens=4, temperature=0.0, cache_dtype="bfloat16")
        assert out.shape == (2, 9)
        # tables that are outgrown after the conversion
        assert m.generate(_tokens(1, 70), max_new_tokens=2, temperature=0.0, cache_dtype="float8_e4m3fn").shape == (1, 72)
    assert answers[0].dtype == getattr(torch, "float16" if half == "half" else half)
    assert torch.equal(*answers)


# ---- prompts -------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["dense", "moe"])
@pytest.mark.parametrize("last", [True, False])
def test_prompts_padded_in_front(kind, last):
    """Without counts a row's real tokens are its last ones; a prompt is no exception."""
    m = _model(kind)
    tokens, S, have = _tokens(4, 20)._t, 9, [9, 5, 0, 1]
    with genesis.no_grad():
        full = [m(genesis.Tensor(tokens[b:b + 1]))._t[0] for b in range(4)]
        cache = PagedKVCache(8, 2, 16, page_size=16, num_layers=2, dtype="float32")
        table = cache.page_table(cache.allocate([20] * 4))
        idx = torch.full((4, S), 96)
        for b, n in enumerate(have):
            idx[b, S - n:] = tokens[b, :n]
        out = m.forward_paged(genesis.Tensor(idx), cache, table, _ints(*have), prompt=True, last=last)._t
        assert out.shape == (4, 1 if last else S, 97)
        for b, n in enumerate(have):
            assert torch.allclose(out[b, -min(n, out.shape[1]):][:n], full[b][n - min(n, out.shape[1]):n], atol=1e-4)
        for _ in range(3):                                 # what has been put into the cache goes on
            nxt = torch.stack([tokens[b, n:n + 1] for b, n in enumerate(have)])
            have = [n + 1 for n in have]
            out = m.forward_paged(genesis.Tensor(nxt), cache, table, _ints(*have))._t
            for b, n in enumerate(have):
                assert torch.allclose(out[b, 0], full[b][n - 1], atol=1e-4)
        with pytest.raises(TypeError, match="lengths must be an int32 Tensor"):
            m.forward_paged(genesis.Tensor(idx), cache, table, [9, 5, 0, 1], prompt=True)
        with pytest.raises(ValueError, match="lengths must be"):
            m.forward_paged(genesis.Tensor(idx), cache, table, _ints(9, 5), prompt=True)


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_a_refused_generation_leaves_the_mode_as_it_was(kind):
    m = _model(kind).train()
    with pytest.raises(ValueError, match="a cache holds one of"):
        m.generate(_tokens(1, 3), max_new_tokens=1, cache_dtype="int8")
    assert m.training and all(x.training for x in m.modules())
    with pytest.raises(Exception):
        m.generate(_tokens(3), max_new_tokens=1, cache_dtype="float32")          # no [B, S]
    assert m.training
    m.eval()
    with pytest.raises(ValueError):
        m.generate(_tokens(1, 3), max_new_tokens=1, cache_dtype="int8")
    assert not m.training


def test_names_of_the_package():
    """The operators are functions of nn.functional and of the package; what their module imports is neither's."""
    for name in ("paged_attention", "paged_kv_read", "paged_kv_write", "paged_qkv_rope"):
        assert getattr(genesis, name) is getattr(F, name)
    assert not any(hasattr(genesis, name) or hasattr(F, name) for name in ("PagedKVLayer", "PagedKVCache", "pools_of"))
    assert not hasattr(F, "grad_mode") and not hasattr(F, "P")
    assert sorted(genesis.nn.paged.__all__) == ["PagedKVCache", "PagedKVLayer"]


@pytest.mark.parametrize("kind", ["dense", "moe"])
def test_slots_that_rest(kind):
    """Lengths advance by the slots that are active, which are the step's counts: a slot out of use stays so."""
    m = _model(kind)
    tokens = _tokens(3, 20)._t
    cache = PagedKVCache(4, 2, 16, page_size=16, num_layers=2, dtype="float32")
    table = cache.page_table(cache.allocate([20, 0, 20]))
    lengths, active = _ints(5, 0, 7), _ints(1, 0, 1)
    with genesis.no_grad():
        full = [m(genesis.Tensor(tokens[b:b + 1]))._t[0] for b in range(3)]
        m.forward_paged(genesis.Tensor(tokens[:, :7]), cache, table, lengths, lengths, prompt=True)
        have = [5, 0, 7]
        for step in range(6):
            if step == 3:
                active._t[2] = 0                            # this one rests with what it has
            nxt = torch.stack([tokens[b, n:n + 1] for b, n in enumerate(have)])
            have = [n + int(a) for n, a in zip(have, active._t)]
            lengths._t += active._t
            out = m.forward_paged(genesis.Tensor(nxt), cache, table, lengths, active)._t
            for b in range(3):
                if int(active._t[b]):
                    assert torch.allclose(out[b, 0], full[b][have[b] - 1], atol=1e-4)
    assert lengths._t.tolist() == [11, 0, 10]


def test_pieces_read_back_for_flash_attention():
    """Of sequences that are equally long, and of each one alone where they are not."""
    B, Hq, H, D, S = 3, 4, 2, 16, 5
    for lengths in ([30, 30, 30], [30, 17, 9]):
        t = R.Setup(lengths, H, D, "fp32")
        q = t.tensor(t.normal(B, S, Hq, D, dtype="fp32"))
        want = F.paged_attention(q, t.layer, t.table, t.lens)._t
        if len(set(lengths)) == 1:
            k, v = F.paged_kv_read(t.layer, t.table, t.lens, lengths[0])
            assert torch.allclose(F.flash_attention(q, k, v, causal=True)._t, want, atol=1e-5)
        for b, n in enumerate(lengths):
            one = t.tensor(t.table._t[b:b + 1]), t.ints([n])
            k, v = F.paged_kv_read(t.layer, *one, n)
            assert torch.allclose(F.flash_attention(q[b:b + 1], k, v, causal=True)._t, want[b:b + 1], atol=1e-5)


def test_tables_that_cannot_grow_stay_as_they_are(monkeypatch):
    """As while a stream is captured: the next call tries again, and none reads behind the tables' end."""
    rot = RotaryEmbedding(16, 32)
    cos, sin = rot.cos_cached, rot.sin_cached
    with monkeypatch.context() as patch:
        patch.setattr(RotaryEmbedding, "_values", lambda *a: (_ for _ in ()).throw(RuntimeError("capturing")))
        with pytest.raises(RuntimeError, match="capturing"):
            rot.reserve(33)
    assert rot.max_seq_len_cached == 32 and rot.cos_cached is cos and rot.sin_cached is sin and len(rot._outgrown) == 0
    assert F.rope(genesis.Tensor(torch.ones(1, 33, 2, 16)), *rot(seq_len=33)).shape == (1, 33, 2, 16)


def test_lengths_that_blocks_of_16_cannot_count():
    t = R.Setup([3], 1, 8, "fp32")
    for n in (2 ** 31 - 15, 2 ** 31 - 1, 2 ** 40):
        with pytest.raises(ValueError, match="max_length"):
            F.paged_kv_read(t.layer, t.table, t.lens, n)


def test_modules_that_were_pickled_without_a_place_for_old_tables():
    rot = RotaryEmbedding(16, 32)
    del rot._outgrown, rot._exact
    rot.reserve(40)
    assert rot.max_seq_len_cached == 64 and len(rot._outgrown) == 1
    rot.bfloat16()
    cos, _ = rot.tables32()
    assert cos._t.dtype == torch.float32 and cos.shape == (64, 16) and rot.tables32()[0] is cos
