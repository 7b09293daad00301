"""Next-token sampling shared by the dense and MoE language models: temperature, top-k, nucleus (top-p), drawn with
the Gumbel-max trick so the whole step stays on the device (top-k / sort / arg-max are the framework's own kernels,
the noise comes from its Philox generator).  Reference counterpart: the sampling loop of
genesis/models/transformers/moe.py:546-590 (softmax + multinomial on the host library)."""
import torch

from ... import random as _random
from ...ops import dispatch as K


def sample_next(logits, temperature=1.0, top_k=None, top_p=None):
    """logits: raw float tensor [B, V] -> int64 token ids [B, 1].  temperature 0 means greedy."""
    x = logits.float()
    if temperature is None or temperature <= 0.0:
        return K.argmax(x, -1, True)
    if temperature != 1.0:
        x = x / temperature
    V = x.shape[-1]
    if top_k is not None and 0 < top_k < V:
        kth = K.topk(x, int(top_k), -1, True)[0][:, -1:]
        x = torch.where(x < kth, torch.full_like(x, float("-inf")), x)
    if top_p is not None and 0.0 < top_p < 1.0:
        sv, si = K.sort(x, -1, True)
        sp = torch.softmax(sv, -1)
        before = torch.cumsum(sp, -1) - sp                     # probability mass ranked above each token
        sv = torch.where(before >= top_p, torch.full_like(sv, float("-inf")), sv)
        x = torch.full_like(x, float("-inf")).scatter_(-1, si, sv)
    seed, offset = _random.default_generator().next_philox()
    u = K.random_fill("uniform", tuple(x.shape), torch.float32, x.device, seed, offset, 0.0, 1.0)
    u = u.clamp_(1e-20, 1.0 - 1e-7)
    gumbel = -torch.log(-torch.log(u))
    return K.argmax(x + gumbel, -1, True)


def generate_paged(model, input_ids, max_new_tokens, temperature, top_k, top_p, cache_dtype, page_size=64):
    """Appends `max_new_tokens` sampled tokens to `input_ids` [B, S], with keys and values kept in a paged cache of
    `cache_dtype`: the prompt is encoded once, then one token of each sequence a step.  `model` has a `config` and
    `forward_paged`."""
    from ... import grad_mode
    from ...nn.paged import PagedKVCache
    from ...tensor import Tensor
    cfg, out = model.config, input_ids._t
    B, S = out.shape
    with grad_mode.no_grad():
        most = S + max_new_tokens
        per = -(-most // page_size)
        cache = PagedKVCache(max(1, B * per), cfg.num_key_value_heads, cfg.head_dim, page_size=page_size,
                             num_layers=cfg.num_hidden_layers, dtype=cache_dtype, device=out.device)
        table = cache.page_table(cache.allocate([most] * B))
        lengths = Tensor._wrap(torch.full((B,), S, dtype=torch.int32, device=out.device))
        step = out
        for i in range(max_new_tokens):
            if i > 0:
                lengths._t += 1
            logits = model.forward_paged(Tensor._wrap(step), cache, table, lengths, lengths if i == 0 else None, prompt=i == 0)
            step = sample_next(logits._t[:, -1, :], temperature, top_k, top_p).to(out.dtype)
            out = torch.cat((out, step), dim=1)
    return Tensor._wrap(out)
