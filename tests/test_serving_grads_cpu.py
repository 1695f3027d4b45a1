"""The packed products and the latent attention have no backward pass: what would lose a gradient
is refused or takes another path. Decided on the host, so without a GPU."""
import types

import torch
import torch.nn as nn

from lightcompress_amd import deepseekv3 as D


def attention():
    """What _lcq_mla_past asks of an attention module."""
    attn = nn.Linear(4, 4).requires_grad_(False).eval()
    attn.attention_dropout, attn.layer_idx = 0.0, 0
    attn.qk_nope_head_dim, attn.qk_rope_head_dim = 128, 64
    attn.v_head_dim, attn.kv_lora_rank = 128, 512
    attn.config = types.SimpleNamespace(_attn_implementation='sdpa')
    return attn


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on the device."""
    is_cuda = True


def hidden(requires_grad=False, S=5):
    x = torch.zeros(1, S, 4, dtype=torch.bfloat16).as_subclass(OnDevice)
    return x.requires_grad_(requires_grad)


def rotary(requires_grad=False):
    t = torch.zeros(1, 5, 64, dtype=torch.bfloat16, requires_grad=requires_grad)
    return t, t


def past(attn, x, pos, cache=None):
    return D._lcq_mla_past(attn, x, pos, None, cache, {})


def test_attention_keeps_the_gradient_of_its_inputs():
    """Frozen parameters, an input that requires a gradient: the stock forward runs."""
    attn = attention()
    assert past(attn, hidden(), rotary()) == 0
    assert past(attn, hidden(True), rotary()) is None
    assert past(attn, hidden(), rotary(True)) is None
    with torch.no_grad():
        assert past(attn, hidden(True), rotary(True)) == 0
    attn.requires_grad_(True)
    assert past(attn, hidden(), rotary()) is None


def test_attention_keeps_the_gradient_of_cached_tokens():
    from transformers import DynamicCache
    attn, cache = attention(), DynamicCache()
    k = torch.zeros(1, 1, 3, 512, requires_grad=True)
    cache.update(k, torch.zeros(1, 1, 3, 64), 0)
    assert past(attn, hidden(S=1), rotary(), cache) is None
    with torch.no_grad():
        assert past(attn, hidden(S=1), rotary(), cache) == 3
    cache = DynamicCache()
    cache.update(k.detach(), torch.zeros(1, 1, 3, 64), 0)
    assert past(attn, hidden(S=1), rotary(), cache) == 3
