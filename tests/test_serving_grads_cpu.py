"""The packed products and the latent attention have no backward pass: what would lose a gradient
is refused or takes another path. Decided on the host, so without a GPU."""
import types

import pytest
import torch
import torch.nn as nn

from lightcompress_amd import _native as N
from lightcompress_amd import deepseekv3 as D
from lightcompress_amd import ops


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


def test_operators_refuse_inputs_that_require_a_gradient():
    qw, s = torch.zeros(64, 32, dtype=torch.int32), torch.ones(64, 2, dtype=torch.float16)
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    off, rows = torch.tensor([0, 3]), torch.arange(3)
    tab = ops.int4_weight_table([(qw, s)], 'cpu')
    q = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    kr = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    ql = torch.zeros(1, 1, 2, 512, dtype=torch.bfloat16)
    c = torch.zeros(3, 16, 576, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    bias = torch.zeros(64, dtype=torch.bfloat16)
    calls = [
        (lambda x, s, bias: ops.int4_linear(x, qw, s, bias=bias), (x, s, bias)),
        (lambda x: ops.int4_linear_grouped(x, off, tab, 64, 128, a_rows=rows), (x,)),
        (lambda *a: ops.mla_fwd_causal(*a, 0.1),
         (q, q[..., :64].clone(), q.clone(), kr, q.clone())),
        (lambda *a: ops.mla_decode(*a, t, n, 0.1),
         (ql, ql[..., :64].clone(), c[..., :512].clone(), c[..., 512:].clone()))]
    for fn, args in calls:
        for i in range(len(args)):
            a = [u.detach().clone().requires_grad_(j == i) for j, u in enumerate(args)]
            with pytest.raises(RuntimeError, match='gradient'):
                fn(*a)
            with torch.no_grad(), pytest.raises(N.LcqError, match='GPU only'):
                fn(*a)          # past that check


def test_experts_keep_the_gradient_of_the_combine(monkeypatch):
    """Routing weights that require a gradient: the experts run one by one, where the combine has
    a backward pass."""
    experts = D.ExpertList([nn.Linear(4, 4).requires_grad_(False) for _ in range(2)])
    monkeypatch.setattr(D.ExpertList, '_grouped_fp8_ok', lambda *a: False)
    monkeypatch.setattr(D.ExpertList, '_grouped_int4_ok', lambda *a: True)
    monkeypatch.setattr(D.ExpertList, '_forward_grouped_int4', lambda *a: 'grouped')
    x, idx = torch.randn(3, 4), torch.tensor([[0, 1], [1, 0], [0, 1]])
    w = torch.rand(3, 2)
    assert experts(x, idx, w) == 'grouped'
    w.requires_grad_(True)
    experts(x, idx, w).square().sum().backward()
    out = torch.stack([experts[e](x) for e in range(2)])             # [2, 3, 4]
    h = torch.stack([out[idx[:, j], torch.arange(3)] for j in range(2)], 1)   # [3, 2, 4]
    y = (h * w.detach()[..., None]).sum(1)
    # sums of 4 fp32 products of size about 1, each step off by 2^-24 of it
    assert torch.allclose(w.grad, (2 * y[:, None] * h).sum(-1), atol=1e-5)
    with torch.no_grad():
        assert experts(x, idx, w) == 'grouped'
