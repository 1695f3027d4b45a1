"""The DeepSeek-V3 attention on latents behind caches of several kinds: a preallocated cache hands
back its whole buffer, of which only the tokens written so far count."""
import copy

import pytest
import torch

from oracle import int4_ref as R
from test_packed_model_gpu import VLLM, adapter, buffers, dsv3, pack

pytestmark = pytest.mark.gpu


def logits_of(model, cache, prompts):
    """Logits of prompts run one after the other, the cache reset before each: the first tokens at
    once, then the last two one by one."""
    out = []
    with torch.no_grad():
        for ids in prompts:
            cache.reset()
            n = ids.shape[1] - 2
            steps = [ids[:, :n], ids[:, n:n + 1], ids[:, n + 1:]]
            out.append(torch.cat([model(t, past_key_values=cache, use_cache=True).logits
                                  for t in steps], 1).float().cpu())
    return out


@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('kind', ['static', 'dynamic'])
def test_dsv3_prompt_and_decode_behind_a_cache(dev, monkeypatch, kind, packed):
    """model.attention 'lcq' against the stock forward with the same cache, both against float32
    without one: its error is within twice the stock bf16 forward's. The second prompt is shorter
    than what the first left behind."""
    from transformers import DynamicCache, StaticCache

    from lightcompress_amd import ops
    hf = dsv3(dev)
    if packed:
        for layer in hf.model.layers:
            layer.self_attn.kv_b_proj = pack('vllm_quant', VLLM, layer.self_attn.kv_b_proj.to(dev))
    ref = copy.deepcopy(hf)
    for layer in ref.model.layers if packed else ():
        c, z, s = R.unpack(*buffers(layer.self_attn.kv_b_proj))
        lin = torch.nn.Linear(c.shape[1], c.shape[0], bias=False)
        lin.weight.data = ((c - z) * s).float()
        layer.self_attn.kv_b_proj = lin
    ref = ref.cpu().float()
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 128, (2, n), generator=g) for n in (37, 20)]
    with torch.no_grad():
        want = [ref(ids).logits for ids in prompts]

    def cache():
        return (StaticCache(config=hf.config, max_cache_len=64) if kind == 'static'
                else DynamicCache())
    prompts = [ids.to(dev) for ids in prompts]
    if kind == 'dynamic':      # nothing to reset: a new one for each prompt
        def run(m):
            return [logits_of(m, cache(), [ids])[0] for ids in prompts]
    else:
        def run(m):
            return logits_of(m, cache(), prompts)
    stock = run(adapter(copy.deepcopy(hf), dev, 'sdpa').model)
    calls = []
    for f in ('mla_fwd_causal', 'mla_decode'):
        fn = getattr(ops, f)
        monkeypatch.setattr(ops, f, lambda *a, _f=f, _fn=fn, **k: calls.append(_f) or _fn(*a, **k))
    got = run(adapter(hf, dev, 'lcq').model)
    assert 'mla_fwd_causal' in calls
    assert ('mla_decode' in calls) == (kind == 'dynamic' and not packed)
    for a, b, w in zip(got, stock, want):
        e_got, e_stock = (a - w).norm(), (b - w).norm()
        assert e_got <= 2 * e_stock, (e_got, e_stock)
