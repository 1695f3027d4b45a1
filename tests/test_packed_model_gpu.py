"""The packed model runs: the deployed int4 linears' own forward, the routed experts in one launch
per projection, latent attention in the DeepSeek-V3 forwards, and all of them together."""
import copy

import pytest
import torch
import torch.nn as nn

from oracle import int4_ref as R
from test_pipeline_gpu import calib, tiny_model

pytestmark = pytest.mark.gpu

VLLM = {'bit': 4, 'symmetric': True, 'granularity': 'per_group', 'group_size': 128,
        'need_pack': True}
AWQ = {'bit': 4, 'symmetric': False, 'granularity': 'per_group', 'group_size': 128,
       'pack_version': 'gemm_pack'}
FORMATS = [('vllm_quant', VLLM), ('autoawq_quant', AWQ)]


def pack(fmt, weight, lin):
    """lin as the deployed module of this format."""
    from functools import partial

    from lightcompress_amd.module_utils import _REALQUANT_LINEAR_MAP_
    from lightcompress_amd.quant import IntegerQuantizer
    wq = IntegerQuantizer(**{k: v for k, v in weight.items() if k not in ('need_pack',)})
    return _REALQUANT_LINEAR_MAP_[fmt].new(
        lin, partial(lambda m, wquantizer: wquantizer.real_quant_weight_dynamic(m.weight.data),
                     wquantizer=wq), {'weight': weight})


def lin(g, i, o, dev, bias=False, dt=torch.bfloat16):
    m = nn.Linear(i, o, bias=bias)
    m.weight.data = (torch.randn(o, i, generator=g) * 0.05).to(dt)
    if bias:
        m.bias.data = torch.randn(o, generator=g).to(dt)
    return m.to(dev)


def buffers(m):
    from lightcompress_amd.module_utils import AutoawqRealQuantLinear
    if isinstance(m, AutoawqRealQuantLinear):
        return m.qweight, m.scales, m.qzeros
    return m.weight_packed, m.weight_scale, None


@pytest.mark.parametrize('fmt,weight', FORMATS + [
    ('vllm_quant', {**VLLM, 'granularity': 'per_channel'}),
    ('sgl_quant', {**VLLM, 'group_size': 64}), ('mlcllm_quant', {**AWQ, 'group_size': 64})])
def test_deployed_linear_forward(dev, fmt, weight):
    """The forward is the product with the packed weight, and that weight is the layer's own within
    its quantization step. (AutoAWQ packs unclamped codes: one outside 0..15 spills into its word's
    other seven columns, so those words are left out.)"""
    g = torch.Generator().manual_seed(1)
    weight = {k: v for k, v in weight.items()
              if k != 'group_size' or weight['granularity'] == 'per_group'}
    m = lin(g, 384, 264, dev, bias=True)
    p = pack(fmt, weight, m)
    for shape in ((2, 5, 384), (150, 384)):
        x = torch.randn(*shape, generator=g).to(torch.bfloat16).to(dev)
        y, tol = R.linear(x.reshape(-1, 384), *buffers(p), bias=p.bias)
        assert R.close(p(x).reshape(-1, 264), y, tol)
    c, z, s = R.unpack(*buffers(p))
    w = m.weight.detach().cpu().double()
    code = (w / s + z).round()
    ok = ((code >= 0) & (code <= 15)).view(264 // 8, 8, 384).all(1, keepdim=True).expand(
        -1, 8, -1).reshape(264, 384)
    if weight['symmetric']:
        ok = torch.ones_like(ok)
    assert ok.float().mean() > 0.9
    assert (((c - z) * s - w).abs() <= s * (1 if weight['symmetric'] else 2))[ok].all()


def test_deployed_linear_refusals(dev):
    """What the packed buffers cannot say stays an error: zero points vLLM's layout does not hold,
    other bit widths, quantized activations."""
    g = torch.Generator().manual_seed(2)
    m = lin(g, 256, 64, dev)
    x = torch.randn(3, 256, device=dev).to(torch.bfloat16)
    for w in ({**VLLM, 'symmetric': False}, {**VLLM, 'bit': 8}, {**VLLM, 'need_pack': False}):
        with pytest.raises(NotImplementedError):
            pack('vllm_quant', w, m)(x)
    p = pack('vllm_quant', VLLM, m)
    from lightcompress_amd.module_utils import _vllm_int4
    assert _vllm_int4({'weight': VLLM}) and not _vllm_int4({'weight': VLLM, 'act': {'bit': 8}})
    with pytest.raises(TypeError):
        p(x.float())
    with pytest.raises(ValueError):
        p(x[:, :128])
    from lightcompress_amd._native import LcqError
    with pytest.raises((ValueError, LcqError)):
        p(x.cpu())


@pytest.mark.parametrize('fmt,weight', FORMATS)
def test_packed_llama_forward(dev, fmt, weight):
    """A Llama deployed to a packed format runs; against the same weights as float linears."""
    from lightcompress_amd.pipeline import build_algo
    from lightcompress_amd.utils import load_config
    model = tiny_model(dev)
    inp = calib(model)
    algo = build_algo(model, load_config({'quant': {'method': 'RTN', 'weight': dict(weight)}}),
                      None)
    algo.run_block_loop()
    algo.deploy(fmt)

    def run(x=None):
        x = inp['data'][0] if x is None else x
        for b in model.blocks:
            x = b(x, **inp['kwargs'][0])
            x = x[0] if isinstance(x, tuple) else x
        return x.float()
    with torch.no_grad():
        got = run()
        x = inp['data'][0].clone()
        run(x)
        x.data = -x.data            # the same tensor object, another content and version
        assert torch.equal(run(x), run(x.clone()))
        for b in model.blocks:                      # the same weights, unpacked
            for name, m in list(b.named_modules()):
                if hasattr(m, 'int4_forward'):
                    c, z, s = R.unpack(*buffers(m))
                    f = nn.Linear(m.in_features, m.out_features, bias=False, device=dev,
                                  dtype=torch.bfloat16)
                    f.weight.data = ((c - z) * s).to(torch.bfloat16).to(dev)
                    parent, leaf = name.rsplit('.', 1)
                    setattr(b.get_submodule(parent), leaf, f)
        want = run()
    # bf16 roundings of the weights (2^-9) and of the activations after each of the 14 linears
    assert (got - want).norm() <= 16 * 2. ** -9 * want.norm()


def experts_of(dev, fmt, weight, E, H, inter, seed):
    from transformers.models.deepseek_v3 import modeling_deepseek_v3 as md

    from lightcompress_amd.deepseekv3 import ExpertList
    cfg = md.DeepseekV3Config(hidden_size=H, intermediate_size=inter, hidden_act='silu')
    g = torch.Generator().manual_seed(seed)
    out = ExpertList()
    for _ in range(E):
        mlp = md.DeepseekV3MLP(cfg, intermediate_size=inter)
        for p in ('gate_proj', 'up_proj', 'down_proj'):
            f = getattr(mlp, p)
            setattr(mlp, p, pack(fmt, weight, lin(g, f.in_features, f.out_features, dev)))
        out.append(mlp)
    return out


@pytest.mark.parametrize('fmt,weight', FORMATS)
@pytest.mark.parametrize('T', [1, 7, 300])
def test_packed_experts_grouped(dev, monkeypatch, fmt, weight, T):
    """ExpertList's one launch per projection against the per-expert loop of packed modules. They
    differ by the loop's extra bf16 roundings of gate, up and silu (2^-9 each) and the gate / up
    sums' order: a few 2^-9 of the expert outputs' size."""
    from lightcompress_amd.deepseekv3 import ExpertList
    E, H, inter, k = 8, 512, 384, 3
    experts = experts_of(dev, fmt, weight, E, H, inter, seed=4)
    g = torch.Generator().manual_seed(T)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(dev)
    w = torch.rand(T, k, generator=g).to(dev)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(dev)
    assert experts._grouped_int4_ok(x)
    got = experts(x, idx, w)
    hook = experts[2].up_proj.register_forward_hook(lambda *a: None)
    assert not experts._grouped_int4_ok(x)         # observed experts run one by one
    hook.remove()
    monkeypatch.setattr(ExpertList, '_grouped_int4_ok', lambda self, x: False)
    want = experts(x, idx, w)
    assert got.shape == want.shape
    assert (got - want).float().norm() <= 4 * 2. ** -9 * want.float().norm()
    assert not experts._grouped_fp8_ok(x)


def dsv3(dev, seed=0, layers=2):
    """A DeepSeek-V3 with the checkpoint's head dims, small elsewhere; every token goes to all
    experts, so a rounding cannot reroute one."""
    from transformers.models.deepseek_v3 import modeling_deepseek_v3 as md
    cfg = md.DeepseekV3Config(
        hidden_size=256, intermediate_size=384, moe_intermediate_size=128, num_hidden_layers=layers,
        num_attention_heads=4, num_key_value_heads=4, n_routed_experts=4, num_experts_per_tok=4,
        n_shared_experts=1, n_group=1, topk_group=1, first_k_dense_replace=1, q_lora_rank=128,
        kv_lora_rank=512, qk_nope_head_dim=128, qk_rope_head_dim=64, v_head_dim=128,
        vocab_size=128, max_position_embeddings=512, attn_implementation='sdpa')
    torch.manual_seed(seed)
    model = md.DeepseekV3ForCausalLM(cfg)
    for n, p in model.named_parameters():
        if p.dim() > 1:
            p.data = torch.randn(p.shape) * (2.0 if 'embed' in n else p.shape[-1] ** -0.5)
    return model.to(torch.bfloat16)


def adapter(hf, dev, attention):
    from lightcompress_amd.deepseekv3 import DeepseekV3
    return DeepseekV3({'model': {'attention': attention}}, hf_model=hf, device=dev)


def logits_of(model, ids, steps):
    """Prompt logits, then `steps` single-token decodes through the cache."""
    from transformers import DynamicCache
    cache = DynamicCache()
    out = []
    n = ids.shape[1] - steps
    with torch.no_grad():
        out.append(model(ids[:, :n], past_key_values=cache, use_cache=True).logits)
        for t in range(n, ids.shape[1]):
            out.append(model(ids[:, t:t + 1], past_key_values=cache, use_cache=True).logits)
    return torch.cat(out, 1).float().cpu()


@pytest.mark.parametrize('B,S,steps', [(1, 40, 3), (2, 130, 2)])
def test_dsv3_attention_prompt_and_decode(dev, monkeypatch, B, S, steps):
    """model.attention 'lcq' against transformers' sdpa, both against float32: its error is within
    twice the stock bf16 forward's. The prompt runs expanded, the new tokens absorbed."""
    from lightcompress_amd import ops
    hf = dsv3(dev)
    ref = copy.deepcopy(hf).float()
    ids = torch.randint(0, 128, (B, S), generator=torch.Generator().manual_seed(S))
    with torch.no_grad():
        want = ref(ids).logits
    stock = logits_of(adapter(copy.deepcopy(hf), dev, 'sdpa').model, ids.to(dev), steps)
    calls = []
    for f in ('mla_fwd_causal', 'mla_decode'):
        fn = getattr(ops, f)
        monkeypatch.setattr(ops, f, lambda *a, _f=f, _fn=fn, **k: calls.append(_f) or _fn(*a, **k))
    got = logits_of(adapter(hf, dev, 'lcq').model, ids.to(dev), steps)
    assert calls == ['mla_fwd_causal'] * 2 + ['mla_decode'] * 2 * steps
    e_got, e_stock = (got - want).norm(), (stock - want).norm()
    assert e_got <= 2 * e_stock, (e_got, e_stock)


def test_dsv3_attention_masked_batch_takes_the_stock_forward(dev, monkeypatch):
    from lightcompress_amd import ops
    hf = dsv3(dev)
    ids = torch.randint(0, 128, (2, 20), generator=torch.Generator().manual_seed(3)).to(dev)
    mask = torch.ones_like(ids)
    mask[0, :6] = 0
    with torch.no_grad():
        want = adapter(copy.deepcopy(hf), dev, 'sdpa').model(ids, attention_mask=mask).logits
        got = adapter(hf, dev, 'lcq').model(ids, attention_mask=mask).logits
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        adapter(hf, dev, 'flash')


@pytest.mark.parametrize('fmt,weight', FORMATS)
def test_packed_dsv3_prompt_and_decode(dev, monkeypatch, fmt, weight):
    """All of it together: a DeepSeek-V3 deployed to a packed format, prompt and decode with the
    lcq attention and grouped experts, against float32 on the unpacked weights: its error within
    twice that of the stock bf16 forward on those weights."""
    from lightcompress_amd import ops
    from lightcompress_amd.pipeline import build_algo
    from lightcompress_amd.utils import load_config
    hf = dsv3(dev, seed=1)
    model = adapter(hf, dev, 'lcq')
    algo = build_algo(model, load_config({'quant': {'method': 'RTN', 'weight': dict(weight)}}),
                      None)
    algo.run_block_loop()
    algo.deploy(fmt)
    ids = torch.randint(0, 128, (2, 50), generator=torch.Generator().manual_seed(5))
    calls = []
    for f in ('mla_fwd_causal', 'int4_linear', 'int4_linear_grouped'):
        fn = getattr(ops, f)
        monkeypatch.setattr(ops, f, lambda *a, _f=f, _fn=fn, **k: calls.append(_f) or _fn(*a, **k))
    got = logits_of(model.model, ids.to(dev), 2)
    assert {'mla_fwd_causal', 'int4_linear', 'int4_linear_grouped'} == set(calls)
    monkeypatch.undo()
    plain = copy.deepcopy(model.model)
    for m in plain.modules():
        m.__dict__.pop('forward', None)            # the stock attention and linears
        m.__dict__.pop('_lcq_int4_tables', None)
    for name, m in list(plain.named_modules()):
        if hasattr(m, 'int4_forward'):
            c, z, s = R.unpack(*buffers(m))
            f = nn.Linear(m.in_features, m.out_features, bias=False)
            f.weight.data = ((c - z) * s).float()
            parent, leaf = name.rsplit('.', 1)
            setattr(plain.get_submodule(parent), leaf, f)
    plain = plain.cpu().float()
    with torch.no_grad():
        want = plain(ids).logits
    stock = logits_of(plain.to(torch.bfloat16).to(dev), ids.to(dev), 2)
    e_got, e_stock = (got - want).norm(), (stock - want).norm()
    assert e_got <= 2 * e_stock, (e_got, e_stock)
