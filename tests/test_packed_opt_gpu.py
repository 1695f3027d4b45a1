"""A deployed OPT runs: fp16, linears with biases, several steps through a cache."""
import copy

import pytest
import torch
import torch.nn as nn

from oracle import int4_ref as R
from test_packed_model_gpu import FORMATS, buffers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('fmt,weight', FORMATS)
def test_packed_opt_prompt_and_decode(dev, fmt, weight):
    """Against float32 on the unpacked weights: the packed model's error is within twice that of
    the fp16 forward on those weights."""
    from transformers import DynamicCache, OPTConfig, OPTForCausalLM

    from lightcompress_amd.opt import Opt
    from lightcompress_amd.pipeline import build_algo
    from lightcompress_amd.utils import load_config
    torch.manual_seed(0)
    hf = OPTForCausalLM(OPTConfig(
        hidden_size=256, ffn_dim=384, num_attention_heads=4, num_hidden_layers=2, vocab_size=128,
        max_position_embeddings=128, word_embed_proj_dim=256))
    for n, p in hf.named_parameters():
        p.data = torch.randn(p.shape) * (p.shape[-1] ** -0.5 if p.dim() > 1 else 0.3)
    model = Opt({'model': {}}, hf_model=hf.to(torch.float16), device=dev)
    algo = build_algo(model, load_config({'quant': {'method': 'RTN', 'weight': dict(weight)}}),
                      None)
    algo.run_block_loop()
    algo.deploy(fmt)
    plain = copy.deepcopy(model.model)
    n = 0
    for name, m in list(plain.named_modules()):
        m.__dict__.pop('forward', None)
        if hasattr(m, 'int4_forward'):
            assert m.int4_forward and m.bias is not None
            c, z, s = R.unpack(*buffers(m))
            f = nn.Linear(m.in_features, m.out_features)
            f.weight.data, f.bias.data = ((c - z) * s).float(), m.bias.data.float().cpu()
            parent, leaf = name.rsplit('.', 1)
            setattr(plain.get_submodule(parent), leaf, f)
            n += 1
    assert n == 12
    plain = plain.cpu().float()
    ids = torch.randint(0, 128, (2, 40), generator=torch.Generator().manual_seed(1))

    def run(m, ids):
        cache, out = DynamicCache(), []
        with torch.no_grad():
            for t in (ids[:, :38], ids[:, 38:39], ids[:, 39:]):
                out.append(m(t, past_key_values=cache, use_cache=True).logits)
        return torch.cat(out, 1).float().cpu()
    with torch.no_grad():
        want = plain(ids).logits
    got = run(model.model, ids.to(dev))
    stock = run(plain.to(torch.float16).to(dev), ids.to(dev))
    e_got, e_stock = (got - want).norm(), (stock - want).norm()
    assert e_got <= 2 * e_stock, (e_got, e_stock)
