"""Modules whose calls are observed are called: the latent attention's absorbed form, which takes
kv_b_proj's weight, is not for them."""
import pytest
import torch.nn as nn
from torch.nn.modules import module as M

from lightcompress_amd.deepseekv3 import _plain_weight


@pytest.mark.parametrize('register', [
    lambda lin: lin.register_forward_hook(lambda *a: None),
    lambda lin: lin.register_forward_pre_hook(lambda *a: None),
    lambda lin: M.register_module_forward_hook(lambda *a: None),
    lambda lin: M.register_module_forward_pre_hook(lambda *a: None)])
def test_observed_linears_are_not_plain_weights(register):
    lin = nn.Linear(8, 4, bias=False)
    assert _plain_weight(lin) is lin.weight
    hook = register(lin)
    try:
        assert _plain_weight(lin) is None
    finally:
        hook.remove()
    assert _plain_weight(lin) is lin.weight
    assert _plain_weight(nn.Linear(8, 4)) is None       # a bias
