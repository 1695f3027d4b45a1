"""The packed products and latent attention at the far end of their sizes: words, scales and keys
whose offsets pass 31 and 32 bits."""
import pytest
import torch

from oracle import int4_ref as R
from oracle import mla_ref as M

pytestmark = pytest.mark.gpu

N, K, GROUP = 262656, 16352, 32        # n k just below 2^32: 2.1 GB of words


@pytest.mark.parametrize('layout', ['vllm', 'autoawq'])
def test_int4_products_of_the_largest_weight(dev, layout):
    """One row, a few and many against the oracle on columns from both ends and the middle."""
    from lightcompress_amd import ops
    assert N * K < 1 << 32 < (N + 256) * K
    g = torch.Generator(device=dev).manual_seed(1)
    ng = K // GROUP
    shape = (N, K // 8) if layout == 'vllm' else (K, N // 8)
    qw = torch.randint(-2**31, 2**31 - 1, shape, generator=g, dtype=torch.int32, device=dev)
    sshape = (N, ng) if layout == 'vllm' else (ng, N)
    s = torch.rand(sshape, generator=g, device=dev, dtype=torch.float16).mul_(0.01).add_(0.004)
    z = None if layout == 'vllm' else torch.randint(
        -2**31, 2**31 - 1, (ng, N // 8), generator=g, dtype=torch.int32, device=dev)
    for at in (0, N // 2, N - 40):
        cols, words = slice(at, at + 40), slice(at // 8, at // 8 + 5)
        part = ((qw[cols], s[cols].contiguous(), None) if layout == 'vllm' else
                (qw[:, words].contiguous(), s[:, cols].contiguous(), z[:, words].contiguous()))
        for m in (1, 20, 130):
            x = torch.randn(m, K, generator=g, device=dev).bfloat16()
            got = ops.int4_linear(x, qw, s, z)
            y, tol = R.linear(x, *part)
            assert R.close(got[:, cols], y, tol)


def test_mla_prefill_keys_past_32_bits(dev):
    """A few queries behind 70000 tokens of 128 heads: 4.6 GB of keys and values."""
    from lightcompress_amd import ops
    g = torch.Generator(device=dev).manual_seed(2)
    H, Sq, T, dt = 128, 3, 70000, torch.bfloat16
    kv = torch.empty(1, T, H, 256, dtype=dt, device=dev)
    for t in range(0, T, 10000):
        kv[:, t:t + 10000] = torch.randn(1, 10000, H, 256, generator=g, device=dev).to(dt)
    kv = kv.transpose(1, 2)
    kr = torch.randn(1, T, 64, generator=g, device=dev).to(dt)
    q = torch.randn(1, Sq, H, 192, generator=g, device=dev).to(dt).transpose(1, 2)
    x = (q[..., :128], q[..., 128:], kv[..., :128], kr, kv[..., 128:])
    got = ops.mla_fwd_causal(*x, 192 ** -0.5)
    for h in (0, 77, H - 1):
        part = [t if t.dim() == 3 else t[:, h:h + 1] for t in x]
        y, tol = M.fwd_causal(*part, 192 ** -0.5)
        assert M.close(got[:, :, h:h + 1], y, tol)
