"""Lengths and positions past the buffers, and tensors that repeat one row, in latent attention."""
import pytest
import torch

from oracle import mla_ref as R
from test_mla_gpu import DTYPES, SCALE, cache, prefill_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('H,Sq,Skv,split', [(3, 140, 270, False), (2, 77, 1500, True)])
def test_prefill_lengths_past_the_keys(dev, dt, H, Sq, Skv, split):
    """kv_lens is cut at the keys there are: every row as with Skv. Queries past the last key."""
    from lightcompress_amd import _native as N, ops
    B = 5
    assert (N.load().lcq_mla_fwd_causal_workspace_bytes(B, H, Sq, Skv) > 0) == split
    x = prefill_inputs(torch.Generator().manual_seed(Skv), B, H, Sq, Skv, dt, dev)
    lens = torch.tensor([Skv, Skv + 1, Skv + 64, 1 << 30, (1 << 31) - 1], dtype=torch.int32)
    for start in (None, [Skv - Sq, Skv - Sq, Skv, 1 << 30, 40]):
        s = None if start is None else torch.tensor(start, dtype=torch.int32)
        got = ops.mla_fwd_causal(*x, SCALE, q_start=None if s is None else s.to(dev),
                                 kv_lens=lens.to(dev))
        y, tol = R.fwd_causal(*x, SCALE, q_start=s, kv_lens=lens)
        assert R.close(got, y, tol)
        full = torch.full((B,), Skv, dtype=torch.int32, device=dev)
        assert torch.equal(got, ops.mla_fwd_causal(
            *x, SCALE, q_start=None if s is None else s.to(dev), kv_lens=full))


@pytest.mark.parametrize('Skv', [200, 1500])
def test_prefill_repeated_rows(dev, Skv):
    """Keys and values that all heads share, a query that all sequences share: strides of zero."""
    from lightcompress_amd import ops
    B, H, Sq, dt = 2, 4, 33, torch.bfloat16
    qn, qr, kn, kr, v = prefill_inputs(torch.Generator().manual_seed(1), B, H, Sq, Skv, dt, dev)
    x = (qn[:1].expand(B, -1, -1, -1), qr[:1].expand(B, -1, -1, -1),
         kn[:, :1].expand(-1, H, -1, -1), kr, v[:, :1].expand(-1, H, -1, -1))
    assert R.close(ops.mla_fwd_causal(*x, SCALE), *R.fwd_causal(*x, SCALE))


def test_decode_repeated_rows(dev):
    """One sequence's pages named by several, one query for all heads."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(5)
    ckv, kr, table = cache(g, 1, [300], 16, torch.bfloat16, dev)
    table = table.expand(4, -1).contiguous()
    lens = torch.tensor([300, 1, 17, 299], dtype=torch.int32, device=dev)
    ql = torch.randn(4, 1, 1, 512, generator=g).bfloat16().to(dev).expand(-1, 2, 20, -1)
    qr = torch.randn(4, 1, 1, 64, generator=g).bfloat16().to(dev).expand(-1, 2, 20, -1)
    got = ops.mla_decode(ql, qr, ckv, kr, table, lens, SCALE)
    assert R.close(got, *R.decode(ql, qr, ckv, kr, table, lens, SCALE))
