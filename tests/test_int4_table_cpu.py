"""A table of packed weights knows what its addresses lead to: a product that would read them as
anything else is refused on the host, before any launch, so without a GPU."""
import copy

import pytest
import torch

from lightcompress_amd import _native as N
from lightcompress_amd import ops

K, NC, G = 256, 64, 3


def weights(layout, n=NC, k=K, group=128):
    ng = k // group
    if layout == 'vllm':
        return [(torch.zeros(n, k // 8, dtype=torch.int32),
                 torch.ones(n, ng, dtype=torch.float16)) for _ in range(G)]
    return [(torch.zeros(k, n // 8, dtype=torch.int32), torch.ones(ng, n, dtype=torch.float16),
             torch.zeros(ng, n // 8, dtype=torch.int32)) for _ in range(G)]


def product(tab, n=NC, k=K, group=128, layout='vllm', **kw):
    x, off = torch.zeros(5, k, dtype=torch.bfloat16), torch.zeros(G + 1, dtype=torch.int64)
    return ops.int4_linear_grouped(x, off, tab, n, group, layout, **kw)


@pytest.mark.parametrize('layout', ['vllm', 'autoawq'])
def test_products_on_a_table_of_other_weights_are_refused(layout):
    w = weights(layout)
    tab = ops.int4_weight_table(w, 'cpu')
    two = torch.stack([tab, ops.int4_weight_table(weights(layout), 'cpu')]).contiguous()
    other = 'autoawq' if layout == 'vllm' else 'vllm'
    for t in (tab, two, ops.int4_weight_table(w, 'cpu', w)):
        for kw in (dict(n=NC + 8), dict(n=NC // 2), dict(k=2 * K), dict(k=128), dict(group=64),
                   dict(group=256), dict(layout=other)):
            with pytest.raises(ValueError, match='wtab'):
                product(t, **{'layout': layout, **kw})
        with pytest.raises(N.LcqError, match='GPU only'):      # the weights' own: past the checks
            product(t, layout=layout)


def test_bare_addresses_are_refused():
    with pytest.raises(ValueError, match='int4_weight_table'):
        product(torch.zeros(G, 3, dtype=torch.int64))


def test_tables_of_different_weights_do_not_mix():
    a, b = (ops.int4_weight_table(weights('vllm', k=k), 'cpu') for k in (K, 2 * K))
    with pytest.raises(ValueError, match='int4_weight_table'):
        product(torch.stack([a, b]))
    c = ops.int4_weight_table(weights('vllm'), 'cpu')
    c.copy_(b)                                                 # now a table of b's weights
    with pytest.raises(ValueError, match='wtab holds'):
        product(c)


def test_a_table_stays_one_where_tensors_do():
    tab = ops.int4_weight_table(weights('vllm'), 'cpu')
    for t in (tab.clone(), tab.to('cpu'), tab.contiguous(), tab.detach(), copy.deepcopy(tab),
              torch.stack([tab, tab])[1], torch.cat([tab[:1], tab[1:]]),
              torch.empty_like(tab).copy_(tab)):
        assert torch.equal(t, tab)
        with pytest.raises(N.LcqError, match='GPU only'):
            product(t)
    off = torch.zeros(G, dtype=torch.int64)                    # as many groups as row_off names
    with pytest.raises(ValueError, match='row_off'):
        ops.int4_linear_grouped(torch.zeros(5, K, dtype=torch.bfloat16), off, tab, NC, 128)


def test_what_is_computed_from_a_table_is_none():
    """New contents, a memory of the same shape, arithmetic: no addresses of those weights."""
    tab = ops.int4_weight_table(weights('vllm'), 'cpu')
    written, added = tab.clone(), tab.clone()
    written[0] = torch.zeros(3, dtype=torch.int64)
    added.add_(16)
    for t in (torch.empty_like(tab), torch.zeros_like(tab), tab + 16, tab.flip(0), written, added,
              tab.clone().zero_(), tab.clone().copy_(torch.zeros(G, 3, dtype=torch.int64))):
        with pytest.raises(ValueError, match='int4_weight_table'):
            product(t)
    with pytest.raises(N.LcqError, match='GPU only'):
        product(tab)


class Elsewhere(torch.Tensor):
    """A CPU tensor that says it is on another device."""
    device = None


def test_weights_of_two_devices_are_refused():
    """'cuda' names no device: the table goes where its weights are, which is one device."""
    def at(w, device):
        w = [tuple(t.as_subclass(Elsewhere) for t in one) for one in w]
        for one in w:
            for t in one:
                t.device = torch.device(device)
        return w
    a, b = at(weights('vllm'), 'cuda:0'), at(weights('vllm'), 'cuda:1')
    for args in ((a[:1] + b[1:], 'cuda'), (a, 'cuda', b), (a, 'cuda:1')):
        with pytest.raises(ValueError, match='cuda:'):
            ops.int4_weight_table(*args)
