"""The address tables of the packed experts: how they are made and when they are made again.
Host work, so without a GPU (the tables are on the CPU here)."""
import pytest
import torch
import torch.nn as nn

from lightcompress_amd import deepseekv3 as D
from lightcompress_amd.deepseekv3 import ExpertList
from lightcompress_amd.module_utils import VllmRealQuantLinear


def packed(n, k):
    m = VllmRealQuantLinear(torch.zeros(n, k // 8, dtype=torch.int32), None,
                            torch.ones(n, k // 128, dtype=torch.float16), None, True,
                            'weight_scale')
    m.in_features, m.out_features, m.int4_forward = k, n, True
    return m


def experts_of(E, hidden=256, inter=128):
    out = ExpertList()
    for _ in range(E):
        mlp = nn.Module()
        mlp.gate_proj, mlp.up_proj = packed(inter, hidden), packed(inter, hidden)
        mlp.down_proj = packed(hidden, inter)
        out.append(mlp)
    return out


def addresses(experts, *projections):
    return torch.tensor([[[m.weight_packed.data_ptr(), m.weight_scale.data_ptr(), 0]
                          for m in (getattr(e, p) for e in experts)] for p in projections])


def test_tables_come_to_the_device_by_copies_alone(monkeypatch):
    """A table lives longer than the call that makes it and is read on any stream: it must be
    whole when that call returns. A copy from pageable host memory is; a kernel on the stream of
    the first call, which puts tables together there, need not be."""
    def no_kernel(*a, **k):
        raise AssertionError('a table put together on the device')
    for name in ('stack', 'cat'):
        monkeypatch.setattr(torch, name, no_kernel)
    experts = experts_of(3)
    gate_up, down = experts._int4_tables(torch.device('cpu'))
    monkeypatch.undo()
    assert torch.equal(gate_up, addresses(experts, 'gate_proj', 'up_proj'))
    assert torch.equal(down, addresses(experts, 'down_proj')[0])
    assert gate_up.is_contiguous() and down.is_contiguous()


def test_tables_follow_the_buffers():
    experts = experts_of(4)
    dev = torch.device('cpu')
    first = experts._int4_tables(dev)
    assert experts._int4_tables(dev)[0] is first[0]
    experts[2].up_proj.weight_packed = experts[2].up_proj.weight_packed.clone()
    second = experts._int4_tables(dev)
    assert not torch.equal(second[0], first[0])
    assert torch.equal(second[0], addresses(experts, 'gate_proj', 'up_proj'))
    experts[1].down_proj = packed(256, 128)
    assert torch.equal(experts._int4_tables(dev)[1], addresses(experts, 'down_proj')[0])


def test_weight_table_of_two_sets():
    from lightcompress_amd import ops
    e = experts_of(2)
    gate, up = ([(m.weight_packed, m.weight_scale) for m in (getattr(x, p) for x in e)]
                for p in ('gate_proj', 'up_proj'))
    tab = ops.int4_weight_table(gate, 'cpu', up)
    assert torch.equal(tab, addresses(e, 'gate_proj', 'up_proj'))
    with pytest.raises(ValueError):
        ops.int4_weight_table(gate, 'cpu', up[:1])
    with pytest.raises(ValueError):
        ops.int4_weight_table(gate, 'cpu', [(m.weight_packed, m.weight_scale)
                                            for m in (x.down_proj for x in e)])


def test_what_a_graph_cannot_hold_is_refused(monkeypatch):
    """The tables are uploaded by a copy from pageable memory, and the sort of very many routes
    clears memory by a library call: neither belongs into a captured graph."""
    dev = torch.device('cpu')
    monkeypatch.setattr(D, '_capturing', lambda: True)
    experts = experts_of(2)
    with pytest.raises(RuntimeError, match='captur'):
        experts._int4_tables(dev)
    monkeypatch.undo()
    tables = experts._int4_tables(dev)
    monkeypatch.setattr(D, '_capturing', lambda: True)
    assert experts._int4_tables(dev) is tables
    idx = torch.zeros(40000, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='captur'):
        experts._forward_grouped_int4(torch.zeros(40000, 256, dtype=torch.bfloat16), idx,
                                      torch.ones(idx.shape))


@pytest.mark.parametrize('kind,walks', [('float', 0), ('packed', 1)])
def test_experts_are_walked_once_at_most(monkeypatch, kind, walks):
    """Whether a call can run grouped is asked on every call: the look over all experts is made for
    the kind the first one is, and not for experts that no grouped product takes."""
    experts = experts_of(3)
    if kind == 'float':
        for e in experts:
            e.gate_proj = e.up_proj = nn.Linear(256, 128, bias=False)
            e.down_proj = nn.Linear(128, 256, bias=False)
    seen = []
    monkeypatch.setattr(ExpertList, '_plain_mlps', lambda self, x: seen.append(1))
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    assert not experts._grouped_fp8_ok(x) and not experts._grouped_int4_ok(x)
    assert len(seen) == walks
