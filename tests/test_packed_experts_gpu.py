"""The routed experts of a packed model as a serving loop runs them: a decode step captured into a
graph."""
import pytest
import torch

from test_packed_model_gpu import FORMATS, experts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('fmt,weight', FORMATS)
@pytest.mark.parametrize('T', [1, 16])
def test_experts_decode_step_captured(dev, fmt, weight, T):
    """Replays on new tokens and routes, with eager work between, against the eager call."""
    E, H, inter, k = 8, 512, 384, 3
    experts = experts_of(dev, fmt, weight, E, H, inter, seed=4)
    g = torch.Generator().manual_seed(T)

    def inputs():
        idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
        return (torch.randn(T, H, generator=g).to(torch.bfloat16).to(dev), idx.to(dev),
                torch.rand(T, k, generator=g).to(dev))
    sets = [inputs() for _ in range(4)]
    with torch.no_grad():
        want = [experts(*s) for s in sets]
        x = [t.clone() for t in sets[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = experts(*x)
        for i in (1, 2, 3, 0, 2):
            for t, u in zip(x, sets[i]):
                t.copy_(u)
            graph.replay()
            other = experts(*sets[(i + 1) % 4])
            torch.cuda.synchronize()
            assert torch.equal(out, want[i])
            assert torch.equal(other, want[(i + 1) % 4])


@pytest.mark.parametrize('fmt,weight', FORMATS)
def test_experts_on_streams_of_their_own(dev, fmt, weight):
    """The first call on a stream that is still busy, the next on another one; and a buffer that is
    replaced while a busy stream has a call with the old one outstanding."""
    E, H, inter, k, T = 8, 512, 384, 3, 16
    g = torch.Generator().manual_seed(9)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(dev)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(dev)
    w = torch.rand(T, k, generator=g).to(dev)
    with torch.no_grad():
        want = experts_of(dev, fmt, weight, E, H, inter, seed=4)(x, idx, w)
        experts = experts_of(dev, fmt, weight, E, H, inter, seed=4)
        busy = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(20_000_000)
            a = experts(x, idx, w)
        b = experts(x, idx, w)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)

        name = 'qweight' if fmt == 'autoawq_quant' else 'weight_packed'
        lin = experts[5].up_proj
        old = getattr(lin, name)                   # the caller keeps what the busy stream reads
        with torch.cuda.stream(busy):
            torch.cuda._sleep(20_000_000)
            a = experts(x, idx, w)
        setattr(lin, name, torch.zeros_like(old))
        b = experts(x, idx, w)
        fill = [torch.zeros(n, dtype=torch.int64, device=dev) for n in range(1, 400)]
        torch.cuda.synchronize()
        assert torch.equal(a, want) and not torch.equal(b, want)
        setattr(lin, name, old)
        assert torch.equal(experts(x, idx, w), want)
        assert len(fill) == 399


@pytest.mark.parametrize('fmt,weight', FORMATS)
def test_experts_graph_outlives_a_replaced_buffer(dev, fmt, weight):
    """A graph captured with the old buffers (which the caller keeps) still runs on them."""
    E, H, inter, k, T = 8, 512, 384, 3, 2
    experts = experts_of(dev, fmt, weight, E, H, inter, seed=4)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(dev)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(dev)
    w = torch.rand(T, k, generator=g).to(dev)
    name = 'qweight' if fmt == 'autoawq_quant' else 'weight_packed'
    with torch.no_grad():
        want = experts(x, idx, w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = experts(x, idx, w)
        old = [getattr(e.up_proj, name) for e in experts]
        for e, t in zip(experts, old):
            setattr(e.up_proj, name, torch.zeros_like(t))
        zero = experts(x, idx, w)
        fill = [torch.zeros(n, dtype=torch.int64, device=dev) for n in range(1, 400)]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert torch.equal(experts(x, idx, w), zero) and not torch.equal(zero, want)
        assert len(fill) == 399
