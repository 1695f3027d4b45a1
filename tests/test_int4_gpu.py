"""Products with 4-bit packed weights (lcq_int4_gemm, lcq_int4_gemm_grouped) against the 64-bit
oracle: both deploy layouts, group sizes, row counts from one up, ragged groups, strides."""
import pytest
import torch

from oracle import int4_ref as R

pytestmark = pytest.mark.gpu

LAYOUTS = ['vllm', 'autoawq']
DTYPES = [torch.bfloat16, torch.float16]


def weight(g, layout, n, k, group, dev):
    """Random words (every code occurs), fp16 scales, zero points 0..15 in the AutoAWQ layout."""
    ng = k // group

    def words(*shape):
        return torch.randint(-2**31, 2**31, shape, generator=g, dtype=torch.int64).to(
            torch.int32).to(dev)

    def sc(*shape):
        return (torch.rand(*shape, generator=g) * 0.02 + 0.002).to(torch.float16).to(dev)
    if layout == 'vllm':
        return words(n, k // 8), sc(n, ng), None
    return words(k, n // 8), sc(ng, n), words(ng, n // 8)


def check_linear(dev, layout, dt, m, n, k, group):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(m * 7919 + n * 31 + k + group)
    w = weight(g, layout, n, k, group, dev)
    x = acts(g, m, k, dt=dt, dev=dev)
    got = ops.int4_linear(x, *w)
    assert got.shape == (m, n) and got.dtype == dt
    y, tol = R.linear(x, *w)
    assert R.close(got, y, tol)
    assert torch.equal(got, ops.int4_linear(x, *w))       # the same call, the same bits


@pytest.mark.parametrize('layout', ['vllm', 'autoawq'])
@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('m', [17, 32, 33, 47, 49, 64])
@pytest.mark.parametrize('n,k,group', [
    (72, 3200, 128),      # k split 4 ways, the waves' shares of units uneven or empty
    (264, 9312, 96),      # a last unit that is cut, 32-wide groups of a scale
    (1288, 2112, 64), (16392, 640, 128)])
def test_linear_some_rows(dev, layout, dt, m, n, k, group):
    """17 to 64 rows: two to four row tiles, k split over workgroups where n is small."""
    check_linear(dev, layout, dt, m, n, k, group)


def acts(g, *shape, dt, dev):
    x = torch.randn(*shape, generator=g)
    x[..., :: 37] *= 12          # outlier channels
    return x.to(dt).to(dev)


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('m,n,k,group', [
    (1, 256, 512, 128), (1, 8, 32, 32), (2, 40, 96, 96), (3, 72, 320, 32), (5, 264, 384, 64),
    (16, 128, 1024, 128), (17, 136, 1024, 1024), (31, 520, 4096, 128), (33, 64, 1056, 1056),
    (48, 1024, 256, 256), (64, 256, 640, 64), (65, 392, 2048, 128), (129, 640, 1152, 128),
    (200, 328, 512, 32), (257, 512, 768, 128), (511, 200, 512, 512), (1, 4096, 4096, 128),
    (4, 2048, 7168, 128), (300, 1288, 2048, 64),
    # a long k split over workgroups; the 128-row kernel: partial row and column tiles, every
    # group kind, a last unit of 128 k that is cut, n whose AutoAWQ rows are not 16-byte aligned
    (1, 64, 16384, 128), (7, 264, 12288, 64), (300, 8224, 384, 128), (129, 12320, 256, 256),
    (1300, 2592, 352, 32), (700, 4160, 448, 64), (513, 4968, 256, 128), (900, 3360, 96, 96)])
def test_linear(dev, layout, dt, m, n, k, group):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(m * 7919 + n * 31 + k + group)
    w = weight(g, layout, n, k, group, dev)
    x = acts(g, m, k, dt=dt, dev=dev)
    got = ops.int4_linear(x, *w)
    assert got.shape == (m, n) and got.dtype == dt
    y, tol = R.linear(x, *w)
    assert R.close(got, y, tol)
    assert torch.equal(got, ops.int4_linear(x, *w))       # the same call, the same bits


@pytest.mark.parametrize('m', [1, 16, 70, 300])
def test_linear_odd_columns_vllm(dev, m):
    """n of the vLLM layout is any number."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(m)
    for n in (1, 15, 33, 131, 257) + ((8201,) if m == 300 else ()):
        w = weight(g, 'vllm', n, 256, 64, dev)
        x = acts(g, m, 256, dt=torch.bfloat16, dev=dev)
        y, tol = R.linear(x, *w)
        assert R.close(ops.int4_linear(x, *w), y, tol), n


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('m,n', [(3, 264), (150, 264), (150, 6240)])
def test_linear_shapes_strides_bias(dev, layout, m, n):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(5)
    k = 512
    w = weight(g, layout, n, k, 128, dev)
    b = torch.randn(n, generator=g).to(torch.bfloat16).to(dev)
    big = acts(g, m, 2, k + 24, dt=torch.bfloat16, dev=dev)
    for x in (big[..., 8:k + 8],          # 3-D, row stride k + 24
              big[..., 3:k + 3],          # rows not 16-byte aligned
              big[:, 0, :k], big[:, 1, :k].unsqueeze(1),
              big[..., :k].transpose(0, 1)):
        got = ops.int4_linear(x, *w, bias=b)
        assert got.shape == (*x.shape[:-1], n)
        y, tol = R.linear(x.reshape(-1, k), *w, bias=b)
        assert R.close(got.reshape(-1, n), y, tol)
    assert ops.int4_linear(big[:0, 0, :k], *w).shape == (0, n)


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('m,n', [(4, 256), (140, 256), (140, 12288)])
def test_linear_nan_and_inf_stay_in_their_row(dev, layout, m, n):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(8)
    w = weight(g, layout, n, 512, 64, dev)
    x = acts(g, m, 512, dt=torch.float16, dev=dev)
    x[1, 100], x[3, 511] = float('nan'), float('inf')
    got = ops.int4_linear(x, *w)
    assert got[[1, 3]].isnan().all()
    keep = [i for i in range(m) if i not in (1, 3)]
    y, tol = R.linear(x[keep], *w)
    assert R.close(got[keep], y, tol)


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('counts,n,k,group', [
    ([1], 128, 256, 128), ([0, 3, 0, 1, 0], 264, 512, 32), ([16, 17, 15, 0, 64], 136, 384, 128),
    ([0] * 70 + [5] + [0] * 90 + [33, 1], 128, 256, 64), ([300, 1, 129, 0, 40], 520, 1024, 128),
    ([2] * 40, 72, 160, 160), ([130, 0, 257], 288, 192, 64), ([64, 200], 104, 256, 128),
    ([500], 416, 224, 32)])
def test_grouped(dev, layout, dt, counts, n, k, group):
    """One and two weight sets, the SiLU product, gathered and sorted rows."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(sum(counts) + n)
    rows, E = sum(counts), len(counts)
    off = torch.tensor([0] + counts).cumsum(0)
    ws = [[weight(g, layout, n, k, group, dev) for _ in range(E)] for _ in range(2)]
    tabs = [ops.int4_weight_table(w, dev) for w in ws]
    both = torch.stack(tabs).contiguous()
    x = acts(g, rows, k, dt=dt, dev=dev)
    pick = torch.randint(0, rows, (rows,), generator=g)
    for src in (None, pick):
        xs = x if src is None else x[src.to(dev)]
        kw = dict(layout=layout, a_rows=None if src is None else src.to(dev))
        one = ops.int4_linear_grouped(x, off.to(dev), tabs[0], n, group, **kw)
        two = ops.int4_linear_grouped(x, off.to(dev), both, n, group, **kw)
        h = ops.int4_linear_grouped(x, off.to(dev), both, n, group, silu_mul=True, **kw)
        assert one.shape == (rows, n) and two.shape == (2, rows, n) and h.shape == (rows, n)
        for e in range(E):
            s = slice(int(off[e]), int(off[e + 1]))
            if s.start == s.stop:
                continue
            gu = [R.linear(xs[s], *w[e]) for w in ws]
            assert R.close(one[s], *gu[0])
            assert R.close(two[0, s], *gu[0]) and R.close(two[1, s], *gu[1])
            assert R.close(h[s], *R.silu_mul(*gu))


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('counts,n,k,group', [
    ([13, 0, 40, 7, 3], 72, 1152, 128),       # a mean of 13 rows: two row tiles
    ([1, 70, 33, 20], 264, 416, 32), ([48, 49, 1, 17, 50], 520, 640, 64), ([38] * 6, 40, 96, 96),
    ([47] * 3 + [0], 1032, 2176, 128)])
def test_grouped_some_rows(dev, layout, counts, n, k, group):
    """Groups of a few row tiles each."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(sum(counts) + n)
    rows, E = sum(counts), len(counts)
    off = torch.tensor([0] + counts).cumsum(0)
    ws = [[weight(g, layout, n, k, group, dev) for _ in range(E)] for _ in range(2)]
    both = torch.stack([ops.int4_weight_table(w, dev) for w in ws]).contiguous()
    x = acts(g, rows, k, dt=torch.bfloat16, dev=dev)
    two = ops.int4_linear_grouped(x, off.to(dev), both, n, group, layout=layout)
    h = ops.int4_linear_grouped(x, off.to(dev), both, n, group, layout=layout, silu_mul=True)
    for e in range(E):
        s = slice(int(off[e]), int(off[e + 1]))
        if s.start == s.stop:
            continue
        gu = [R.linear(x[s], *w[e]) for w in ws]
        assert R.close(two[0, s], *gu[0]) and R.close(two[1, s], *gu[1])
        assert R.close(h[s], *R.silu_mul(*gu))


@pytest.mark.parametrize('rows', [40, 300])
def test_grouped_rows_outside_groups_and_bad_gather(dev, rows):
    """Rows behind the last group stay as they were; a gather index out of range reads zeros;
    offsets outside the rows are clamped."""
    from lightcompress_amd import _native as N
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(3)
    n, k = 128, 256
    ws = [weight(g, 'vllm', n, k, 128, dev) for _ in range(3)]
    tab = ops.int4_weight_table(ws, dev)
    x = acts(g, rows, k, dt=torch.bfloat16, dev=dev)
    a_rows = torch.arange(rows, device=dev)
    a_rows[4], a_rows[21] = -1, rows
    off = torch.tensor([2, 10, 10, 30], device=dev)

    def go(off):
        y = torch.full((rows, n), 7., dtype=torch.bfloat16, device=dev)
        N.call('lcq_int4_gemm_grouped', N.ptr(x), N.BF16, k, rows, N.ptr(a_rows), rows,
               N.ptr(off), N.ptr(tab), 3, 1, 0, 0, 128, n, k, N.ptr(y), N.stream_of(x))
        return y
    y = go(off)
    assert (y[:2] == 7).all() and (y[30:] == 7).all()
    assert (y[4] == 0).all() and (y[21] == 0).all()
    for e, (a, b) in ((0, (2, 10)), (2, (10, 30))):
        keep = [i for i in range(a, b) if i not in (4, 21)]
        assert R.close(y[keep], *R.linear(x[keep], *ws[e]))
    z = go(torch.tensor([-5, 10, 1 << 40, 3], device=dev))
    assert R.close(z[10:21], *R.linear(x[10:21], *ws[1]))


def test_other_stream_and_graph(dev):
    """On a side stream, and captured into a graph that is replayed on new inputs."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(4)
    for m, n in ((2, 256), (90, 256), (200, 12288)):
        w = weight(g, 'autoawq', n, 1024, 128, dev)
        x = acts(g, m, 1024, dt=torch.bfloat16, dev=dev)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            a = ops.int4_linear(x, *w)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(a, ops.int4_linear(x, *w))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.int4_linear(x, *w)
        for _ in range(3):
            x.copy_(acts(g, m, 1024, dt=torch.bfloat16, dev=dev))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.int4_linear(x, *w))


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('m,n,k,group', [
    (65, 136, 4096, 128), (130, 1000, 3200, 64), (257, 72, 2080, 32), (600, 40, 1536, 128)])
def test_linear_more_rows_split(dev, layout, m, n, k, group):
    """More than 64 rows of few columns: several row tiles, k split over workgroups."""
    from lightcompress_amd import _native as N
    assert N.load().lcq_int4_gemm_workspace_bytes(m, n, k, LAYOUTS.index(layout)) > 0
    check_linear(dev, layout, torch.bfloat16, m, n, k, group)


def test_streams_at_once_and_graphs_with_workspaces(dev):
    """Products whose k is split, on two streams at once and in two graphs replayed in turn: each
    has its own partial sums."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(31)
    cases = []
    for m, n, k in ((37, 200, 4096), (2, 136, 9216)):
        w = weight(g, 'autoawq', n, k, 128, dev)
        xs = [acts(g, m, k, dt=torch.bfloat16, dev=dev) for _ in range(3)]
        cases.append((w, xs, [ops.int4_linear(x, *w) for x in xs]))
        y, tol = R.linear(xs[0], *w)
        assert R.close(cases[-1][2][0], y, tol)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(3):
        for s, (w, xs, _) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(ops.int4_linear(xs[i], *w))
    torch.cuda.synchronize()
    for j, y in enumerate(got):
        assert torch.equal(y, cases[j % 2][2][j // 2])
    graphs = []
    for w, xs, _ in cases:
        xi = xs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = ops.int4_linear(xi, *w)
        graphs.append((gr, xi, y))
    for i in (1, 2, 0, 1):
        for (gr, xi, _), (w, xs, _) in zip(graphs, cases):
            xi.copy_(xs[i])
            gr.replay()
            ops.int4_linear(xs[(i + 1) % 3], *w)
        torch.cuda.synchronize()
        for (_, _, y), (_, _, want) in zip(graphs, cases):
            assert torch.equal(y, want[i])


@pytest.mark.parametrize('layout', LAYOUTS)
def test_nothing_to_do(dev, layout):
    from lightcompress_amd import ops
    w = weight(torch.Generator().manual_seed(1), layout, 64, 256, 64, dev)
    x = torch.zeros(0, 256, dtype=torch.bfloat16, device=dev)
    assert ops.int4_linear(x, *w).shape == (0, 64)
    assert ops.int4_linear(x.view(2, 0, 256), *w).shape == (2, 0, 64)
    tab = ops.int4_weight_table([w], dev)
    off = torch.zeros(2, dtype=torch.int64, device=dev)
    assert ops.int4_linear_grouped(x, off, tab, 64, 64, layout=layout).shape == (0, 64)


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('m', [20, 100])
def test_linear_split_bias_and_strided_rows(dev, layout, m):
    """A split k with a bias (added once), rows of x inside a wider tensor, leading batch dims."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(m)
    n, k = 72, 3200
    w = weight(g, layout, n, k, 128, dev)
    wide = acts(g, m, k + 64, dt=torch.float16, dev=dev)
    x = wide[:, 32:32 + k]
    b = (torch.randn(n, generator=g) * 3).half().to(dev)
    y, tol = R.linear(x, *w, bias=b)
    got = ops.int4_linear(x, *w, bias=b)
    assert R.close(got, y, tol)
    assert torch.equal(got, ops.int4_linear(x.reshape(2, m // 2, k), *w, bias=b).view(m, n))
