"""Latent attention (lcq_mla_fwd_causal, lcq_mla_decode) against the 64-bit oracle: types, head
counts, lengths from one token up, strides, padded batches, pages, rows that see nothing."""
import pytest
import torch

from oracle import mla_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
SCALE = 192 ** -0.5


def prefill_inputs(g, B, H, Sq, Skv, dt, dev, layout='proj'):
    def t(*shape):
        return (torch.randn(*shape, generator=g) * 1.2).to(dt).to(dev)
    kr = t(B, Skv, 64)
    if layout == 'proj':      # the projections' layouts, seen head by head
        q, kv = t(B, Sq, H, 192).transpose(1, 2), t(B, Skv, H, 256).transpose(1, 2)
        return q[..., :128], q[..., 128:], kv[..., :128], kr, kv[..., 128:]
    return t(B, H, Sq, 128), t(B, H, Sq, 64), t(B, H, Skv, 128), kr, t(B, H, Skv, 128)


@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('B,H,Sq,Skv', [
    (1, 1, 1, 1), (2, 3, 1, 70), (1, 2, 33, 33), (2, 16, 64, 64), (1, 4, 129, 129),
    (3, 3, 100, 165), (1, 2, 128, 500), (1, 5, 300, 301), (1, 16, 511, 511), (2, 2, 200, 1030)])
def test_prefill(dev, dt, B, H, Sq, Skv):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(B * 100 + H * 10 + Sq + Skv)
    for layout in ('proj', 'heads'):
        x = prefill_inputs(g, B, H, Sq, Skv, dt, dev, layout)
        got = ops.mla_fwd_causal(*x, SCALE)
        assert got.shape == (B, Sq, H, 128) and got.dtype == dt and got.is_contiguous()
        y, tol = R.fwd_causal(*x, SCALE)
        assert R.close(got, y, tol)
        assert torch.equal(got, ops.mla_fwd_causal(x[0], x[1], x[2], x[3][:, None], x[4], SCALE))


@pytest.mark.parametrize('dt', DTYPES)
def test_prefill_padded_and_empty_rows(dev, dt):
    """Right-padded batches, chunks behind cached tokens, an empty sequence, queries in front of
    the first key; what lies behind a length may be anything."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(21)
    B, H, Sq, Skv = 6, 3, 140, 270
    x = prefill_inputs(g, B, H, Sq, Skv, dt, dev)
    lens = torch.tensor([270, 0, 1, 64, 199, 65], dtype=torch.int32)
    start = torch.tensor([130, 5, 0, -10, 59, 200], dtype=torch.int32)
    for b in range(B):
        x[2][b, :, int(lens[b]):] = float('nan')
        x[3][b, int(lens[b]):] = float('inf')
        x[4][b, :, int(lens[b]):] = float('nan')
    got = ops.mla_fwd_causal(*x, SCALE, q_start=start.to(dev), kv_lens=lens.to(dev))
    y, tol = R.fwd_causal(*x, SCALE, q_start=start, kv_lens=lens)
    assert R.close(got, y, tol)
    assert (got[1] == 0).all() and (got[3, :10] == 0).all()
    wild = torch.tensor([1 << 30, -(1 << 30), 0, 64, 199, 65], dtype=torch.int32)
    got = ops.mla_fwd_causal(*x, SCALE, q_start=start.to(dev), kv_lens=wild.to(dev)[[1, 1, 1, 3, 4, 5]])
    assert (got[:3] == 0).all()


@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('B,H,Sq,Skv', [
    (1, 1, 1, 1024), (1, 2, 77, 1500), (2, 3, 130, 2049), (1, 16, 200, 1100), (3, 1, 5, 4000)])
def test_prefill_keys_split(dev, dt, B, H, Sq, Skv):
    """Few query tiles against many keys: the keys are shared out and joined. Lengths and positions
    that leave shares, rows and sequences empty; the same call gives the same bits."""
    from lightcompress_amd import _native as N, ops
    assert N.load().lcq_mla_fwd_causal_workspace_bytes(B, H, Sq, Skv) > 0
    g = torch.Generator().manual_seed(B * 100 + H * 10 + Sq + Skv)
    x = prefill_inputs(g, B, H, Sq, Skv, dt, dev)
    got = ops.mla_fwd_causal(*x, SCALE)
    y, tol = R.fwd_causal(*x, SCALE)
    assert R.close(got, y, tol)
    assert torch.equal(got, ops.mla_fwd_causal(*x, SCALE))
    for lens, start in (([Skv] * 3, [3, Skv, -2]), ([65, Skv - 1, 0], [70, 600, 9]),
                        ([0, 0, 1], [0, 0, 0])):
        lens, start = (torch.tensor(t[:B], dtype=torch.int32) for t in (lens, start))
        z = [t.clone() for t in x]
        for b in range(B):
            z[2][b, :, int(lens[b]):] = float('nan')
            z[3][b, int(lens[b]):] = float('inf')
            z[4][b, :, int(lens[b]):] = float('nan')
        got = ops.mla_fwd_causal(*z, SCALE, q_start=start.to(dev), kv_lens=lens.to(dev))
        y, tol = R.fwd_causal(*z, SCALE, q_start=start, kv_lens=lens)
        assert R.close(got, y, tol)


def test_prefill_scores_of_any_size(dev):
    """Scores far from zero (a row's softmax is nearly one key), equal scores, huge scale."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(4)
    x = list(prefill_inputs(g, 1, 2, 96, 96, torch.bfloat16, dev))
    for f, scale in ((30., SCALE), (0., SCALE), (1., 50.)):
        z = [x[0] * f, x[1] * f, *x[2:]]
        got = ops.mla_fwd_causal(*z, scale)
        y, tol = R.fwd_causal(*z, scale)
        assert R.close(got, y, tol)
    z = [x[0].clone(), *x[1:]]
    z[0][0, 1, 40] = float('nan')
    got = ops.mla_fwd_causal(*z, SCALE)
    assert got[0, 40, 1].isnan().all() and got.isnan().sum() == 128


def cache(g, B, lens, ps, dt, dev, P=None, joint=True, nb=None):
    used = [-(-n // ps) for n in lens]
    P = P or max(1, sum(used) + 2)
    nb = nb or max(1, max(used))
    c = (torch.randn(P, ps, 576, generator=g) * 1.1).to(dt).to(dev)
    table = torch.zeros(B, nb, dtype=torch.int32)
    perm = torch.randperm(P, generator=g)
    at = 0
    for b in range(B):
        table[b, :used[b]] = perm[at:at + used[b]]
        at += used[b]
    ckv, kr = c[..., :512], c[..., 512:]
    if not joint:
        ckv, kr = ckv.contiguous(), kr.contiguous()
    return ckv, kr, table.to(dev)


@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('lens,H,Sq,ps', [
    ([1], 1, 1, 16), ([33], 16, 1, 64), ([5, 64, 1], 16, 1, 16), ([200, 31], 16, 2, 1),
    ([97, 640, 13, 300], 128, 1, 64), ([129, 500], 40, 2, 48), ([700], 64, 3, 100),
    ([2500, 40], 16, 1, 64), ([4200], 24, 1, 1), ([1100], 128, 2, 256), ([300] * 9, 33, 1, 32)])
def test_decode(dev, dt, lens, H, Sq, ps):
    from lightcompress_amd import ops
    B = len(lens)
    g = torch.Generator().manual_seed(sum(lens) + H + Sq + ps)
    ckv, kr, table = cache(g, B, lens, ps, dt, dev)
    ql = torch.randn(B, Sq, H, 512, generator=g).to(dt).to(dev)
    qr = torch.randn(B, Sq, H, 64, generator=g).to(dt).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE)
    assert got.shape == (B, Sq, H, 512) and got.dtype == dt and got.is_contiguous()
    y, tol = R.decode(ql, qr, ckv, kr, table, n, SCALE)
    assert R.close(got, y, tol)
    assert torch.equal(got, ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE))


def test_decode_strides(dev):
    """Queries seen through a head-major product, the two cache parts apart, a wide table."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(2)
    lens, H, Sq, dt = [90, 17], 24, 2, torch.bfloat16
    ckv, kr, table = cache(g, 2, lens, 16, dt, dev, joint=False, nb=300)
    ql = torch.randn(H, 2 * Sq, 512, generator=g).to(dt).to(dev)
    ql = ql.view(H, 2, Sq, 512).permute(1, 2, 0, 3)
    qr = torch.randn(2, Sq, H, 192, generator=g).to(dt).to(dev)[..., 128:]
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    assert R.close(ops.mla_decode(ql, qr, ckv, kr, table, n, 0.05),
                   *R.decode(ql, qr, ckv, kr, table, n, 0.05))


def test_decode_empty_rows_bad_pages_and_foreign_data(dev):
    """A length of zero or below the token count leaves rows without a key; page numbers outside
    the pool hide their keys; what the pages hold behind a length may be anything; lengths past
    the table are cut."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(6)
    lens, H, Sq, ps, dt = [0, 1, 100, 61, 200], 16, 3, 16, torch.float16
    ckv, kr, table = cache(g, 5, lens, ps, dt, dev, joint=False)
    for b, v in enumerate(lens):
        if v % ps:
            page = int(table[b, v // ps])
            ckv[page, v % ps:] = float('nan')
            kr[page, v % ps:] = float('inf')
    table[2, 1], table[2, 3] = -1, ckv.shape[0]
    table[3] = torch.tensor([-7] * table.shape[1])
    n = torch.tensor([0, 1, 100, 61, 1 << 30], dtype=torch.int32, device=dev)
    n[4] = -3
    ql = torch.randn(5, Sq, H, 512, generator=g).to(dt).to(dev)
    qr = torch.randn(5, Sq, H, 64, generator=g).to(dt).to(dev)
    got = ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE)
    y, tol = R.decode(ql, qr, ckv, kr, table, n, SCALE)
    assert R.close(got, y, tol)
    for b in (0, 3, 4):
        assert (got[b] == 0).all()
    assert (got[1, :2] == 0).all() and (got[1, 2] != 0).any()
    n[4] = 1 << 30                       # the table's 13 pages, 208 keys
    got = ops.mla_decode(ql, qr, ckv.nan_to_num(0), kr.nan_to_num(0, 0, 0), table, n, SCALE)
    assert R.close(got, *R.decode(ql, qr, ckv.nan_to_num(0), kr.nan_to_num(0, 0, 0), table, n, SCALE))


def test_decode_cache_past_32_bits(dev):
    """Pages more than 4 GB apart."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(9)
    ps, dt = 64, torch.bfloat16
    pool = torch.empty(70000, ps, 576, dtype=dt, device=dev)     # 5.2 GB
    lens = [200, 70]
    table = torch.tensor([[69999, 3, 60001, 12], [2, 65000, 0, 0]], dtype=torch.int32, device=dev)
    for p in (69999, 3, 60001, 12, 2, 65000):
        pool[p] = torch.randn(ps, 576, generator=g).to(dt).to(dev)
    ql = torch.randn(2, 1, 16, 512, generator=g).to(dt).to(dev)
    qr = torch.randn(2, 1, 16, 64, generator=g).to(dt).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = ops.mla_decode(ql, qr, pool[..., :512], pool[..., 512:], table, n, SCALE)
    pages, small = torch.unique(table.cpu().long(), return_inverse=True)
    sub = pool[pages.to(dev)]
    assert R.close(got, *R.decode(ql, qr, sub[..., :512], sub[..., 512:], small, n, SCALE))


def test_other_stream_and_graph(dev):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(12)
    dt, H = torch.bfloat16, 16
    lens = [900, 333]
    ckv, kr, table = cache(g, 2, lens, 64, dt, dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    ql = torch.randn(2, 1, H, 512, generator=g).to(dt).to(dev)
    qr = torch.randn(2, 1, H, 64, generator=g).to(dt).to(dev)
    x = prefill_inputs(g, 1, 4, 150, 150, dt, dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, b = ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE), ops.mla_fwd_causal(*x, SCALE)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE))
    assert torch.equal(b, ops.mla_fwd_causal(*x, SCALE))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE), ops.mla_fwd_causal(*x, SCALE)
    for i in range(3):
        ql.copy_(torch.randn(ql.shape, generator=g).to(dt))
        n.copy_(torch.tensor([900 - 301 * i, 333]))
        x[0].copy_(torch.randn(x[0].shape, generator=g).to(dt))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.mla_decode(ql, qr, ckv, kr, table, n, SCALE))
        assert torch.equal(b, ops.mla_fwd_causal(*x, SCALE))


@pytest.mark.parametrize('B,H,n', [(1, 16, 40), (1, 16, 700), (1, 20, 4500), (9, 128, 900)])
def test_decode_nan_row(dev, B, H, n):
    """A NaN query gives NaN outputs, for its row alone, however many workgroups share the keys."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(n)
    ps = 16
    nb = -(-n // ps)
    ckv = torch.randn(B * nb, ps, 512, generator=g).bfloat16().to(dev)
    kr = torch.randn(B * nb, ps, 64, generator=g).bfloat16().to(dev)
    table = torch.arange(B * nb, dtype=torch.int32).view(B, nb).to(dev)
    lens = torch.full((B,), n, dtype=torch.int32).to(dev)
    ql = torch.randn(B, 1, H, 512, generator=g).bfloat16().to(dev)
    qr = torch.randn(B, 1, H, 64, generator=g).bfloat16().to(dev)
    want = ops.mla_decode(ql, qr, ckv, kr, table, lens, SCALE)
    assert not want.isnan().any()
    ql[B - 1, 0, 3, 100] = float('nan')
    got = ops.mla_decode(ql, qr, ckv, kr, table, lens, SCALE)
    assert got[B - 1, 0, 3].isnan().all() and got.isnan().sum() == 512
    got[B - 1, 0, 3] = want[B - 1, 0, 3]
    assert torch.equal(got, want)


def paged(g, B, lens, H, Sq, ps, dt, dev, spare=3):
    """A cache whose pages are dealt out in a random order, tables wider than any length."""
    nb = max(-(-max(lens) // ps), 1) + spare
    P = B * nb + 5
    ckv = torch.randn(P, ps, 512, generator=g).to(dt).to(dev)
    kr = torch.randn(P, ps, 64, generator=g).to(dt).to(dev)
    table = torch.randperm(P, generator=g)[:B * nb].to(torch.int32).view(B, nb).to(dev)
    ql = torch.randn(B, Sq, H, 512, generator=g).to(dt).to(dev)
    qr = torch.randn(B, Sq, H, 64, generator=g).to(dt).to(dev)
    return ql, qr, ckv, kr, table, torch.tensor(lens, dtype=torch.int32).to(dev)


@pytest.mark.parametrize('lens,H,Sq,spare', [
    ([(7 * i) % 90 for i in range(70)], 16, 1, 0),            # more sequences than a wave's lanes
    ([0] * 66 + [300, 0, 1], 5, 3, 2), ([33, 64], 128, 3, 900),   # a table far wider than lengths
    ([1700] * 3 + [0, 2100], 16, 1, 0), ([1], 1, 1, 0)])
def test_decode_many_sequences_wide_tables(dev, lens, H, Sq, spare):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(len(lens) + H)
    x = paged(g, len(lens), lens, H, Sq, 16, torch.bfloat16, dev, spare)
    got = ops.mla_decode(*x, SCALE)
    y, tol = R.decode(*x, SCALE)
    assert R.close(got, y, tol)
    assert torch.equal(got, ops.mla_decode(*x, SCALE))


def test_nothing_to_do(dev):
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(2)
    x = prefill_inputs(g, 2, 3, 5, 9, torch.bfloat16, dev)
    assert ops.mla_fwd_causal(*[t[:0] for t in x], SCALE).shape == (0, 5, 3, 128)
    assert ops.mla_fwd_causal(x[0][:, :, :0], x[1][:, :, :0], *x[2:], SCALE).shape == (2, 0, 3, 128)
    z = paged(g, 2, [5, 9], 4, 1, 16, torch.bfloat16, dev)
    out = ops.mla_decode(z[0][:0], z[1][:0], z[2], z[3], z[4][:0], z[5][:0], SCALE)
    assert out.shape == (0, 1, 4, 512)


def test_streams_at_once_and_graphs_with_workspaces(dev):
    """Split prefill and decode on two streams at once; two graphs of them replayed in turn on new
    inputs, with eager work between: each has its own partial outputs."""
    from lightcompress_amd import ops
    g = torch.Generator().manual_seed(12)
    f = [list(prefill_inputs(g, 1, 4, 60, 1500, torch.bfloat16, dev)) for _ in range(3)]
    d = [paged(torch.Generator().manual_seed(5), 2, [900, 1300], 16, 1, 16, torch.bfloat16, dev)
         for _ in range(3)]
    for i in range(3):
        d[i][0].normal_()
    want = [(ops.mla_fwd_causal(*f[i], SCALE), ops.mla_decode(*d[i], SCALE)) for i in range(3)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for i in range(3):
        with torch.cuda.stream(s1):
            a = ops.mla_fwd_causal(*f[i], SCALE)
        with torch.cuda.stream(s2):
            b = ops.mla_decode(*d[i], SCALE)
        outs.append((a, b))
    torch.cuda.synchronize()
    for (a, b), (x, y) in zip(outs, want):
        assert torch.equal(a, x) and torch.equal(b, y)
    fi, di = [t.clone() for t in f[0]], [t.clone() for t in d[0]]
    graphs, res = [], []
    for fn, arg in ((ops.mla_fwd_causal, fi), (ops.mla_decode, di)):
        fn(*arg, SCALE)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append(fn(*arg, SCALE))
        graphs.append(gr)
    for i in (1, 2, 0, 1):
        for t, u in zip(fi, f[i]):
            t.copy_(u)
        for t, u in zip(di, d[i]):
            t.copy_(u)
        graphs[0].replay()
        ops.mla_decode(*d[(i + 1) % 3], SCALE)
        graphs[1].replay()
        ops.mla_fwd_causal(*f[(i + 1) % 3], SCALE)
        torch.cuda.synchronize()
        assert torch.equal(res[0], want[i][0]) and torch.equal(res[1], want[i][1])
