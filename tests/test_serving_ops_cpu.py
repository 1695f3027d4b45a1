"""Refusals of the packed-product and latent-attention entry points: checked on the host, before
any launch, so without a GPU."""
import ctypes

import pytest
import torch

from lightcompress_amd import _native as N
from lightcompress_amd import ops


@pytest.fixture(scope='module')
def lib():
    if not N.lib_path().exists():
        import __graft_entry__
        __graft_entry__.build()
    return N.load()


P = 1 << 20   # an address that is never touched


def gemm(lib, dtype=N.BF16, ldx=256, m=4, k=256, x=P, qw=P, sc=P, qz=None, layout=0, group=128,
         n=64, y=P, ldy=64, ws=None, wsb=0):
    rc = lib.lcq_int4_gemm(x, dtype, ldx, m, k, qw, sc, qz, layout, group, n, None, y, ldy, ws, wsb,
                           None)
    return rc, lib.lcq_last_error().decode()


@pytest.mark.parametrize('kw,msg', [
    (dict(dtype=N.F32), 'activations'), (dict(k=264, ldx=264), 'multiple of 32'),
    (dict(group=48), 'group'), (dict(group=96), 'group'), (dict(group=0), 'group'),
    (dict(layout=2), 'layout'), (dict(layout=1, qz=P, n=60), 'multiple of 8'),
    (dict(layout=1), 'qzeros'), (dict(qz=P), 'qzeros'), (dict(x=P + 2), 'aligned'),
    (dict(qw=P + 4), 'aligned'), (dict(sc=P + 2), 'aligned'), (dict(ldx=252), 'stride'),
    (dict(ldx=248), 'stride'), (dict(ldy=63), 'stride'), (dict(x=None), 'null'),
    (dict(m=-1), 'shape'), (dict(n=0), 'shape'), (dict(m=1 << 33), 'large'),
    (dict(n=1 << 26), 'large'), (dict(k=1 << 21, ldx=1 << 21), 'large'),
    (dict(m=1, k=1 << 20, ldx=1 << 20), 'workspace')])
def test_int4_gemm_refuses(lib, kw, msg):
    rc, err = gemm(lib, **kw)
    assert rc == -1 and msg in err, err


def test_int4_gemm_nothing_to_do(lib):
    assert gemm(lib, m=0)[0] == 0


def grouped(lib, rows=4, x_rows=4, a_rows=None, G=2, nsets=1, silu=0, layout=0, group=128, n=64,
            k=256, off=P, tab=P, x=P, y=P):
    rc = lib.lcq_int4_gemm_grouped(x, N.BF16, 256, x_rows, a_rows, rows, off, tab, G, nsets, silu,
                                   layout, group, n, k, y, None)
    return rc, lib.lcq_last_error().decode()


@pytest.mark.parametrize('kw,msg', [
    (dict(G=0), 'group count'), (dict(nsets=3), 'weight sets'), (dict(silu=1), 'silu_mul'),
    (dict(off=None), 'null'), (dict(tab=None), 'null'), (dict(x_rows=3), 'fewer rows'),
    (dict(x=P + 8), 'aligned'), (dict(layout=1, n=63), 'multiple of 8'), (dict(k=512), 'aligned')])
def test_int4_grouped_refuses(lib, kw, msg):
    rc, err = grouped(lib, **kw)
    assert rc == -1 and msg in err, err
    assert grouped(lib, rows=0)[0] == 0


def strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


def fwd(lib, dtype=N.BF16, B=1, H=2, Sq=8, Skv=8, scale=0.1, qn=P, kn_s=(4096, 256, 512),
        q_start=None, kr_s=(512, 64), out=P, ws=P, wsb=None):
    need = lib.lcq_mla_fwd_causal_workspace_bytes(B, H, Sq, Skv)
    q, kr = strides(4096, 192, 384), strides(*kr_s)
    rc = lib.lcq_mla_fwd_causal(qn, q, P, q, P, strides(*kn_s), P, kr, P, strides(4096, 256, 512),
                                dtype, B, H, Sq, Skv, q_start, None, scale, out, ws,
                                need if wsb is None else wsb, None)
    return rc, lib.lcq_last_error().decode()


@pytest.mark.parametrize('kw,msg', [
    (dict(dtype=N.F32), 'bf16'), (dict(H=0), 'shape'), (dict(Skv=0), 'shape'),
    (dict(scale=0.), 'scale'), (dict(scale=-1.), 'scale'), (dict(scale=float('nan')), 'scale'),
    (dict(scale=float('inf')), 'scale'), (dict(qn=None), 'null'), (dict(qn=P + 4), 'aligned'),
    (dict(kn_s=(4096, 256, 516)), 'multiples of 8'), (dict(kn_s=(4096, 256, -512)), '2^24'),
    (dict(kr_s=(512, 1 << 24)), '2^24'), (dict(Sq=9), 'q_start'), (dict(B=1 << 25), 'large'),
    (dict(B=1 << 20, H=1 << 20), 'large'), (dict(Skv=4096, wsb=0), 'workspace'),
    (dict(Skv=4096, ws=None), 'workspace'), (dict(Skv=4096, ws=P + 8), 'workspace'),
    (dict(Sq=1 << 29, Skv=1 << 29), 'too long')])
def test_mla_fwd_refuses(lib, kw, msg):
    rc, err = fwd(lib, **kw)
    assert rc == -1 and msg in err, err
    assert fwd(lib, B=0)[0] == 0 and fwd(lib, Sq=0)[0] == 0


def dec(lib, dtype=N.BF16, pages=9, ps=16, nb=4, B=1, Sq=1, H=16, scale=0.1, ckv=P, table=P,
        c_s=(16 * 576, 576), ws=P, wsb=None):
    need = lib.lcq_mla_decode_workspace_bytes(B, Sq, H, nb * ps)
    q, qr, c = strides(512 * 16, 512 * 16, 512), strides(64 * 16, 64 * 16, 64), strides(*c_s)
    rc = lib.lcq_mla_decode(P, q, P, qr, ckv, c, P, c, pages, ps, table, nb, P, dtype, B, Sq, H,
                            scale, P, ws, need if wsb is None else wsb, None)
    return rc, lib.lcq_last_error().decode()


@pytest.mark.parametrize('kw,msg', [
    (dict(dtype=N.F32), 'bf16'), (dict(pages=0), 'shape'), (dict(ps=0), 'shape'),
    (dict(nb=0), 'shape'), (dict(nb=1 << 20, ps=1 << 12), 'too long'), (dict(scale=0.), 'scale'),
    (dict(H=1 << 21), 'rows'), (dict(B=70000), 'rows'), (dict(ckv=None), 'null'),
    (dict(table=None), 'null'), (dict(ckv=P + 8), 'aligned'),
    (dict(c_s=(16 * 576, 572)), 'multiples of 8'), (dict(nb=64, wsb=0), 'workspace'),
    (dict(nb=64, ws=None), 'workspace')])
def test_mla_decode_refuses(lib, kw, msg):
    rc, err = dec(lib, **kw)
    assert rc == -1 and msg in err, err
    assert dec(lib, B=0)[0] == 0 and dec(lib, Sq=0)[0] == 0


def test_python_checks():
    """Shapes, dtypes and devices are refused with a message before the library is called."""
    qw, s = torch.zeros(64, 32, dtype=torch.int32), torch.ones(64, 2, dtype=torch.float16)
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    with pytest.raises(N.LcqError):                       # no CPU path
        ops.int4_linear(x, qw, s)
    for bad, err in (((x, qw.float(), s), TypeError), ((x, qw, s.float()), TypeError),
                     ((x, qw, s[:32]), ValueError), ((x[:, :128], qw, s), ValueError),
                     ((x.float(), qw, s), TypeError), ((x, qw, s, qw), ValueError),
                     ((x, qw[:, ::2], s), TypeError),
                     ((x, qw, torch.ones(64, 16, dtype=torch.float16)), ValueError),
                     ((x, qw, s, None, torch.zeros(64)), ValueError)):
        with pytest.raises(err):
            ops.int4_linear(*bad)
    with pytest.raises(ValueError):
        ops.int4_weight_table([(qw, s), (qw[:32], s[:32])], 'cpu')
    with pytest.raises(ValueError):
        ops.int4_weight_table([], 'cpu')
    off, tab = torch.zeros(3, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int64)
    for kw in (dict(layout='gptq'), dict(silu_mul=True), dict(row_off=off[:2]),
               dict(wtab=tab[:, :2]), dict(a_rows=off.int())):
        a = dict(row_off=off, wtab=tab, n=64, group=128)
        with pytest.raises(ValueError):
            ops.int4_linear_grouped(x, **{**a, **kw})
    q = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    qr, kr = q[..., :64], torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    n32 = torch.zeros(1, dtype=torch.int32)
    for args, kw, err in (((q, qr, q, kr, q.half()), {}, TypeError),
                          ((q, qr, q, kr, q[..., :64]), {}, ValueError),
                          ((q, qr, q, kr[:, :3], q), {}, ValueError),
                          ((q, qr, q, kr, q), dict(kv_lens=n32.long()), TypeError),
                          ((q, qr, q, kr, q), dict(q_start=n32.repeat(2)), ValueError)):
        with pytest.raises(err):
            ops.mla_fwd_causal(*args, 0.1, **kw)
    with pytest.raises(N.LcqError):
        ops.mla_fwd_causal(q, qr, q, kr, q, 0.1)
    ql = torch.zeros(1, 1, 2, 512, dtype=torch.bfloat16)
    c = torch.zeros(3, 16, 576, dtype=torch.bfloat16)
    t = torch.zeros(1, 2, dtype=torch.int32)
    good = (ql, ql[..., :64], c[..., :512], c[..., 512:], t, n32)
    with pytest.raises(N.LcqError):
        ops.mla_decode(*good, 0.1)
    for i, v, err in ((1, ql[..., :32], ValueError), (2, c, ValueError), (4, t.long(), TypeError),
                      (4, t[:, :0], ValueError), (5, n32.repeat(2), ValueError),
                      (3, c[:2, :, 512:], ValueError), (0, ql.half(), TypeError)):
        with pytest.raises(err):
            ops.mla_decode(*good[:i], v, *good[i + 1:], 0.1)


def test_workspace_sizes_of_any_shape(lib):
    """Never negative, zero for shapes the products refuse."""
    for v in (-1, 0, 1, 64, 1 << 20, (1 << 31) - 1, 1 << 31, 1 << 40, (1 << 63) - 1):
        for w in (-1, 0, 1, 4096, 1 << 31, 1 << 62):
            for lay in (0, 1):
                assert lib.lcq_int4_gemm_workspace_bytes(v, w, w, lay) >= 0
                assert lib.lcq_int4_gemm_workspace_bytes(w, v, 4096, lay) >= 0
            assert lib.lcq_mla_fwd_causal_workspace_bytes(v, w, w, v) >= 0
            assert lib.lcq_mla_fwd_causal_workspace_bytes(w, 1, v, w) >= 0
            assert lib.lcq_mla_decode_workspace_bytes(v, 1, w, w) >= 0
            assert lib.lcq_mla_decode_workspace_bytes(1, w, 1, v) >= 0
