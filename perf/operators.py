"""The serving operators of a packed model, as cases that can be timed and checked.

Four operators of ``lightcompress_amd.ops``: ``int4_linear`` (the product with 4-bit packed
weights and group scales, the two deploy layouts), ``int4_linear_grouped`` (the same products of
an MoE layer's routed experts, ragged row counts), ``mla_fwd_causal`` (latent attention in its
expanded form, for prompts and chunks) and ``mla_decode`` (its absorbed form over a paged latent
cache, for single tokens). With ``own`` false, ``run`` computes each in its plain form from
elementary torch operations in 32 bits, rounded once; with ``own`` true it makes the calls a
user makes. ``exact`` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False  # set by the caller: the framework's kernels instead of the plain forms

DT = {'bf16': torch.bfloat16, 'fp16': torch.float16}
NOPE, ROPE, VDIM, LATENT = 128, 64, 128, 512   # the latent attention's head and latent widths
AWQ_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)           # column of nibble i of an AutoAWQ word


def listed():
    return [
        # one token through a 4096 x 4096 projection of a packed 8B model: launch latency
        dict(name='linear_token', op='linear', layout='vllm', dtype='bf16', m=1, n=4096, k=4096,
             group=128),
        # one token through its MLP's down projection, zero points, AutoAWQ layout
        dict(name='linear_token_awq', op='linear', layout='autoawq', dtype='fp16', m=1, n=4096,
             k=14336, group=128),
        # a batch of 37 sequences' tokens through the gate projection, smaller groups
        dict(name='linear_batch', op='linear', layout='autoawq', dtype='bf16', m=37, n=14336,
             k=4096, group=64),
        # a prompt of 2048 tokens through the gate projection
        dict(name='linear_prompt', op='linear', layout='vllm', dtype='bf16', m=2048, n=14336,
             k=4096, group=128),
        # 16 tokens, top 8 of 64 experts: gate and up with the SiLU product
        dict(name='experts_decode', op='grouped', layout='vllm', dtype='bf16', tokens=16, topk=8,
             experts=64, n=2048, k=7168, group=128, silu=True, gather=True),
        # one token's 8 experts: down projection
        dict(name='experts_token', op='grouped', layout='autoawq', dtype='bf16', tokens=1, topk=8,
             experts=32, n=7168, k=2048, group=128, silu=False, gather=False),
        # a prompt of 1000 tokens, top 8 of 32 experts
        dict(name='experts_prompt', op='grouped', layout='vllm', dtype='bf16', tokens=1000,
             topk=8, experts=32, n=2048, k=7168, group=128, silu=True, gather=True),
        # a short padded batch of a small-headed model
        dict(name='prefill_padded', op='prefill', dtype='fp16', batch=4, heads=16, sq=301,
             skv=301, padded=True),
        # a prompt of 2048 tokens at 128 heads (calibration and prefill)
        dict(name='prefill_prompt', op='prefill', dtype='bf16', batch=1, heads=128, sq=2048,
             skv=2048, padded=False),
        # a chunk of 77 tokens behind 4096 cached ones
        dict(name='prefill_chunk', op='prefill', dtype='bf16', batch=1, heads=128, sq=77,
             skv=4173, padded=False),
        # one short sequence, few heads (one rank of eight): launch latency
        dict(name='decode_one', op='decode', dtype='bf16', batch=1, heads=16, sq=1, ctx=777,
             page=64),
        # 32 sequences of up to 8192 tokens at 128 heads, one speculated token each
        dict(name='decode_batch', op='decode', dtype='bf16', batch=32, heads=128, sq=2, ctx=8192,
             page=64),
    ]


def draw(rng):
    """One more case of the same ranges, no dearer than the listed ones."""
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(['linear', 'grouped', 'prefill', 'decode'])
    dtype = rng.choice(['bf16', 'fp16'])
    while True:
        if op == 'linear':
            k = 128 * log(4, 112)
            layout = rng.choice(['vllm', 'autoawq'])
            n = log(256, 14336)
            c = dict(op=op, layout=layout, dtype=dtype, m=log(1, 2048),
                     n=n if layout == 'vllm' else 8 * (n // 8), k=k,
                     group=rng.choice([32, 64, 128, 128, k]))
            ok = c['m'] * c['n'] * k <= 2048 * 14336 * 4096
        elif op == 'grouped':
            k = 128 * log(8, 56)
            c = dict(op=op, layout=rng.choice(['vllm', 'autoawq']), dtype=dtype,
                     tokens=log(1, 1000), topk=rng.choice([2, 4, 6, 8]),
                     experts=rng.choice([8, 16, 27, 32, 64]), n=8 * log(96, 256), k=k,
                     group=rng.choice([32, 64, 128, 128]), silu=rng.random() < 0.5,
                     gather=rng.random() < 0.5)
            ok = True
        elif op == 'prefill':
            sq = log(1, 2048)
            c = dict(op=op, dtype=dtype, batch=log(1, 8), heads=rng.choice([8, 16, 32, 128]),
                     sq=sq, skv=sq + rng.choice([0, log(1, 4096)]),
                     padded=rng.random() < 0.3)
            ok = c['batch'] * c['heads'] * sq * c['skv'] <= 128 * 2048 * 2048
        else:
            c = dict(op=op, dtype=dtype, batch=log(1, 32), heads=rng.choice([8, 16, 32, 64, 128]),
                     sq=rng.choice([1, 1, 2, 3]), ctx=log(16, 65536),
                     page=rng.choice([1, 16, 48, 64, 256]))
            ok = c['batch'] * c['ctx'] * c['heads'] * c['sq'] <= 32 * 8192 * 128 * 2
        if ok:
            return c


# ---- inputs ----------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) % (1 << 62))


def _acts(g, *shape, dtype):
    """Hidden states: unit normal with a few channels ten times as large."""
    x = torch.randn(*shape, generator=g, device='cuda')
    big = torch.rand(shape[-1], generator=g, device='cuda') < 0.004
    return torch.where(big, x * 10, x).to(dtype)


def _codes(g, rows, cols):
    """4-bit codes of normal weights under a min-max range per group."""
    c = torch.randn(rows, cols, generator=g, device='cuda')
    return c.mul_(2.7).add_(7.5).round_().clamp_(0, 15).to(torch.int32)


def _pack_cols(codes, order):
    """Words of 8 codes along the last axis; nibble i holds code order[i] of its word."""
    c = codes.view(codes.shape[0], -1, 8)
    w = torch.zeros(c.shape[:2], dtype=torch.int32, device=c.device)
    for i, o in enumerate(order):
        w |= c[..., o] << (4 * i)
    return w


def _weight(g, layout, n, k, group):
    """(qweight, scales, qzeros) of one projection as the deploy path stores it."""
    ng = k // group
    if layout == 'vllm':     # [n, k/8] words along k, code + 8, symmetric
        qw = _pack_cols(_codes(g, n, k), range(8))
        s = torch.rand(n, ng, generator=g, device='cuda')
        return qw, s.mul_(0.008).add_(0.004).to(torch.float16), None
    qw = _pack_cols(_codes(g, k, n), AWQ_ORDER)  # [k, n/8] words along n, zero points
    s = torch.rand(ng, n, generator=g, device='cuda').mul_(0.008).add_(0.004).to(torch.float16)
    z = torch.randint(5, 11, (ng, n), generator=g, device='cuda', dtype=torch.int32)
    return qw, s, _pack_cols(z, AWQ_ORDER)


def _lens(case, full):
    """Ragged lengths of a batch, from full down to about a quarter, one of them a single token
    where the batch is large enough; the same multiset for every seed."""
    b = case['batch']
    out = [max(1, full - (3 * full * i) // (4 * b)) for i in range(b)]
    if b >= 4:
        out[b // 2] = 1
    return out


def prepare(case, seed):
    g = _gen(seed)
    rng = np.random.default_rng(seed)
    dt = DT[case['dtype']]
    st = dict(case=case)
    if case['op'] == 'linear':
        st['w'] = _weight(g, case['layout'], case['n'], case['k'], case['group'])
        st['x'] = _acts(g, case['m'], case['k'], dtype=dt)
    elif case['op'] == 'grouped':
        E, T, k = case['experts'], case['tokens'], case['topk']
        sets = 2 if case['silu'] else 1
        st['w'] = [[_weight(g, case['layout'], case['n'], case['k'], case['group'])
                    for _ in range(E)] for _ in range(sets)]
        # top k of random router scores per token, the slots sorted by expert
        choice = np.argsort(rng.random((T, E)), axis=1)[:, :min(k, E)].reshape(-1)
        order = np.argsort(choice, kind='stable')
        off = np.concatenate([[0], np.cumsum(np.bincount(choice, minlength=E))])
        st['off'] = [int(v) for v in off]
        st['row_off'] = torch.tensor(off, dtype=torch.int64, device='cuda')
        rows = len(choice)
        st['a_rows'] = None
        if case['gather']:
            st['a_rows'] = torch.tensor(order // min(k, E), dtype=torch.int64, device='cuda')
        st['x'] = _acts(g, T if case['gather'] else rows, case['k'], dtype=dt)
        if own:
            from lightcompress_amd import ops
            tabs = [ops.int4_weight_table(ws, st['x'].device) for ws in st['w']]
            st['wtab'] = torch.stack(tabs).contiguous() if sets == 2 else tabs[0]
    elif case['op'] == 'prefill':
        B, H, sq, skv = case['batch'], case['heads'], case['sq'], case['skv']
        q = torch.randn(B, sq, H, NOPE + ROPE, generator=g, device='cuda').to(dt)
        kv = torch.randn(B, skv, H, NOPE + VDIM, generator=g, device='cuda').to(dt)
        kr = torch.randn(B, skv, ROPE, generator=g, device='cuda').to(dt)
        # the projections' own layouts, seen head by head
        st['q_nope'], st['q_rope'] = q.transpose(1, 2).split([NOPE, ROPE], -1)
        st['k_nope'], st['v'] = kv.transpose(1, 2).split([NOPE, VDIM], -1)
        st['k_rope'] = kr
        st['q_start'] = st['kv_lens'] = None
        if case['padded']:
            past = skv - sq
            lens = [past + v for v in _lens(case, sq)]
            rng.shuffle(lens)
            st['kv_lens'] = torch.tensor(lens, dtype=torch.int32, device='cuda')
            st['q_start'] = torch.full((B,), past, dtype=torch.int32, device='cuda')
    else:
        B, H, sq, ps = case['batch'], case['heads'], case['sq'], case['page']
        lens = _lens(case, case['ctx'])
        rng.shuffle(lens)
        nb = -(-case['ctx'] // ps)
        used = [-(-v // ps) for v in lens]
        pages = sum(used) + 3
        perm = rng.permutation(pages)
        table = np.zeros((B, nb), dtype=np.int32)
        at = 0
        for b in range(B):
            table[b, :used[b]] = perm[at:at + used[b]]
            at += used[b]
        cache = torch.randn(pages, ps, LATENT + ROPE, generator=g, device='cuda').to(dt)
        st['ckv'], st['k_rope'] = cache.split([LATENT, ROPE], -1)
        st['q_latent'] = torch.randn(B, sq, H, LATENT, generator=g, device='cuda').to(dt)
        st['q_rope'] = torch.randn(B, sq, H, ROPE, generator=g, device='cuda').to(dt)
        st['block_table'] = torch.tensor(table, device='cuda')
        st['kv_lens'] = torch.tensor(lens, dtype=torch.int32, device='cuda')
        st['lens'] = [int(v) for v in lens]
    return st


# ---- one pass --------------------------------------------------------------------------------
SCALE = (NOPE + ROPE) ** -0.5


def _unpack(words, order):
    """Codes [rows, 8 words] of packed words, in 32 bits."""
    out = torch.empty(*words.shape, 8, dtype=torch.int32, device=words.device)
    for i, o in enumerate(order):
        out[..., o] = (words >> (4 * i)) & 15
    return out.flatten(-2)


def _dequant(w, layout):
    """The float weight [n, k] of a packed one, in 32 bits."""
    qw, s, z = w
    if layout == 'vllm':
        q = (_unpack(qw, range(8)) - 8).float()
        n, k = q.shape
        return (q.view(n, s.shape[1], -1) * s.float()[..., None]).view(n, k)
    q = _unpack(qw, AWQ_ORDER).float()
    k, n = q.shape
    z = _unpack(z, AWQ_ORDER).float()
    return ((q.view(s.shape[0], -1, n) - z[:, None]) * s.float()[:, None]).view(k, n).t()


def _plain_attention(s, v):
    """softmax over the last axis of masked scores, times v; rows without a key give zero."""
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(torch.where(total > 0, p / total, torch.zeros_like(p)), v)


def _run_plain(st):
    c = st['case']
    dt = DT[c['dtype']]
    if c['op'] == 'linear':
        return torch.matmul(st['x'].float(), _dequant(st['w'], c['layout']).t()).to(dt)
    if c['op'] == 'grouped':
        x = st['x'].float() if st['a_rows'] is None else st['x'].float()[st['a_rows']]
        out = torch.empty(x.shape[0], c['n'], dtype=dt, device=x.device)
        for e in range(c['experts']):
            a, b = st['off'][e], st['off'][e + 1]
            if a == b:
                continue
            y = [torch.matmul(x[a:b], _dequant(ws[e], c['layout']).t()) for ws in st['w']]
            out[a:b] = (y[0] / (1 + torch.exp(-y[0])) * y[1] if c['silu'] else y[0]).to(dt)
        return out
    if c['op'] == 'prefill':
        B, H, sq, skv = c['batch'], c['heads'], c['sq'], c['skv']
        kr = st['k_rope'].float()[:, None].transpose(2, 3)
        s = torch.matmul(st['q_nope'].float(), st['k_nope'].float().transpose(2, 3))
        s = (s + torch.matmul(st['q_rope'].float(), kr)) * SCALE
        key = torch.arange(skv, device=s.device)
        start = (torch.full((B,), skv - sq, device=s.device) if st['q_start'] is None
                 else st['q_start'])
        pos = start[:, None] + torch.arange(sq, device=s.device)
        seen = key <= pos[:, :, None]
        if st['kv_lens'] is not None:
            seen &= key < st['kv_lens'][:, None, None]
        s.masked_fill_(~seen[:, None], -math.inf)
        return _plain_attention(s, st['v'].float()).transpose(1, 2).contiguous().to(dt)
    B, H, sq, ps = c['batch'], c['heads'], c['sq'], c['page']
    out = torch.empty(B, sq, H, LATENT, dtype=dt, device=st['ckv'].device)
    for b, n in enumerate(st['lens']):
        pages = st['block_table'][b, :-(-n // ps)].long()
        kv = st['ckv'][pages].reshape(-1, LATENT)[:n].float()
        kr = st['k_rope'][pages].reshape(-1, ROPE)[:n].float()
        s = torch.matmul(st['q_latent'][b].float(), kv.t())
        s = (s + torch.matmul(st['q_rope'][b].float(), kr.t())) * SCALE
        pos = n - sq + torch.arange(sq, device=s.device)
        s.masked_fill_((torch.arange(n, device=s.device) > pos[:, None])[:, None], -math.inf)
        out[b] = _plain_attention(s, kv).to(dt)
    return out


def _run_own(st):
    from lightcompress_amd import ops
    c = st['case']
    if c['op'] == 'linear':
        return ops.int4_linear(st['x'], *st['w'])
    if c['op'] == 'grouped':
        return ops.int4_linear_grouped(st['x'], st['row_off'], st['wtab'], c['n'], c['group'],
                                       layout=c['layout'], a_rows=st['a_rows'],
                                       silu_mul=c['silu'])
    if c['op'] == 'prefill':
        return ops.mla_fwd_causal(st['q_nope'], st['q_rope'], st['k_nope'], st['k_rope'],
                                  st['v'], SCALE, q_start=st['q_start'], kv_lens=st['kv_lens'])
    return ops.mla_decode(st['q_latent'], st['q_rope'], st['ckv'], st['k_rope'],
                          st['block_table'], st['kv_lens'], SCALE)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits -----------------------------------------------------------------
def _exact_weight(w, layout):
    qw, s, z = w
    dev = qw.device
    shift = torch.arange(0, 32, 4, device=dev)
    if layout == 'vllm':   # W[r, c] = (code - 8) * scale[r, c // group]
        code = ((qw[:, :, None].long() >> shift) & 15).reshape(qw.shape[0], -1).double()
        return (code - 8) * s.double().repeat_interleave(code.shape[1] // s.shape[1], dim=1)
    inv = torch.tensor([AWQ_ORDER.index(j) for j in range(8)], device=dev)
    code = ((qw[:, :, None].long() >> shift[inv]) & 15).reshape(qw.shape[0], -1).double()
    zero = ((z[:, :, None].long() >> shift[inv]) & 15).reshape(z.shape[0], -1).double()
    rep = code.shape[0] // s.shape[0]
    return ((code - zero.repeat_interleave(rep, dim=0))
            * s.double().repeat_interleave(rep, dim=0)).T


def _exact_softmax(s, ok, v):
    """Rows of scores s [rows, keys] with the visible keys ok, over values v [keys, d]."""
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    p = torch.softmax(s, dim=-1)
    return torch.where(ok.any(-1, keepdim=True), p, torch.zeros_like(p)) @ v


def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'linear':
        return st['x'].double() @ _exact_weight(st['w'], case['layout']).T
    if case['op'] == 'grouped':
        rows = st['off'][-1]
        src = st['a_rows'] if st['a_rows'] is not None else torch.arange(rows, device='cuda')
        out = torch.empty(rows, case['n'], dtype=torch.float64, device='cuda')
        for e in range(case['experts']):
            sel = slice(st['off'][e], st['off'][e + 1])
            if sel.start == sel.stop:
                continue
            x = st['x'][src[sel]].double()
            y = x @ _exact_weight(st['w'][0][e], case['layout']).T
            if case['silu']:
                y = y * torch.sigmoid(y) * (x @ _exact_weight(st['w'][1][e], case['layout']).T)
            out[sel] = y
        return out
    if case['op'] == 'prefill':
        B, H, sq, skv = case['batch'], case['heads'], case['sq'], case['skv']
        out = torch.empty(B, sq, H, VDIM, dtype=torch.float64, device='cuda')
        j = torch.arange(skv, device='cuda')[None]
        i = torch.arange(sq, device='cuda')[:, None]
        for b in range(B):
            first = skv - sq if st['q_start'] is None else int(st['q_start'][b])
            n = skv if st['kv_lens'] is None else int(st['kv_lens'][b])
            ok = (j <= first + i) & (j < n)
            for h in range(H):
                q = torch.cat([st['q_nope'][b, h], st['q_rope'][b, h]], -1).double()
                k = torch.cat([st['k_nope'][b, h], st['k_rope'][b]], -1).double()
                out[b, :, h] = _exact_softmax(q @ k.T * SCALE, ok, st['v'][b, h].double())
        return out
    B, H, sq, ps = case['batch'], case['heads'], case['sq'], case['page']
    out = torch.empty(B, sq, H, LATENT, dtype=torch.float64, device='cuda')
    for b, n in enumerate(st['lens']):
        j = torch.arange(n, device='cuda')
        page, slot = st['block_table'][b][j // ps].long(), j % ps
        c = st['ckv'][page, slot].double()
        k = torch.cat([c, st['k_rope'][page, slot].double()], -1)
        for i in range(sq):
            q = torch.cat([st['q_latent'][b, i], st['q_rope'][b, i]], -1).double()
            ok = (j <= n - sq + i)[None].expand(H, n)
            out[b, i] = _exact_softmax(q @ k.T * SCALE, ok, c)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------
def _weight_bytes(case):
    n, k, ng = case['n'], case['k'], case['k'] // case['group']
    return n * k // 2 + 2 * n * ng + (n * ng // 2 if case['layout'] == 'autoawq' else 0)


def work(case):
    if case['op'] == 'linear':
        m, n, k = case['m'], case['n'], case['k']
        return dict(bytes=_weight_bytes(case) + 2 * m * (n + k), flops=2 * m * n * k)
    if case['op'] == 'grouped':
        E, top = case['experts'], min(case['topk'], case['experts'])
        rows, sets = case['tokens'] * top, 2 if case['silu'] else 1
        hit = E * (1 - (1 - top / E) ** case['tokens'])  # expected experts with a row
        x = case['tokens'] if case['gather'] else rows
        return dict(bytes=int(hit * sets * _weight_bytes(case)) + 2 * x * case['k']
                    + 2 * rows * case['n'] + 8 * (E + 1), flops=2 * rows * case['n'] * case['k'] * sets)
    if case['op'] == 'prefill':
        B, H, sq, skv = case['batch'], case['heads'], case['sq'], case['skv']
        past = skv - sq
        lens = [past + v for v in _lens(case, sq)] if case['padded'] else [skv] * B
        pairs = sum(min(past + i + 1, n) for n in lens for i in range(sq))
        return dict(bytes=2 * (B * sq * H * (NOPE + ROPE + VDIM)
                               + sum(lens) * (H * (NOPE + VDIM) + ROPE)),
                    flops=2 * H * pairs * (NOPE + ROPE + VDIM))
    B, H, sq = case['batch'], case['heads'], case['sq']
    lens = _lens(case, case['ctx'])
    pairs = sum(max(0, n - sq + i + 1) for n in lens for i in range(sq))
    return dict(bytes=2 * (sum(lens) * (LATENT + ROPE) + B * sq * H * (2 * LATENT + ROPE)),
                flops=2 * H * pairs * (2 * LATENT + ROPE))
