"""Cases that measure the operators of the paged decoder: rotary positions, the write into a paged key/value cache, attention
of a chunk of new tokens over that cache, and sampling of the next token.

Sizes: 8 heads of 64 and 96 columns, contexts of 250 and 500 tokens and 10000 words are those of configs/*.yaml and
bench.py; the longer contexts, shared key/value heads and larger vocabularies are generic serving sizes.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = 'cuda'
TYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
BASE = 10000.0


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the queries and keys of one decoding step of four hypotheses: a launch's latency
        dict(name='rotary step', op='rotary', rows=4, heads=16, dh=64, rot=64, layout='half', scaling='none', factor=1.0, far=500,
             dtype='bf16', backward=False, packed=True),
        # the 16 query and key heads inside the packed projection of 32 x 500 encoder frames, forward and backward
        dict(name='rotary training', op='rotary', rows=16000, heads=16, dh=96, rot=96, layout='half', scaling='none', factor=1.0,
             far=500, dtype='bf16', backward=True, packed=True),
        # a long context stretched 16 times, half of each head rotated in neighbouring pairs, at odd far positions
        dict(name='rotary far', op='rotary', rows=4099, heads=9, dh=96, rot=48, layout='interleaved', scaling='parts', factor=16.0,
             far=1 << 20, dtype='fp32', backward=True, packed=False),
        # 64 hypotheses write one token each, their queries and keys rotated on the way
        dict(name='append step', op='append', seqs=64, most_new=1, most_ctx=500, hq=8, hkv=8, dh=96, page=16, rot=96, dtype='bf16', lens=1),
        # forced prefixes of several lengths enter the cache at once
        dict(name='append chunk', op='append', seqs=37, most_new=700, most_ctx=1500, hq=8, hkv=8, dh=64, page=64, rot=64, dtype='bf16', lens=2),
        # one decoding step of a small batch, few keys: latency
        dict(name='attend step', op='attend', seqs=8, most_new=1, most_ctx=500, hq=8, hkv=8, dh=64, page=16, causal=True, dtype='bf16', lens=3),
        # one decoding step over long contexts with four query heads to a key/value head: the cache's bytes
        dict(name='attend step long', op='attend', seqs=32, most_new=1, most_ctx=32000, hq=32, hkv=8, dh=128, page=64, causal=True,
             dtype='bf16', lens=4),
        # ragged prefixes over ragged caches, single precision
        dict(name='attend chunk fp32', op='attend', seqs=13, most_new=75, most_ctx=611, hq=8, hkv=8, dh=64, page=16, causal=True, dtype='fp32', lens=5),
        # every query sees every key: hypotheses' prefixes against encoder states kept in pages
        dict(name='attend encoder', op='attend', seqs=32, most_new=40, most_ctx=500, hq=8, hkv=8, dh=96, page=32, causal=False, dtype='bf16', lens=6),
        # long prompts in chunks behind what the cache holds already: the matrix cores
        dict(name='attend prompt', op='attend', seqs=3, most_new=4096, most_ctx=9000, hq=16, hkv=4, dh=128, page=64, causal=True, dtype='bf16', lens=7),
        # the next token of one sentence
        dict(name='sample one', op='sample', rows=1, words=10000, top_k=0, top_p=0.9, min_p=0.0, temperature=0.8, masked=False, dtype='fp32'),
        # a full batch with every filter
        dict(name='sample batch', op='sample', rows=256, words=32003, top_k=200, top_p=0.95, min_p=0.02, temperature=1.1, masked=True, dtype='fp32'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return max(w['bytes'], w['flops'] / 50)


def draw(rng):
    limit = {'rotary': 2 << 28, 'append': 1 << 28, 'attend': 2 << 30, 'sample': 1 << 26}
    op = rng.choice(['rotary', 'append', 'attend', 'attend', 'sample'])
    while True:
        dtype = 'fp32' if rng.random() < 0.25 else 'bf16'
        dh = rng.choice([8, 32, 64, 64, 72, 96, 96, 128, 128, 192, 256])
        if op == 'rotary':
            rot = dh if rng.random() < 0.6 else max(2, 2 * rng.randint(1, dh // 2))
            scaling = rng.choice(['none', 'none', 'linear', 'base', 'parts']) if rot > 2 else 'none'
            c = dict(op=op, rows=_log(rng, 1, 30000), heads=rng.randint(1, 33), dh=dh, rot=rot, layout=rng.choice(['half', 'interleaved']),
                     scaling=scaling, factor=1.0 if scaling == 'none' else rng.uniform(1.5, 32.0), far=_log(rng, 250, 1 << 20), dtype=dtype,
                     backward=rng.random() < 0.5, packed=rng.random() < 0.5)
        elif op == 'sample':
            c = dict(op=op, rows=_log(rng, 1, 600), words=_log(rng, 300, 130000), top_k=0 if rng.random() < 0.4 else _log(rng, 1, 2000),
                     top_p=1.0 if rng.random() < 0.4 else rng.uniform(0.3, 0.99), min_p=0.0 if rng.random() < 0.5 else rng.uniform(0.001, 0.2),
                     temperature=rng.uniform(0.5, 1.6), masked=rng.random() < 0.5, dtype='fp32' if rng.random() < 0.7 else 'bf16')
        else:
            hkv = rng.choice([1, 2, 4, 5, 8, 8, 16])
            hq = hkv * rng.choice([1, 1, 1, 2, 3, 4, 8])
            if hq > 64:
                continue
            new = 1 if rng.random() < 0.4 else _log(rng, 2, 4000)
            c = dict(op=op, seqs=_log(rng, 1, 130), most_new=new, most_ctx=_log(rng, max(new, 16), 32000), hq=hq, hkv=hkv, dh=dh,
                     page=rng.choice([16, 32, 64, 128]), dtype=dtype, lens=rng.randint(10, 1 << 20))
            if op == 'append':
                c['rot'] = rng.choice([0, dh, max(2, dh // 2)])
            else:
                c['causal'] = rng.random() < 0.8
                # the plain form's table of all scores
                if c['seqs'] * hq * new * c['most_ctx'] > (1 << 30) or (dtype == 'fp32' and work(c)['flops'] > 2e11):
                    continue
            if c['seqs'] * c['most_ctx'] * hkv * dh > (1 << 30):
                continue
        if _cost(c) <= limit[op]:
            return c


def _lengths(c):
    """(new tokens, tokens in the cache with them) of every sequence: ragged, with a sequence that brings nothing, one that
    is a fresh prompt and one that is empty where there are enough sequences."""
    r = random.Random(c['lens'])
    new, ctx = [], []
    for i in range(c['seqs']):
        n = c['most_new'] if i == 0 or c['most_new'] == 1 else r.randint(max(1, c['most_new'] // 4), c['most_new'])
        t = c['most_ctx'] if i == 0 else r.randint(max(n, c['most_ctx'] // 4), c['most_ctx'])
        if c['seqs'] >= 6:
            if i == 2:
                t = n
            if i == 3:
                n = 0
            if i == 4:
                n = t = 0
        new.append(n)
        ctx.append(t)
    return new, ctx


def _pairs(c):
    """queries times the keys they see"""
    new, ctx = _lengths(c)
    if not c['causal']:
        return sum(n * t for n, t in zip(new, ctx))
    return sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, ctx))


def work(case):
    c = case
    es = 2 if c['dtype'] == 'bf16' else 4
    if c['op'] == 'rotary':
        n = c['rows'] * c['heads'] * c['dh']
        times = 2 if c['backward'] else 1
        return {'bytes': times * (2 * n * es + 4 * c['rows']), 'flops': times * 3 * c['rows'] * c['heads'] * c['rot']}
    if c['op'] == 'sample':
        return {'bytes': c['rows'] * (c['words'] * es + 12), 'flops': 4 * c['rows'] * c['words']}
    new, ctx = _lengths(c)
    tokens = sum(new)
    if c['op'] == 'append':
        return {'bytes': 2 * tokens * c['dh'] * es * (2 * c['hkv'] + (c['hq'] if c['rot'] else 0)),
                'flops': 3 * tokens * c['rot'] * (c['hq'] + c['hkv'])}
    seen = sum(t for n, t in zip(new, ctx) if n)
    return {'bytes': es * c['dh'] * (2 * tokens * c['hq'] + 2 * seen * c['hkv']), 'flops': 4 * c['hq'] * c['dh'] * _pairs(c)}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _frequencies(rot, scaling, factor):
    """radians per position of each pair, fp64, and the factor on the rotated columns"""
    base = BASE * factor ** (rot / (rot - 2)) if scaling == 'base' else BASE
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == 'linear':
        f = [x / factor for x in f]
    if scaling == 'parts':      # slow pairs stretched, fast ones kept, in between by the turns they make in 4096 positions
        g = [min(1.0, max(0.0, (4096 * x / (2 * math.pi) - 1.0) / (32.0 - 1.0))) for x in f]
        f = [x * ((1 - a) / factor + a) for x, a in zip(f, g)]
    return f, (0.1 * math.log(factor) + 1.0 if scaling == 'parts' else 1.0)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[c['dtype']]
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV).to(t)
    if c['op'] == 'rotary':
        f, m = _frequencies(c['rot'], c['scaling'], c['factor'])
        rows, heads, dh = c['rows'], c['heads'], c['dh']
        x = normal(rows, heads * dh + (heads // 2 or 1) * dh)[:, :heads * dh] if c['packed'] else normal(rows, heads * dh)
        return dict(c=c, x=x.unflatten(1, (heads, dh)), dy=normal(rows, heads, dh),
                    freq=torch.tensor(f, dtype=torch.float64, device=DEV), mscale=m,
                    pos=torch.randint(0, c['far'], (rows,), generator=g, device=DEV, dtype=torch.int32))
    if c['op'] == 'sample':
        x = 3.0 * torch.randn(c['rows'], c['words'], generator=g, device=DEV)
        if c['masked']:         # words the caller forbids
            x = x.masked_fill(torch.rand(x.shape, generator=g, device=DEV) < 0.1, float('-inf'))
        return dict(c=c, logits=x.to(t), u=torch.rand(c['rows'], generator=g, device=DEV),
                    **{k: float(np.float32(c[k])) for k in ('temperature', 'top_p', 'min_p')})      # numbers that fp32 holds
    new, ctx = _lengths(c)
    page = c['page']
    wide = -(-c['most_ctx'] // page)
    used = sum(-(-n // page) for n in ctx)
    order = torch.randperm(used + 3, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in ctx:
        k = -(-n // page)
        table.append(order[at:at + k] + [-1] * (wide - k))
        at += k
    tokens = sum(new)
    hq, hkv, dh = c['hq'], c['hkv'], c['dh']
    s = dict(c=c, k_pages=normal(used + 3, hkv, page, dh), v_pages=normal(used + 3, hkv, dh, page),
             table=torch.tensor(table, dtype=torch.int32).to(DEV), ctx=torch.tensor(ctx, dtype=torch.int32).to(DEV),
             cu=torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).to(DEV))
    if c['op'] == 'append':
        packed = normal(tokens, (hq + 2 * hkv) * dh)
        s['q'], s['k'], s['v'] = (x.unflatten(1, (-1, dh)) for x in packed.split([hq * dh, hkv * dh, hkv * dh], 1))
        s['freq'] = torch.tensor(_frequencies(c['rot'], 'none', 1.0)[0], dtype=torch.float64, device=DEV) if c['rot'] else None
    else:
        s['q'] = normal(tokens, hq, dh)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state['c']
    if own:
        from neurst_amd import ops
        if c['op'] == 'rotary':
            y = ops.rotary(s['x'], s['freq'], s['pos'], layout=c['layout'], mscale=s['mscale'])
            if not c['backward']:
                return y
            return y, ops.rotary(s['dy'], s['freq'], s['pos'], layout=c['layout'], mscale=s['mscale'], inverse=True)
        if c['op'] == 'sample':
            return ops.sample(s['logits'], s['u'], temperature=s['temperature'], top_k=c['top_k'], top_p=s['top_p'], min_p=s['min_p'])
        if c['op'] == 'append':
            q = ops.paged_append(s['k'], s['v'], s['k_pages'], s['v_pages'], s['table'], s['cu'], s['ctx'],
                                 q=s['q'] if c['rot'] else None, freq=s['freq'])
            return (s['k_pages'], s['v_pages'], q) if c['rot'] else (s['k_pages'], s['v_pages'])
        return ops.paged_attention(s['q'], s['k_pages'], s['v_pages'], s['table'], s['cu'], s['ctx'], causal=c['causal'])
    if c['op'] == 'rotary':
        y = _turn(s['x'], s['freq'], s['pos'], c['layout'], s['mscale'], 1.0)
        return (y, _turn(s['dy'], s['freq'], s['pos'], c['layout'], s['mscale'], -1.0)) if c['backward'] else y
    if c['op'] == 'sample':
        return _choose(s, s['u'], c['top_k'])
    if c['op'] == 'append':
        return _write(s)
    return _attend(s)


def _turn(x, freq, pos, layout, mscale, sign):
    """x [rows, heads, dh]: the first 2 * len(freq) columns of each head rotated by sign * position * frequency"""
    n = freq.numel()
    a = (pos.double()[:, None] * freq)[:, None]
    cos, sin = (torch.cos(a) * mscale).float(), (torch.sin(a) * (mscale * sign)).float()
    x32 = x.float()
    u, v = (x32[..., :n], x32[..., n:2 * n]) if layout == 'half' else (x32[..., 0:2 * n:2], x32[..., 1:2 * n:2])
    p, q = u * cos - v * sin, v * cos + u * sin
    y = torch.cat([p, q], -1) if layout == 'half' else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([y, x32[..., 2 * n:]], -1).to(x.dtype)


def _places(s):
    """sequence and position of every new token (int64)"""
    cu, ctx = s['cu'].long(), s['ctx'].long()
    new = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=DEV), new, output_size=s['q'].shape[0])
    return seq, torch.arange(seq.numel(), device=DEV) - cu[seq] + (ctx - new)[seq]


def _write(s):
    page = s['c']['page']
    seq, pos = _places(s)
    at, slot = s['table'][seq, pos // page].long(), pos % page
    k, q = s['k'], None
    if s['freq'] is not None:
        k, q = _turn(k, s['freq'], pos, 'half', 1.0, 1.0), _turn(s['q'], s['freq'], pos, 'half', 1.0, 1.0)
    s['k_pages'][at, :, slot] = k
    s['v_pages'][at, :, :, slot] = s['v']
    return (s['k_pages'], s['v_pages'], q) if q is not None else (s['k_pages'], s['v_pages'])


def _attend(s):
    c = s['c']
    dh, hkv, group, page = c['dh'], c['hkv'], c['hq'] // c['hkv'], c['page']
    seq, pos = _places(s)
    table = s['table'].long().clamp(min=0)
    B, wide = table.shape
    long = wide * page
    k = s['k_pages'][table].float().permute(0, 2, 1, 3, 4).reshape(B, hkv, long, dh)
    v = s['v_pages'][table].float().permute(0, 2, 1, 4, 3).reshape(B, hkv, long, dh)
    key = torch.arange(long, device=DEV)
    there = key < s['ctx'].long()[:, None]
    v = torch.where(there[:, None, :, None], v, 0.0)
    most = c['most_new']
    row = torch.arange(seq.numel(), device=DEV) - s['cu'].long()[seq]
    q = torch.zeros(B, most, c['hq'], dh, device=DEV)
    q[seq, row] = s['q'].float()
    where = torch.full((B, most), -1, dtype=torch.int64, device=DEV)
    where[seq, row] = pos if c['causal'] else long
    q = q.view(B, most, hkv, group, dh).permute(0, 2, 3, 1, 4).reshape(B, hkv, group * most, dh)
    w = torch.matmul(q, k.transpose(2, 3)) * dh ** -0.5
    see = (there[:, None, :] & (key <= where[:, :, None]))[:, None, None]
    w = w.view(B, hkv, group, most, long).masked_fill_(~see, float('-inf'))
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, hkv, group * most, long), v).view(B, hkv, group, most, dh) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, c['hq'], dh)
    return o[seq, row].to(s['q'].dtype)


def _choose(s, u, top_k):
    """ids int32 and their log-probabilities among the words kept; sums of 64 bits, since a draw that falls next to a border
    would otherwise go to either side"""
    x = s['logits'].double()
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((top - top[:, :1]) / s['temperature'])
    keep = torch.ones_like(w, dtype=torch.bool)
    if top_k > 0:
        keep[:, top_k:] = False
    w = w * keep
    if s['top_p'] < 1.0:
        keep &= torch.cumsum(w, 1) - w < s['top_p'] * w.sum(1, keepdim=True)
    keep &= w >= s['min_p']
    p = torch.zeros_like(w).scatter_(1, order, w * keep)
    run_sum = torch.cumsum(p, 1)
    total = run_sum[:, -1:]
    ids = ((run_sum <= u.double()[:, None] * total) | (p <= 0)).int().argmin(1)
    logp = torch.log(p.gather(1, ids[:, None]) / total)[:, 0]
    return ids.int(), logp.float()


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------------
def _spin(x, f, pos, layout, mscale, sign):
    """rotation as a product of complex numbers"""
    n = len(f)
    x = x.double()
    phase = torch.polar(torch.full((pos.numel(), n), mscale, dtype=torch.float64, device=x.device),
                        sign * torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device=x.device)))[:, None]
    y = x.clone()
    if layout == 'half':
        z = torch.complex(x[..., :n], x[..., n:2 * n]) * phase
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * phase
        y[..., :2 * n] = torch.view_as_real(z).flatten(-2)
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c['op'] == 'rotary':
        f, m = _frequencies(c['rot'], c['scaling'], c['factor'])
        y = _spin(s['x'], f, s['pos'], c['layout'], m, 1.0)
        return (y, _spin(s['dy'], f, s['pos'], c['layout'], m, -1.0)) if c['backward'] else y
    if c['op'] == 'sample':
        return _exact_choice(s, c)
    new, ctx = _lengths(c)
    page, table = c['page'], s['table'].tolist()
    if c['op'] == 'append':
        k_pages, v_pages, begin, turned = s['k_pages'].double(), s['v_pages'].double(), 0, []
        for b, (n, t) in enumerate(zip(new, ctx)):
            if not n:
                continue
            pos = torch.arange(t - n, t, device=DEV)
            k, v, q = s['k'][begin:begin + n].double(), s['v'][begin:begin + n].double(), s['q'][begin:begin + n].double()
            if c['rot']:
                f = _frequencies(c['rot'], 'none', 1.0)[0]
                k, q = _spin(k, f, pos, 'half', 1.0, 1.0), _spin(q, f, pos, 'half', 1.0, 1.0)
            turned.append(q)
            for first in range((t - n) // page * page, t, page):
                lo, hi = max(first, t - n), min(first + page, t)
                at = table[b][first // page]
                k_pages[at, :, lo - first:hi - first] = k[lo - (t - n):hi - (t - n)].transpose(0, 1)
                v_pages[at, :, :, lo - first:hi - first] = v[lo - (t - n):hi - (t - n)].permute(1, 2, 0)
            begin += n
        q = torch.cat(turned) if turned else s['q'][:0].double()
        return (k_pages, v_pages, q) if c['rot'] else (k_pages, v_pages)
    o, begin, group = torch.zeros_like(s['q'], dtype=torch.float64), 0, c['hq'] // c['hkv']
    for b, (n, t) in enumerate(zip(new, ctx)):
        if n and t:
            at = table[b][:-(-t // page)]
            for h in range(c['hkv']):
                k = s['k_pages'][at, h].double().reshape(-1, c['dh'])[:t]
                v = s['v_pages'][at, h].double().transpose(1, 2).reshape(-1, c['dh'])[:t]
                for j in range(group):
                    q = s['q'][begin:begin + n, h * group + j].double()
                    w = q @ k.t() / math.sqrt(c['dh'])
                    if c['causal']:
                        w = w + torch.full_like(w, float('-inf')).triu(t - n + 1)
                    o[begin:begin + n, h * group + j] = torch.softmax(w, -1) @ v
        begin += n
    return o


def _exact_choice(s, c):
    ids, logs = [], []
    for row, u in zip(s['logits'].double().cpu().numpy(), s['u'].double().cpu().numpy()):
        order = np.lexsort((np.arange(row.size), -row))
        if c['top_k']:
            order = order[:c['top_k']]
        w = np.exp((row[order] - row[order[0]]) / s['temperature'])
        if s['top_p'] < 1:
            cut = int(np.searchsorted(np.cumsum(w), s['top_p'] * w.sum())) + 1
            order, w = order[:cut], w[:cut]
        fine = w >= s['min_p']
        order, w = order[fine], w[fine]
        back = np.argsort(order)
        order, w = order[back], w[back]
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u * sums[-1], side='right')), w.size - 1)
        ids.append(order[at])
        logs.append(math.log(w[at] / sums[-1]))
    return torch.tensor(np.array(ids), dtype=torch.int32), torch.tensor(logs, dtype=torch.float64)
