"""Rotary positions, the paged cache, attention over it and sampling on the GPU against plain 64-bit implementations of their
formulas.

Tolerances, derived: half a step of a type is eps / 2 relative.
  rotary: angle good to 1e-9, sine and cosine to 2^-23 absolute, two products and a sum of 2^-24 each: (|u| + |v|) 2^-21, plus
    half a step of the result.
  attention: with w the weights, A = sum_j w_j |v_j| bounds what a relative error of the weights can move the result by.
    Scores: a dh-term fp32 dot product, at most (dh + 8) 2^-24 sum |q k| off, twice that for the pair of errors of a weight and
    its sum; exp2, the running rescales and the sums of n terms: (n + 64) 2^-23; weights rounded to bf16: half a step; the
    result rounded: half a step of itself.
  sampling: ids equal; logp one fp32 rounding, plus one unit of the integer weights over the weight drawn."""
import math

import numpy as np
import pytest
import torch

from neurst_amd import lib, ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}
half_step = lambda t: torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def within(got, want, bound, what=''):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - bound
    assert (off <= 0).all(), '%s: %g over the bound of %g at %d' % (what, off.max(), bound.flatten()[off.argmax()] if torch.is_tensor(bound) else bound, off.argmax())


# ---- rotary ----------------------------------------------------------------------------------------------------------------
def turn(x, freq, pos, layout='half', mscale=1.0, sign=1.0):
    """fp64; also the columns' partner magnitudes, for the bound"""
    n = freq.numel()
    x = x.double()
    a = (pos.double()[:, None] * freq.double())[:, None]
    c, s = torch.cos(a) * mscale, torch.sin(a) * mscale * sign
    y, size = x.clone(), x.abs().clone()
    at = (slice(0, n), slice(n, 2 * n)) if layout == 'half' else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    u, v = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = u * c - v * s, v * c + u * s
    size[..., at[0]] = size[..., at[1]] = (u.abs() + v.abs()) * abs(mscale)
    return y, size


def rot_bound(y, size, t):
    return size * 2.0 ** -21 + y.abs() * half_step(t) * (1 + 2.0 ** -8) + 1e-30


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('rows,heads,dh,rot', [(1, 1, 2, 2), (5, 3, 8, 8), (7, 2, 96, 48), (33, 5, 72, 36), (64, 16, 64, 64), (3, 4, 10, 6),
                                               (2, 1, 256, 256), (1025, 9, 96, 96), (4, 2, 24, 14)])
def test_rotary(dtype, layout, rows, heads, dh, rot):
    t, g = TYPES[dtype], gen(rows * dh + rot)
    freq, m = ops.rotary_frequencies(rot, scaling='parts' if rot > 8 else None, factor=4.0 if rot > 8 else 1.0, device=DEV)
    x = normal(g, rows, heads, dh, dtype=t)
    pos = torch.randint(-1000, 1 << 20, (rows,), generator=g, device=DEV, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    y = ops.rotary(x, freq, pos, layout=layout, mscale=m)
    want, size = turn(x, freq, pos, layout, m)
    within(y, want, rot_bound(want, size, t), 'forward')
    assert torch.equal(y[..., rot:], x[..., rot:])
    # the gradient: the transposed matrix, checked as the formula and as <R x, dy> = <x, R' dy>
    dy = normal(g, rows, heads, dh, dtype=t)
    dx = ops.rotary(dy, freq, pos, layout=layout, mscale=m, inverse=True)
    want_dx, size_dx = turn(dy, freq, pos, layout, m, -1.0)
    within(dx, want_dx, rot_bound(want_dx, size_dx, t), 'gradient')
    lhs, rhs = (want * dy.double()).sum(), (x.double() * want_dx).sum()
    assert abs(lhs - rhs) <= 1e-10 * (want.abs() * dy.double().abs()).sum()
    # in place, and inside rows that hold more than these heads
    z = x.clone()
    assert ops.rotary(z, freq, pos, layout=layout, mscale=m, out=z) is z and torch.equal(z, y)
    wide = normal(g, rows, heads * dh + 2 * dh, dtype=t)
    kept = wide.clone()
    part = wide[:, dh:dh + heads * dh].unflatten(1, (heads, dh))
    part.copy_(x)
    ops.rotary(part, freq, pos, layout=layout, mscale=m, out=part)
    assert torch.equal(part, y) and torch.equal(wide[:, :dh], kept[:, :dh]) and torch.equal(wide[:, (heads + 1) * dh:], kept[:, (heads + 1) * dh:])


def test_rotary_gradient_against_differences():
    g = gen(3)
    freq, _ = ops.rotary_frequencies(16, device=DEV)
    x, dy = normal(g, 5, 2, 16), normal(g, 5, 2, 16)
    pos = i32([0, 1, 17, 400, 70000])
    dx = ops.rotary(dy, freq, pos, inverse=True)
    f = lambda z: (turn(z, freq, pos)[0] * dy.double()).sum()
    for at in [(0, 0, 0), (1, 1, 3), (2, 0, 15), (3, 1, 8), (4, 0, 7)]:
        hi, lo = x.double().clone(), x.double().clone()
        hi[at] += 1e-4
        lo[at] -= 1e-4
        # linear in x: the difference quotient is the derivative up to its own rounding; dx up to the rotary bound
        assert abs(((f(hi) - f(lo)) / 2e-4 - dx[at].double()).item()) <= 1e-9 + 2.0 ** -20 * float(dy.abs().max())


def test_rotary_positions_from_rows():
    g = gen(4)
    freq, _ = ops.rotary_frequencies(32, device=DEV)
    x = normal(g, 21, 2, 32)
    assert torch.equal(ops.rotary(x, freq, pos0=5), ops.rotary(x, freq, i32(list(range(5, 26)))))
    assert torch.equal(ops.rotary(x, freq, pos0=9, period=7), ops.rotary(x, freq, i32([9 + r % 7 for r in range(21)])))
    assert ops.rotary(x[:0], freq).shape == (0, 2, 32)


# ---- the paged cache ---------------------------------------------------------------------------------------------------------
class Paged:
    """lengths, pages and index arrays of a ragged batch; the pool is larger than needed and full of NaN"""

    def __init__(self, g, new, ctx, hkv, dh, page, t, spare=3, fill=float('nan')):
        self.new, self.ctx, self.page = new, ctx, page
        wide = max(1, max(-(-c // page) for c in ctx))
        used = sum(-(-c // page) for c in ctx)
        order = torch.randperm(used + spare, generator=torch.Generator().manual_seed(sum(ctx))).tolist()
        rows, at = [], 0
        for c in ctx:
            n = -(-c // page)
            rows.append(order[at:at + n] + [-1] * (wide - n))
            at += n
        self.rows = rows
        self.table, self.ctx_len = i32(rows), i32(ctx)
        self.cu = i32([0] + list(np.cumsum(new)))
        self.tokens = sum(new)
        self.k_pages, self.v_pages = ops.paged_cache(used + spare, hkv, page, dh, t, DEV)
        self.k_pages.fill_(fill)
        self.v_pages.fill_(fill)
        # every token of the cache, dense: [ctx, hkv, dh] per sequence
        self.k = [normal(g, c, hkv, dh, dtype=t) for c in ctx]
        self.v = [normal(g, c, hkv, dh, dtype=t) for c in ctx]
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def index(self):
        return self.table, self.cu, self.ctx_len

    def put(self, upto=None):
        """the dense tokens into the pages with plain indexing"""
        for b, c in enumerate(self.ctx):
            c = c if upto is None else upto[b]
            for p in range(c):
                at, slot = self.rows[b][p // self.page], p % self.page
                self.k_pages[at, :, slot] = self.k[b][p]
                self.v_pages[at, :, :, slot] = self.v[b][p]
        return self


LENGTHS = {'single': ([1], [1]), 'steps': ([1] * 5, [1, 16, 17, 33, 100]), 'fresh': ([5, 64, 1, 130], [5, 64, 1, 130]),
           'ragged': ([3, 0, 1, 70, 0, 16, 9], [50, 20, 1, 131, 0, 16, 257]), 'edges': ([15, 16, 17, 31, 33], [63, 64, 65, 128, 97])}


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('lengths', list(LENGTHS))
@pytest.mark.parametrize('hkv,hq,dh,page,rot,layout', [(2, 4, 8, 16, 8, 'half'), (1, 3, 96, 32, 48, 'interleaved'), (3, 3, 72, 16, 36, 'half'),
                                                       (2, 2, 64, 64, 0, 'half'), (1, 8, 128, 16, 128, 'interleaved')])
def test_paged_append(dtype, lengths, hkv, hq, dh, page, rot, layout):
    t, g = TYPES[dtype], gen(7)
    new, ctx = LENGTHS[lengths]
    c = Paged(g, new, ctx, hkv, dh, page, t)
    packed = normal(g, c.tokens + 2, (hq + 2 * hkv) * dh, dtype=t)
    q, k, v = (x.unflatten(1, (-1, dh)) for x in packed.split([hq * dh, hkv * dh, hkv * dh], 1))
    before_k, before_v = c.k_pages.clone(), c.v_pages.clone()
    q_out = torch.full((c.tokens + 2, hq, dh), 7.0, dtype=t, device=DEV)
    freq = ops.rotary_frequencies(rot, device=DEV)[0] if rot else None
    got = ops.paged_append(k, v, c.k_pages, c.v_pages, *c.index(), q=q, freq=freq, layout=layout, mscale=1.25 if rot else 1.0, q_out=q_out, status=c.status)
    assert got is q_out and int(c.status) == 0
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(new, ctx)]).to(DEV)
    if rot:
        (wk, sk), (wq, sq) = (turn(x[:c.tokens], freq, pos, layout, 1.25) for x in (k, q))
    else:
        wk, wq = k[:c.tokens].double(), q[:c.tokens].double()
        sk, sq = wk.abs() * 0, wq.abs() * 0
    within(q_out[:c.tokens], wq, rot_bound(wq, sq, t), 'queries')
    assert (q_out[c.tokens:] == 7.0).all()                      # rows of no sequence
    seen_k, seen_v = torch.zeros_like(before_k, dtype=torch.bool), torch.zeros_like(before_v, dtype=torch.bool)
    at = 0
    for b, (m, n) in enumerate(zip(new, ctx)):
        for p in range(n - m, n):
            pg, slot = c.rows[b][p // page], p % page
            within(c.k_pages[pg, :, slot], wk[at], rot_bound(wk[at], sk[at], t), 'key')
            assert torch.equal(c.v_pages[pg, :, :, slot], v[at])
            seen_k[pg, :, slot] = True
            seen_v[pg, :, :, slot] = True
            at += 1
    bits = lambda x: x.view(torch.int16 if t == torch.bfloat16 else torch.int32)
    assert torch.equal(bits(c.k_pages)[~seen_k], bits(before_k)[~seen_k]) and torch.equal(bits(c.v_pages)[~seen_v], bits(before_v)[~seen_v])


def test_paged_append_in_place_of_a_packed_projection():
    """queries turned where they lie between the keys and values; queries that are the keys are refused"""
    t, g = torch.bfloat16, gen(89)
    c = Paged(g, [70, 5], [70, 40], 2, 64, 16, t)
    packed = normal(g, 75, 6 * 64, dtype=t)
    freq = ops.rotary_frequencies(64, device=DEV)[0]
    parts = lambda x: x.unflatten(1, (6, 64)).split([2, 2, 2], 1)
    q, k, v = parts(packed.clone())
    want = ops.paged_append(k, v, c.k_pages, c.v_pages, *c.index(), q=q, freq=freq)
    keys, values = c.k_pages.clone(), c.v_pages.clone()
    q, k, v = parts(packed)
    kept = k.clone(), v.clone()
    assert ops.paged_append(k, v, c.k_pages, c.v_pages, *c.index(), q=q, q_out=q, freq=freq) is q
    bits = lambda x: x.contiguous().view(torch.int16)
    assert torch.equal(q, want) and torch.equal(bits(keys), bits(c.k_pages)) and torch.equal(bits(values), bits(c.v_pages))
    assert torch.equal(k, kept[0]) and torch.equal(v, kept[1])
    for other in (k, v):
        with pytest.raises((ValueError, lib.NeurstLibError), match='apart'):
            ops.paged_append(k, v, c.k_pages, c.v_pages, *c.index(), q=other, q_out=other, freq=freq)
    square = torch.zeros(4, 2, 64, 64, dtype=t, device=DEV)      # page_size 64, dh 64: both pools have one shape
    with pytest.raises((ValueError, lib.NeurstLibError), match='apart'):
        ops.paged_append(k, v, square, square, i32([[0, 1], [2, 3]]), c.cu, c.ctx_len)
    assert torch.equal(k, kept[0]) and not square.any()


def attend(c, q, causal=True, scale=None):
    """fp64 result and the bound of the docstring"""
    dh, t = q.shape[2], q.dtype
    scale = dh ** -0.5 if scale is None else scale
    out, bound, at = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0
    for b, (m, n) in enumerate(zip(c.new, c.ctx)):
        if m and n:
            group = q.shape[1] // c.k[b].shape[1]
            k, v = (x.double().repeat_interleave(group, 1).permute(1, 0, 2) for x in (c.k[b], c.v[b]))
            x = q[at:at + m].double().permute(1, 0, 2)
            s = x @ k.transpose(1, 2) * scale
            if causal:
                s = s.masked_fill(torch.ones(m, n, dtype=torch.bool, device=DEV).triu(n - m + 1), float('-inf'))
            w = torch.softmax(s, -1)
            o, size = w @ v, w @ v.abs()
            dot = (x.abs() @ k.abs().transpose(1, 2)).amax() * abs(scale)
            rel = 2 * (dh + 8) * 2.0 ** -24 * dot + (n + 64) * 2.0 ** -23 + (half_step(t) if t == torch.bfloat16 else 0)
            out[at:at + m], bound[at:at + m] = o.permute(1, 0, 2), (size * rel * 1.01 + o.abs() * half_step(t) * 1.01).permute(1, 0, 2)
        at += m
    return out, bound + 1e-30


def crowded(c, q, how):
    """(queries, page table) that ask for the same at sizes of many products, where bf16 goes to the kernel for many rows: behind
    the last sequence more rows of no sequence ('rows': so many that the keys stay whole; 'split': with a table of 4096 keys)"""
    if not how:
        return q, c.table
    (B, wide), (_, hq, dh) = c.table.shape, q.shape
    table = c.table
    if how == 'split' and wide * c.page < 4096:
        table = torch.cat([table, torch.full((B, 4096 // c.page - wide), -1, dtype=torch.int32, device=DEV)], 1)
    rows = max(-(-(5 << 27) // (hq * table.shape[1] * c.page * dh)) + B, 33 * B)
    if how == 'rows':
        rows = max(rows, 512 * 128 * 2)
    more = torch.ones(max(0, rows - q.shape[0]), hq, dh, dtype=q.dtype, device=DEV)
    return torch.cat([torch.cat([q, more]).flatten(1), torch.ones(max(rows, q.shape[0]), 64, dtype=q.dtype, device=DEV)], 1)[:, :-64].unflatten(1, (hq, dh)), table


FORMS = [('fp32', ''), ('bf16', ''), ('bf16', 'rows'), ('bf16', 'split')]


@pytest.mark.parametrize('dtype,how', FORMS)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('lengths', list(LENGTHS))
@pytest.mark.parametrize('hkv,group,dh,page', [(2, 1, 8, 16), (1, 3, 96, 32), (3, 1, 72, 16), (2, 2, 64, 64), (1, 8, 128, 16), (1, 1, 192, 32),
                                               (1, 5, 256, 16), (2, 1, 32, 128)])
def test_paged_attention(dtype, how, causal, lengths, hkv, group, dh, page):
    t, g = TYPES[dtype], gen(11)
    new, ctx = LENGTHS[lengths]
    c = Paged(g, new, ctx, hkv, dh, page, t).put()
    q, c.table = crowded(c, normal(g, c.tokens + 3, hkv * group, dh, dtype=t), how)
    need = ops.paged_attention_workspace_bytes(q.shape[0], *c.table.shape, page, hkv * group, hkv, dh, ops.dt_of(q))
    if how == 'rows':
        assert 0 < need < 65536 * 4             # the order of the tiles, no parts
    elif how == 'split':
        assert need >= 2 * q.shape[0] * hkv * group * dh * 4
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, c.k_pages, c.v_pages, *c.index(), causal=causal, out=out, status=c.status)
    want, bound = attend(c, q[:c.tokens], causal)
    assert int(c.status) == 0
    within(out[:c.tokens], want, bound, 'attention')
    assert (out[c.tokens:] == 7.0).all()


@pytest.mark.parametrize('dtype,how', FORMS)
@pytest.mark.parametrize('new,ctx,hkv,group,dh,page', [([1, 1, 1], [3001, 17, 4096], 2, 4, 64, 16), ([1], [20000], 1, 1, 128, 64),
                                                       ([300, 1, 129], [1500, 900, 129], 2, 2, 64, 32), ([257, 700], [257, 1000], 1, 4, 128, 16),
                                                       ([1000], [1000], 2, 1, 96, 64), ([520, 3], [520, 2000], 1, 2, 192, 64),
                                                       ([260, 40], [300, 40], 1, 3, 256, 32), ([150] * 4, [333] * 4, 2, 1, 40, 16)])
def test_paged_attention_long(dtype, how, new, ctx, hkv, group, dh, page):
    """split contexts and chunks of many rows"""
    t, g = TYPES[dtype], gen(13)
    c = Paged(g, new, ctx, hkv, dh, page, t, fill=0.0)
    for b, n in enumerate(ctx):      # page by page
        for i in range(-(-n // page)):
            m = min(page, n - i * page)
            c.k_pages[c.rows[b][i], :, :m] = c.k[b][i * page:i * page + m].transpose(0, 1)
            c.v_pages[c.rows[b][i], :, :, :m] = c.v[b][i * page:i * page + m].permute(1, 2, 0)
    packed = normal(g, c.tokens, hkv * group * dh + 64, dtype=t)
    q = packed[:, 64:].unflatten(1, (-1, dh))
    many, c.table = crowded(c, q, how)
    for causal in (True, False):
        want, bound = attend(c, q, causal)
        within(ops.paged_attention(many, c.k_pages, c.v_pages, *c.index(), causal=causal)[:c.tokens], want, bound, 'causal %s' % causal)
    want, bound = attend(c, q, True, -0.3)
    within(ops.paged_attention(many, c.k_pages, c.v_pages, *c.index(), scale=-0.3)[:c.tokens], want, bound, 'scale')


@pytest.mark.parametrize('dtype,how', FORMS)
def test_contexts_shorter_than_the_chunk(dtype, how):
    """not causal: a chunk may be longer than what it attends to (a long prefix against few encoder states), or see nothing"""
    t, g = TYPES[dtype], gen(59)
    c = Paged(g, [40, 3, 90, 1], [5, 0, 64, 30], 2, 96, 16, t).put()
    q = normal(g, c.tokens, 4, 96, dtype=t)
    want, bound = attend(c, q, False)
    q, c.table = crowded(c, q, how)
    got = ops.paged_attention(q, c.k_pages, c.v_pages, *c.index(), causal=False, status=c.status)
    within(got[:c.tokens], want, bound)
    assert int(c.status) == 0 and (got[40:43] == 0).all()
    ops.paged_attention(q, c.k_pages, c.v_pages, *c.index(), causal=True, status=c.status)
    assert int(c.status) == 2


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dh', [32, 64])
def test_more_workgroups_than_run_at_once(causal, dh):
    """tiles of rows sorted by their work: ragged chunks of many heads, one sequence without tokens, one of a single token"""
    t, g = torch.bfloat16, gen(61)
    new, ctx = [300, 1, 0, 150, 129], [420, 77, 30, 150, 900]
    c = Paged(g, new, ctx, 40, dh, 32, t, fill=0.0)
    for b, n in enumerate(ctx):
        for i in range(-(-n // 32)):
            m = min(32, n - i * 32)
            c.k_pages[c.rows[b][i], :, :m] = c.k[b][i * 32:i * 32 + m].transpose(0, 1)
            c.v_pages[c.rows[b][i], :, :, :m] = c.v[b][i * 32:i * 32 + m].permute(1, 2, 0)
    q = normal(g, c.tokens + 5, 120, dh, dtype=t)
    out = torch.full_like(q, 7.0)
    wide = c.table.shape[1]
    assert ops.paged_attention_workspace_bytes(c.tokens + 5, 5, wide, 32, 120, 40, dh, lib.BF16) < (c.tokens + 5) * 120 * 4      # the order, no parts
    ops.paged_attention(q, c.k_pages, c.v_pages, *c.index(), causal=causal, out=out, status=c.status)
    want, bound = attend(c, q[:c.tokens], causal)
    within(out[:c.tokens], want, bound)
    assert (out[c.tokens:] == 7.0).all() and int(c.status) == 0


@pytest.mark.parametrize('dtype,how', FORMS)
@pytest.mark.parametrize('n,dh', [(40, 64), (200, 96), (300, 128)])
def test_masked_values_that_are_not_finite(dtype, how, n, dh):
    """a chunk whose later keys and values are inf and NaN: earlier queries do not see them, later ones do"""
    t, g = TYPES[dtype], gen(17)
    c = Paged(g, [n], [n + 20], 2, dh, 16, t)
    clean = [c.k[0].clone()], [c.v[0].clone()]
    first = n // 2 + 20
    c.v[0][first, :, 1] = float('inf')
    c.v[0][first + 3] = float('nan')
    c.k[0][first + 1] = float('nan')
    c.put()
    q = normal(g, n, 2, dh, dtype=t)
    many, c.table = crowded(c, q, how)
    got = ops.paged_attention(many, c.k_pages, c.v_pages, *c.index())[:n]
    c.k, c.v = clean
    want, bound = attend(c, q)
    cut = n // 2
    within(got[:cut], want[:cut], bound[:cut], 'before')
    assert torch.isinf(got[cut, :, 1]).all() and torch.isfinite(got[cut, :, 2:]).all()
    assert torch.isnan(got[cut + 3:]).all()


@pytest.mark.parametrize('dtype,n,wide,how', [('bf16', 1, 8192, ''), ('fp32', 1, 8192, ''), ('bf16', 20, 8192, ''), ('bf16', 40, 4096, 'split'),
                                              ('bf16', 40, 1024, ''), ('fp32', 40, 1024, '')])
def test_what_is_not_finite_and_seen_reaches_the_result(dtype, n, wide, how):
    """a query, a key or a value that a row sees is NaN or infinite, wherever the keys are split and however little the value
    counts: the row is not finite, and others stay as they are"""
    t, g = TYPES[dtype], gen(83)
    hkv, dh, page, ctx = 2, 64, 16, 3000 if wide > 3000 else 900
    c = Paged(g, [n], [ctx], hkv, dh, page, t, fill=0.0)
    c.k_pages.copy_(normal(g, *c.k_pages.shape)), c.v_pages.copy_(normal(g, *c.v_pages.shape))
    c.table = torch.cat([c.table, torch.full((1, wide // page - c.table.shape[1]), -1, dtype=torch.int32, device=DEV)], 1)
    q = normal(g, n, hkv, dh, dtype=t)
    q[:, :, 0] = 1.0
    far = 700                                                  # one key that counts for nothing, in fp32 exactly
    c.k_pages[c.rows[0][far // page], :, far % page] = 0.0
    c.k_pages[c.rows[0][far // page], :, far % page, 0] = -2.0 ** 14
    many, c.table = crowded(c, q, how)
    need = ops.paged_attention_workspace_bytes(many.shape[0], *c.table.shape, page, hkv, hkv, dh, ops.dt_of(q))
    assert (need >= 2 * many.shape[0] * hkv * dh * 4) == (wide > 1024)
    run = lambda: ops.paged_attention(many, c.k_pages, c.v_pages, *c.index())[:n]
    good = run()
    assert torch.isfinite(good).all()
    bad = many.clone()
    bad[0, 1, 5] = float('nan')
    got = ops.paged_attention(bad, c.k_pages, c.v_pages, *c.index())[:n]
    assert torch.isnan(got[0, 1]).all() and torch.equal(got[0, 0], good[0, 0]) and torch.equal(got[1:], good[1:])
    for at in (3, 600, far, ctx - n):
        pg, slot = c.rows[0][at // page], at % page
        for value in (float('nan'), float('inf'), -float('inf')):
            if at != far and value != value:
                kept = c.k_pages[pg, 0, slot].clone()
                c.k_pages[pg, 0, slot, 7] = value
                got = run()
                assert torch.isnan(got[:, 0]).all() and torch.equal(got[:, 1], good[:, 1]), ('key', at)
                c.k_pages[pg, 0, slot] = kept
            kept = c.v_pages[pg, 1, 9, slot].clone()
            c.v_pages[pg, 1, 9, slot] = value
            got = run()
            assert not torch.isfinite(got[:, 1, 9]).any(), ('value', at, value)
            rest = torch.arange(dh, device=DEV) != 9
            assert torch.equal(got[:, 0], good[:, 0]) and torch.equal(got[:, 1, rest], good[:, 1, rest]), ('value', at, value)
            c.v_pages[pg, 1, 9, slot] = kept
    # a part whose only keys are NaN
    pages = c.rows[0][512 // page:1024 // page if wide > 1024 else 800 // page]
    kept = c.k_pages[pages].clone()
    c.k_pages[pages] = float('nan')
    assert torch.isnan(run()).all()
    c.k_pages[pages] = kept
    assert torch.equal(run(), good)


def test_pages_shared_by_sequences():
    """hypotheses of one utterance against the same pages, and one key page for every position"""
    t, g = torch.bfloat16, gen(19)
    c = Paged(g, [1], [50], 2, 64, 16, t).put()
    table, ctx, cu = c.table.expand(6, -1), i32([50, 50, 50, 33, 1, 50]), i32([0, 1, 2, 4, 5, 6, 9])
    q = normal(g, 9, 2, 64, dtype=t)
    got = ops.paged_attention(q, c.k_pages, c.v_pages, table, cu, ctx, causal=False)
    again = ops.paged_attention(q, c.k_pages, c.v_pages, table.contiguous(), cu, ctx, causal=False)
    assert torch.equal(got, again)
    c.new, c.ctx = [1, 1, 2, 1, 1, 3], [50, 50, 50, 33, 1, 50]
    c.k, c.v = [c.k[0][:n] for n in c.ctx], [c.v[0][:n] for n in c.ctx]
    want, bound = attend(c, q, False)
    within(got, want, bound)
    one = i32([[c.rows[0][0]] * 4])
    c.new, c.ctx, c.k, c.v = [1], [64], [c.k[0][:16].repeat(4, 1, 1)], [c.v[0][:16].repeat(4, 1, 1)]
    want, bound = attend(c, q[:1])
    within(ops.paged_attention(q[:1], c.k_pages, c.v_pages, one, i32([0, 1]), i32([64])), want, bound)


@pytest.mark.parametrize('n,how', [(1, ''), (40, ''), (200, ''), (1, 'rows'), (40, 'rows'), (200, 'rows'), (40, 'split'), (200, 'split')])
def test_bad_pages_and_lengths_are_left_out(n, how):
    """the index arithmetic's own test runs on the CPU; here the kernels keep to it and report"""
    t, g = torch.bfloat16, gen(23)
    hkv, dh, page = 2, 64, 16
    c = Paged(g, [n, n, n], [n + 40, n + 40, n + 40], hkv, dh, page, t).put()
    q = normal(g, 3 * n, hkv, dh, dtype=t)
    many, c.table = crowded(c, q, how)
    good = ops.paged_attention(many, c.k_pages, c.v_pages, *c.index(), status=c.status)
    ops.paged_check(c.status)
    table = c.table.clone()
    table[1, 1] = 10 ** 6
    got = ops.paged_attention(many, c.k_pages, c.v_pages, table, c.cu, c.ctx_len, status=c.status)
    assert int(c.status) == 1 and torch.equal(got[:n], good[:n]) and torch.equal(got[2 * n:3 * n], good[2 * n:3 * n])
    d = Paged(g, [n], [n + 40 - page], hkv, dh, page, t)         # the same without the page's keys: later queries, not causal
    d.k, d.v = [torch.cat([c.k[1][:page], c.k[1][2 * page:]])], [torch.cat([c.v[1][:page], c.v[1][2 * page:]])]
    want, bound = attend(d, q[n:2 * n], False)
    within(ops.paged_attention(many, c.k_pages, c.v_pages, table, c.cu, c.ctx_len, causal=False)[n:2 * n], want, bound)
    with pytest.raises(lib.NeurstLibError, match='page id'):
        ops.paged_check(c.status)
    for ctx in ([n + 40, n - 1, n + 40], [n + 40, 10 ** 9, n + 40], [n + 40, -5, n + 40]):
        c.status.zero_()
        got = ops.paged_attention(many, c.k_pages, c.v_pages, c.table, c.cu, i32(ctx), status=c.status)
        assert int(c.status) == 2 and torch.equal(got[:n], good[:n]) and torch.equal(got[2 * n:3 * n], good[2 * n:3 * n])
        assert (got[n:2 * n] == 0).all()
    kp, vp = c.k_pages.clone(), c.v_pages.clone()
    k = normal(g, 3 * n, hkv, dh, dtype=t)
    for tab, cu, ctx, want_status in ((table * 0 - 1, c.cu, c.ctx_len, 1), (c.table, i32([0, 5, 3 * n + 1, 2]), c.ctx_len, 2),
                                      (c.table, c.cu, i32([n - 1, 0, -1]), 2)):
        c.status.zero_()
        ops.paged_append(k, k, kp, vp, tab, cu, ctx, status=c.status)
        assert int(c.status) & want_status
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))
    if n > 5:       # of the three calls the second may write its one fitting sequence, rows 0 .. 4
        assert same(c.v_pages[c.rows[1][0]], vp[c.rows[1][0]])
    else:
        assert same(c.k_pages, kp) and same(c.v_pages, vp)


@pytest.mark.parametrize('n,how', [(1, ''), (40, ''), (40, 'rows'), (40, 'split')])
def test_lengths_that_no_tile_leads_to_are_reported(n, how):
    """all rows past the tensors: no workgroup finds a sequence, the status tells all the same; correct lengths leave it zero"""
    t, g = torch.bfloat16, gen(73)
    hkv, dh, page = 2, 64, 16
    c = Paged(g, [n, n, n], [n + 40, n + 40, n + 40], hkv, dh, page, t).put()
    q, c.table = crowded(c, normal(g, 3 * n, hkv, dh, dtype=t), how)
    tokens = q.shape[0]
    k = normal(g, 3 * n, hkv, dh, dtype=t)
    bits = lambda x: x.view(torch.int16)
    kp, vp = c.k_pages.clone(), c.v_pages.clone()
    for cu in ([tokens + 1] * 4, [2 ** 31 - 1] * 4, [tokens + 5, tokens + 6, tokens + 7, tokens + 9]):
        for causal in (True, False):
            c.status.zero_()
            out = torch.full_like(q, 7.0)
            ops.paged_attention(q, kp, vp, c.table, i32(cu), c.ctx_len, causal=causal, out=out, status=c.status)
            assert int(c.status) == 2 and (out == 7.0).all(), cu
        c.status.zero_()
        ops.paged_append(k, k, kp, vp, c.table, i32(cu), c.ctx_len, status=c.status)
        assert int(c.status) == 2 and torch.equal(bits(kp), bits(c.k_pages)) and torch.equal(bits(vp), bits(c.v_pages)), cu
    c.status.zero_()
    ops.paged_attention(q, kp, vp, *c.index(), status=c.status)
    ops.paged_append(k, k, kp, vp, *c.index(), status=c.status)
    ops.paged_check(c.status)
    with pytest.raises(lib.NeurstLibError, match='lengths'):
        ops.paged_check(c.status.fill_(2))


@pytest.mark.parametrize('dtype,n,how', [('bf16', 1, ''), ('bf16', 40, ''), ('fp32', 40, ''), ('bf16', 40, 'rows'), ('bf16', 40, 'split'),
                                         ('bf16', 1, 'long'), ('bf16', 40, 'long'), ('fp32', 1, 'long'), ('fp32', 40, 'long')])
def test_rows_of_refused_sequences_stay_as_they_are(dtype, n, how):
    """cu_new that does not fit, with whole keys and with parts of them, whatever the workspace holds ('long': the kernel for few
    rows over a table of 8192 keys)"""
    t, g = TYPES[dtype], gen(79)
    hkv, dh, page = 2, 64, 16
    c = Paged(g, [n, n, n], [n + 40, n + 40, n + 40], hkv, dh, page, t).put()
    q = normal(g, 3 * n, hkv, dh, dtype=t)
    if how == 'long':
        c.table = torch.cat([c.table, torch.full((3, 8192 // page - c.table.shape[1]), -1, dtype=torch.int32, device=DEV)], 1)
    else:
        q, c.table = crowded(c, q, how)
    tokens, far = q.shape[0], 2 ** 30
    need = ops.paged_attention_workspace_bytes(tokens, 3, c.table.shape[1], page, hkv, hkv, dh, ops.dt_of(q))
    parts = need >= 2 * tokens * hkv * dh * 4
    assert parts == (how in ('split', 'long'))
    ws = torch.empty(max(need, 16) // 4, device=DEV)

    def attend_with(cu):
        ws.fill_(3.0)
        c.status.zero_()
        out = torch.full_like(q, 7.0)
        ops.paged_attention(q, c.k_pages, c.v_pages, c.table, i32(cu), c.ctx_len, out=out, status=c.status, workspace=ws)
        return out

    good = attend_with([0, n, 2 * n, 3 * n])
    assert int(c.status) == 0 and (good[3 * n:] == 7.0).all()
    for cu, kept in (([0, n, far, 3 * n], [(0, n)]), ([-5, n, 2 * n, 3 * n], [(n, 3 * n)]), ([0, n, 2 * n, far], [(0, 2 * n)]),
                     ([0, n, tokens + 1, 3 * n], [(0, n)])):
        got = attend_with(cu)
        want = torch.full_like(q, 7.0)
        for a, b in kept:
            want[a:b] = good[a:b]
        assert int(c.status) == 2 and torch.equal(got, want), cu


def test_offsets_beyond_32_bits():
    """the pool holds more than 2^32 elements; the sequence's pages lie at its end"""
    t, g = torch.bfloat16, gen(29)
    hkv, dh, page = 8, 128, 64
    n_pages = (1 << 32) // (hkv * dh * page) + 40
    k_pages, v_pages = ops.paged_cache(n_pages, hkv, page, dh, t, DEV)
    c = Paged(g, [70], [150], hkv, dh, page, t, fill=0.0)
    table = i32([[n_pages - 1, 5, n_pages - 7]])
    old = i32([0, 80]), i32([80])
    ops.paged_append(c.k[0][:80], c.v[0][:80], k_pages, v_pages, table, *old)
    ops.paged_append(c.k[0][80:], c.v[0][80:], k_pages, v_pages, table, c.cu, c.ctx_len)
    assert torch.equal(k_pages[n_pages - 1], c.k[0][:64].transpose(0, 1)) and torch.equal(v_pages[n_pages - 7, :, :, :22], c.v[0][128:].permute(1, 2, 0))
    q = normal(g, 70, hkv, dh, dtype=t)
    want, bound = attend(c, q)
    for how in ('', 'rows'):
        c.table = table
        many, wide = crowded(c, q, how)
        within(ops.paged_attention(many, k_pages, v_pages, wide, c.cu, c.ctx_len)[:70], want, bound, how)
    del k_pages, v_pages
    torch.cuda.empty_cache()


# ---- sampling ------------------------------------------------------------------------------------------------------------------
def choose(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """one row, numpy fp64 -> (id, logp, bound on logp)"""
    f = lambda v: float(np.float32(v))
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    if not (x > -np.inf).any():
        return -1, -np.inf, 0.0
    if temperature <= 0:
        temperature, top_k = 1.0, 1
    order = np.lexsort((np.arange(x.size), -x))
    order = order[:top_k] if top_k else order
    with np.errstate(invalid='ignore', over='ignore'):
        w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / f(temperature)))
    w = np.rint(w * 2.0 ** 44).astype(np.int64)                  # whole multiples of 2^-44: what is below half of one is never drawn
    if f(top_p) < 1:
        cut = int(np.searchsorted(np.cumsum(w), math.ceil(f(top_p) * float(w.sum())))) + 1
        order, w = order[:cut], w[:cut]
    keep = w >= f(min_p) * 2.0 ** 44
    order, w = order[keep], w[keep]
    back = np.argsort(order)
    order, w = order[back], w[back]
    sums = np.cumsum(w)
    at = min(int(np.searchsorted(sums, math.floor(f(u) * float(sums[-1])), side='right')), int(np.searchsorted(sums, sums[-1])))
    lp = math.log(int(w[at]) / int(sums[-1]))
    return int(order[at]), lp, abs(lp) * 2.0 ** -24 + 1.0 / int(w[at]) + w.size / int(sums[-1]) + 1e-12


def check_rows(logits, u, got, **par):
    ids, logp = got
    x, uu = logits.float().cpu().numpy(), u.cpu().numpy()
    for r in range(x.shape[0]):
        row = {k: (float(v[r]) if k != 'top_k' else int(v[r])) if torch.is_tensor(v) else v for k, v in par.items()}
        want, lp, bound = choose(x[r], uu[r], **row)
        assert int(ids[r]) == want, (r, int(ids[r]), want, row)
        assert float(logp[r]) == lp or abs(float(logp[r]) - lp) <= bound, (r, float(logp[r]), lp, bound)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('V', [1, 2, 63, 300, 4096, 4097, 10000, 32003, 70001])
@pytest.mark.parametrize('par', [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
                                 dict(temperature=0.7, top_k=50, top_p=0.8, min_p=0.01), dict(temperature=5.0, top_p=0.3), dict(temperature=0.01, top_p=0.99),
                                 dict(top_k=10 ** 9, top_p=1e-6), dict(min_p=1.0)])
def test_sample(dtype, V, par):
    g = gen(V)
    R = 12 if V < 20000 else 4
    x = (3 * torch.randn(R, V, generator=g, device=DEV)).to(TYPES[dtype])
    if V > 4:
        x[1] = x[1].round()                                        # many ties
        x[2].masked_fill_(torch.rand(V, generator=g, device=DEV) < 0.6, float('-inf'))
        x[3] = 2.5                                                 # nothing but ties
    u = torch.rand(R, generator=g, device=DEV)
    u[0] = 0.0
    check_rows(x, u, ops.sample(x, u, **par), **par)


def test_sample_many_rows():
    """rows that share a CU: fewer threads a row"""
    g = gen(71)
    x, u = 3 * normal(g, 520, 6001), torch.rand(520, generator=g, device=DEV)
    for par in (dict(top_p=0.9), dict(top_k=300, top_p=0.95, min_p=0.01), dict(top_k=1)):
        check_rows(x, u, ops.sample(x, u, **par), **par)


def test_sample_odd_rows():
    """rows with nothing to draw, infinities, NaN, the type's lowest value, signed zeros, a step between neighbours"""
    V = 501
    low, inf, nan = torch.finfo(torch.float32).min, float('inf'), float('nan')
    rows = []

    def at(base, **kv):
        x = torch.full((V,), base)
        for k, v in kv.items():
            x[int(k[1:])] = v
        return x
    rows = [at(-inf), at(nan), at(-inf, i7=nan), at(-inf, i7=-3.0), at(nan, i9=1.0, i3=1.0), at(low), at(low, i100=low), at(low, i5=0.0, i6=0.0),
            at(0.0, i50=inf), at(0.0, i50=inf, i60=inf, i70=-inf), at(-0.0, i3=0.0), at(0.0, i0=-0.0, i4=-0.0), at(1.0, i250=1.0 + 2.0 ** -23),
            at(3e38, i1=-3e38), at(-200.0, i400=0.0), torch.linspace(-40, 0, V), torch.linspace(0, 1e-4, V), 1e-38 * torch.arange(V), -torch.arange(V).float() ** 3]
    x = torch.stack(rows).to(DEV)
    for u in (0.0, 0.25, 0.5, 0.999, 1 - 2.0 ** -24):
        uu = torch.full((x.shape[0],), u, device=DEV)
        for par in (dict(), dict(top_k=1), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.5), dict(top_k=250, top_p=0.7), dict(min_p=0.5), dict(top_k=2, min_p=1.0)):
            check_rows(x, uu, ops.sample(x, uu, **par), **par)
        tiny = 2.0 ** -133 * torch.arange(V, device=DEV)[None]      # denormal steps at the smallest normal temperature
        for par in (dict(), dict(top_p=0.5), dict(top_k=9, top_p=0.5), dict(min_p=0.5)):
            check_rows(tiny, uu[:1], ops.sample(tiny, uu[:1], temperature=2.0 ** -126, **par), temperature=2.0 ** -126, **par)
    # u outside [0, 1) is brought inside
    assert ops.sample(x[6:7], torch.ones(1, device=DEV))[0].item() == V - 1
    assert ops.sample(x[6:7], torch.full((1,), nan, device=DEV))[0].item() == 0


def raised_rows(V, k, t, rows=4):
    """rows with k words 0.035 to 0.05 above a plateau of all others, every one of the k read by a lane of its own, so that
    they fill a step of the kernel's histogram (1 / 32 at temperature 1) and the plateau the one or two behind it"""
    nw, e = (16 if V > 4096 else 4), 128 // torch.finfo(t).bits
    own = -(-V // (nw * 64)) * 64                              # words of a wave
    if -(-V // (nw * 64)) * nw * 64 * torch.finfo(t).bits // 8 > 132 * 1024:
        e = 1                                                  # rows read again from memory: a lane reads single words
    i = torch.arange(k)
    at = (i % nw) * own + (i // nw) * e
    assert int(at.max()) < V and k // nw < 64
    x = torch.zeros(rows, V)
    x[:, at] = 0.05 - 0.015 * (torch.arange(k) % 7) / 7.0
    x[1::2] += 1.0                                             # bf16: coarser there, all of them one value
    return x.to(t).to(DEV)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('V', [3001, 5000, 32003, 70001])
@pytest.mark.parametrize('k', [2, 8, 40, 200])
def test_sample_top_k_ends_before_a_plateau(dtype, V, k):
    """exactly k words lie in the steps that can hold the k-th, and more words than a list takes right behind them"""
    x = raised_rows(V, k, TYPES[dtype])
    for u in (0.0, 0.3, 0.6, 0.95):
        uu = torch.full((x.shape[0],), u, device=DEV)
        for par in (dict(), dict(min_p=0.5), dict(top_p=0.9), dict(top_p=0.5, min_p=0.97)):
            par = dict(par, top_k=k)
            check_rows(x, uu, ops.sample(x, uu, **par), **par)
    R = x.shape[0]
    preds = torch.zeros(R, 1, dtype=torch.int32, device=DEV)
    tokens, fin, ln, left = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (R, R, R, 1))
    scores, uu = torch.zeros(R, device=DEV), torch.linspace(0.1, 0.9, R, device=DEV)
    ops.sample_step(x, uu, tokens, preds, fin, ln, left, scores, 0, V - 1, top_k=k, top_p=0.9)
    check_rows(x, uu, (tokens, scores), top_k=k, top_p=0.9)
    assert torch.equal(preds[:, 0], tokens) and int(left) == R


def test_sample_parameters_per_row_and_strides():
    g = gen(31)
    R, V = 40, 1000
    wide = 3 * torch.randn(R, V + 77, generator=g, device=DEV)
    x, u = wide[:, 5:5 + V], torch.rand(R, generator=g, device=DEV)
    par = dict(temperature=torch.rand(R, generator=g, device=DEV) * 2, top_k=torch.randint(0, 60, (R,), generator=g, device=DEV, dtype=torch.int32),
               top_p=torch.rand(R, generator=g, device=DEV).clamp(min=0.01), min_p=torch.rand(R, generator=g, device=DEV) * 0.1)
    par['temperature'][0] = 0.0
    got = ops.sample(x, u, **par)
    check_rows(x, u, got, **par)
    odd = dict(temperature=torch.full((R,), -1.0, device=DEV), top_k=torch.full((R,), -3, device=DEV, dtype=torch.int32),
               top_p=torch.full((R,), float('nan'), device=DEV), min_p=torch.full((R,), float('nan'), device=DEV))
    assert torch.equal(ops.sample(x, u, **odd)[0].long(), x.argmax(1))
    # the draw does not depend on the launch: rows alone, and copied to other places
    one = torch.cat([ops.sample(x[r:r + 1].clone(), u[r:r + 1], **{k: v[r:r + 1] for k, v in par.items()})[0] for r in range(R)])
    assert torch.equal(one, got[0])


def test_sample_frequencies():
    """20000 draws of one row: counts within six standard deviations of the exact probabilities"""
    g = gen(37)
    x = torch.randn(1, 40, generator=g, device=DEV)
    n = 20000
    u = (torch.arange(n, device=DEV) + 0.5) / n                   # an even grid: counts within one of n p
    ids, logp = ops.sample(x.expand(n, -1).contiguous(), u)
    p = torch.softmax(x[0].double(), 0)
    counts = torch.bincount(ids.long(), minlength=40)
    assert ((counts - n * p).abs() <= 1.0 + 1e-6 * n).all()
    assert (logp.double() - torch.log(p)[ids.long()]).abs().max() <= 2.0 ** -22 * 8


def test_sample_step_keeps_the_books():
    g = gen(41)
    R, V, eos, steps = 9, 50, 3, 6
    x = torch.randn(R, V, generator=g, device=DEV)
    x[:, eos] += 3.0
    x[4] = float('-inf')
    preds = torch.zeros(R, steps, dtype=torch.int32, device=DEV)
    tokens, fin, ln = (torch.zeros(R, dtype=torch.int32, device=DEV) for _ in range(3))
    scores, left = torch.zeros(R, device=DEV), torch.zeros(steps, dtype=torch.int32, device=DEV)
    pf, pl, ps = np.zeros(R, int), np.zeros(R, int), np.zeros(R)
    for s in range(steps):
        u = torch.rand(R, generator=g, device=DEV)
        ids, logp = (t.cpu().numpy() for t in ops.sample(x, u, temperature=1.3))
        ops.sample_step(x, u, tokens, preds, fin, ln, left[s:s + 1], scores, s, eos, temperature=1.3)
        tok = np.where((pf > 0) | (ids < 0), eos, ids)
        ps = ps + np.where((pf == 0) & (ids >= 0), logp, 0)
        pf = pf | (tok == eos)
        pl = pl + 1 - pf
        assert (tokens.cpu().numpy() == tok).all() and (preds[:, s].cpu().numpy() == tok).all()
        assert (fin.cpu().numpy() == pf).all() and (ln.cpu().numpy() == pl).all() and int(left[s]) == int((pf == 0).sum())
    np.testing.assert_allclose(scores.cpu().numpy(), ps, rtol=0, atol=steps * 2.0 ** -22 * 8)


def test_sample_step_tells_of_rows_with_nothing_to_draw():
    """an unfinished row of NaN and -inf raises the status, a finished one does not; the books are the same without it"""
    R, V, eos = 6, 70, 3
    x = normal(gen(97), R, V)
    u = torch.full((R,), 0.5, device=DEV)

    def step(x, done, status):
        preds, left = torch.zeros(R, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        tokens, ln = (torch.zeros(R, dtype=torch.int32, device=DEV) for _ in range(2))
        fin, scores = i32([int(r in done) for r in range(R)]), torch.zeros(R, device=DEV)
        ops.sample_step(x, u, tokens, preds, fin, ln, left, scores, 0, eos, status=status)
        return tokens, preds, fin, ln, left, scores
    for value in (float('nan'), -float('inf')):
        bad = x.clone()
        bad[4] = value
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        for logits, done, bits in ((x, (), 0), (x, (1,), 0), (bad, (4,), 0), (bad, (), 4)):
            status.zero_()
            got = step(logits, done, status)
            assert int(status) == bits, (value, done)
            assert all(torch.equal(a, b) for a, b in zip(got, step(logits, done, None)))
        with pytest.raises(lib.NeurstLibError, match='nothing to draw'):
            ops.paged_check(status)
    with pytest.raises(ValueError, match='status'):
        step(x, (), torch.zeros(2, dtype=torch.int32, device=DEV))


# ---- a run of them together --------------------------------------------------------------------------------------------------------
def decode_run(g, dtype, steps=5, graph=False):
    """a forced prefix for three sequences, then single tokens: rotary -> append -> attention -> logits -> draw, against the
    same on dense fp64 tensors with the drawn tokens fed back"""
    t = TYPES[dtype]
    B, H, Hk, dh, V, page = 3, 4, 2, 32, 97, 16
    d = H * dh
    emb, w = normal(g, V, (H + 2 * Hk) * dh, dtype=t), 0.3 * normal(g, d, V)
    prefix = [5, 20, 1]
    freq, _ = ops.rotary_frequencies(dh, device=DEV)
    n_pages = B * 3
    k_pages, v_pages = ops.paged_cache(n_pages, Hk, page, dh, t, DEV)
    table = torch.arange(n_pages, device=DEV, dtype=torch.int32).view(B, 3)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    tokens = [torch.randint(0, V, (n,), generator=g, device=DEV) for n in prefix]
    us = torch.rand(steps, B, generator=g, device=DEV)
    drawn = torch.zeros(B, dtype=torch.int32, device=DEV)
    rows = [[emb[x] for x in seq] for seq in tokens]
    outs = []

    def step(x, cu, ctx, u):
        q, k, v = (z.unflatten(1, (-1, dh)) for z in x.split([d, Hk * dh, Hk * dh], 1))
        q = ops.paged_append(k, v, k_pages, v_pages, table, cu, ctx, q=q, freq=freq, status=status)
        o = ops.paged_attention(q, k_pages, v_pages, table, cu, ctx, status=status)
        last = o.view(-1, d)[cu[1:].long() - 1].float()
        logits = last @ w
        return o, logits, ops.sample(logits, u, temperature=0.9, top_k=30, top_p=0.95)

    cu = i32([0] + list(np.cumsum(prefix)))
    ctx = i32(prefix)
    x = emb[torch.cat(tokens)]
    for s in range(steps):
        o, logits, (ids, logp) = step(x, cu, ctx, us[s])
        outs.append((x, o, logits, ids, logp, cu.clone(), ctx.clone()))
        check_rows(logits, us[s], (ids, logp), temperature=0.9, top_k=30, top_p=0.95)
        x = emb[ids.long()]
        cu = i32([0, 1, 2, 3])
        ctx = ctx + 1
    ops.paged_check(status)
    # dense
    hist = [None] * B
    for x, o, logits, ids, logp, cu, ctx in outs:
        c = type('C', (), {})()
        cuh = cu.tolist()
        c.new, c.ctx, c.k, c.v = [b - a for a, b in zip(cuh, cuh[1:])], ctx.tolist(), [], []
        qs = []
        for b in range(B):
            part = x[cuh[b]:cuh[b + 1]]
            hist[b] = part if hist[b] is None else torch.cat([hist[b], part])
            pos = torch.arange(hist[b].shape[0], device=DEV)
            q, k, v = (z.unflatten(1, (-1, dh)) for z in hist[b].split([d, Hk * dh, Hk * dh], 1))
            # rounded as the operators round them; a half-step decided the other way is inside the bound below
            qs.append(turn(q, freq, pos)[0].to(t)[-c.new[b]:])
            c.k.append(turn(k, freq, pos)[0].to(t))
            c.v.append(v)
        want, bound = attend(c, torch.cat(qs))
        # rotated queries and keys may differ from these by one step of their type: scores by 2 steps of sum |q k|
        slack = 4 * half_step(t) * max(float((q_.abs().float().amax() * k_.abs().float().amax() * dh ** 0.5)) for q_, k_ in zip(qs, c.k))
        size = max(float(v.abs().max()) for v in c.v)
        within(o, want, bound + 2 * slack * size, 'step')


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_a_decoding_run(dtype):
    decode_run(gen(43), dtype)


def test_replayed_graphs_and_other_streams():
    """two captured steps share nothing but the cache; replays with new inputs equal the eager results, also beside eager
    work and on another stream"""
    g = gen(47)
    t, B, H, dh, V, page = torch.bfloat16, 4, 4, 64, 300, 16
    n_pages = B * 80
    k_pages, v_pages = ops.paged_cache(n_pages, H, page, dh, t, DEV)
    k_pages.copy_(normal(g, *k_pages.shape)), v_pages.copy_(normal(g, *v_pages.shape))
    table = torch.randperm(n_pages, generator=g, device=DEV).int().view(B, 80)
    freq, _ = ops.rotary_frequencies(dh, device=DEV)
    cu = i32([0, 1, 2, 3, 4])
    w = normal(g, H * dh, V)

    class Step:
        def __init__(self):
            self.x, self.ctx, self.u = normal(g, B, 3 * H * dh, dtype=t), i32([900, 17, 1200, 400]), torch.rand(B, generator=g, device=DEV)

        def run(self):
            q, k, v = (z.unflatten(1, (H, dh)) for z in self.x.chunk(3, 1))
            q = ops.paged_append(k, v, k_pages, v_pages, table, cu, self.ctx, q=q, freq=freq)
            o = ops.paged_attention(q, k_pages, v_pages, table, cu, self.ctx)
            y = ops.rotary(o, freq, self.ctx, out=torch.empty_like(o))
            return o, y, ops.sample(y.view(B, -1).float() @ w, self.u, top_p=0.9)

    assert ops.paged_attention_workspace_bytes(B, B, 80, page, H, H, dh, lib.BF16) > 0       # the split form
    steps = [Step(), Step()]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for s in steps:
            s.run()
    torch.cuda.synchronize()
    for s in steps:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(s.run())
        graphs.append(gr)
    for r in range(4):
        for s in steps:
            s.x.copy_(normal(g, *s.x.shape))
            s.ctx.copy_(torch.randint(1, 1280, (B,), generator=g, device=DEV, dtype=torch.int32))
            s.u.copy_(torch.rand(B, generator=g, device=DEV))
        want, cache = [], (k_pages.clone(), v_pages.clone())
        order = (0, 1) if r % 2 else (1, 0)
        for k in order:
            want.append([z.clone() for z in (lambda a: [a[0], a[1], *a[2]])(steps[k].run())])
        torch.cuda.synchronize()
        k_pages.copy_(cache[0]), v_pages.copy_(cache[1])     # the steps write the cache they read
        for k in order:
            graphs[k].replay()
            normal(g, 100)                                   # eager work between the replays
        torch.cuda.synchronize()
        for k, w_ in zip(order, want):
            got = [outs[k][0], outs[k][1], *outs[k][2]]
            assert all(torch.equal(a, b) for a, b in zip(got, w_)), (r, k)
    with torch.cuda.stream(side):
        got = steps[1].run()
    side.synchronize()
    assert torch.equal(got[0], want[1][0])


@pytest.mark.parametrize('how', ['', 'rows', 'split'])
def test_captured_chunks_follow_the_lengths(how):
    """one capture, replays with other lengths and contents beside eager work: two chunks' writes and attention, a workspace
    of the caller's that both calls of the graph use in turn"""
    t, g = torch.bfloat16, gen(67)
    hkv, hq, dh, page = 2, 4, 64, 32
    c = Paged(g, [150, 70, 1], [400, 70, 90], hkv, dh, page, t, fill=0.0, spare=40)
    wide = torch.arange(3 * 16, dtype=torch.int32, device=DEV).view(3, 16)         # 512 keys each
    c.k_pages, c.v_pages = ops.paged_cache(48, hkv, page, dh, t, DEV)
    c.k_pages.copy_(normal(g, *c.k_pages.shape)), c.v_pages.copy_(normal(g, *c.v_pages.shape))
    c.table = wide
    q, table = crowded(c, normal(g, 300, hq, dh, dtype=t), how)
    k, v = normal(g, q.shape[0], hkv, dh, dtype=t), normal(g, q.shape[0], hkv, dh, dtype=t)
    need = ops.paged_attention_workspace_bytes(q.shape[0], *table.shape, page, hq, hkv, dh, lib.BF16)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    cu, ctx = c.cu.clone(), c.ctx_len.clone()
    outs = [torch.full_like(q, 7.0) for _ in range(2)]

    def run():
        ops.paged_append(k, v, c.k_pages, c.v_pages, table, cu, ctx, status=c.status)
        for causal, o in zip((True, False), outs):
            ops.paged_attention(q, c.k_pages, c.v_pages, table, cu, ctx, causal=causal, out=o, status=c.status, workspace=ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for new, upto in (([150, 70, 1], [400, 70, 90]), ([1, 1, 1], [512, 1, 33]), ([0, 300, 0], [5, 301, 0]), ([100, 0, 200], [100, 64, 500])):
        q[:300].copy_(normal(g, 300, hq, dh)), k.copy_(normal(g, *k.shape)), v.copy_(normal(g, *v.shape))
        cu.copy_(i32([0] + list(np.cumsum(new)))), ctx.copy_(i32(upto))
        for o in outs:
            o.fill_(7.0)
        run()
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        normal(g, 100)
        torch.cuda.synchronize()
        assert int(c.status) == 0 and all(torch.equal(o, w) for o, w in zip(outs, want)), new
        assert all((o[sum(new):] == 7.0).all() and not (o[:sum(new)] == 7.0).all() for o in outs)


def test_two_streams_at_once():
    """attention and sampling on two streams at the same time have workspaces of their own"""
    g = gen(53)
    t = torch.bfloat16
    cs = [Paged(g, [1] * 3, [2000, 1500, 900], 2, 64, 64, t, fill=0.0) for _ in range(2)]
    for c in cs:
        c.k_pages.copy_(normal(g, *c.k_pages.shape)), c.v_pages.copy_(normal(g, *c.v_pages.shape))
    qs = [normal(g, 3, 8, 64, dtype=t) for _ in cs]
    x, u = 3 * normal(g, 64, 10000), torch.rand(64, generator=g, device=DEV)
    want = [ops.paged_attention(q, c.k_pages, c.v_pages, *c.index()) for q, c in zip(qs, cs)]
    ids = ops.sample(x, u, top_k=40, top_p=0.9)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append((ops.paged_attention(qs[k], cs[k].k_pages, cs[k].v_pages, *cs[k].index()), ops.sample(x, u, top_k=40, top_p=0.9)[0]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, want[k]) and torch.equal(b, ids) for a, b in got[k])
