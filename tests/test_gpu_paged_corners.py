"""Corners of the paged decoder's operators that test_gpu_paged.py does not go to: the largest pages and batches, head widths that
fill a kernel's only in part, rows of logits closer than a step of the sampling's histogram, rows that begin anywhere, captured
draws, beam search with rotary positions.  Helpers, references and tolerances are those of test_gpu_paged.py."""
import numpy as np
import pytest
import torch

from neurst_amd import ops
from test_gpu_paged import DEV, FORMS, TYPES, Paged, attend, check_rows, crowded, gen, i32, normal, rot_bound, turn, within

pytestmark = pytest.mark.gpu


def pages_of(c):
    """the dense tokens into the pages, a page at a time"""
    for b, n in enumerate(c.ctx):
        for i in range(-(-n // c.page)):
            m = min(c.page, n - i * c.page)
            c.k_pages[c.rows[b][i], :, :m] = c.k[b][i * c.page:i * c.page + m].transpose(0, 1)
            c.v_pages[c.rows[b][i], :, :, :m] = c.v[b][i * c.page:i * c.page + m].permute(1, 2, 0)
    return c


@pytest.mark.parametrize('dtype,how', FORMS)
@pytest.mark.parametrize('page', [256, 1024, 4096])
def test_large_pages(dtype, how, page):
    t, g = TYPES[dtype], gen(page)
    new, ctx = [70, 1, 0, 200], [page + 100, 5000, 17, 200]
    c = Paged(g, new, ctx, 2, 64, page, t)
    q = normal(g, c.tokens, 4, 64, dtype=t)
    # the cache is written by the operator itself: all but the new tokens, then those
    k, v = (torch.cat([x[:n - m] for x, m, n in zip(y, new, ctx)]) for y in (c.k, c.v))
    old = [n - m for m, n in zip(new, ctx)]
    ops.paged_append(k, v, c.k_pages, c.v_pages, c.table, i32([0] + list(np.cumsum(old))), i32(old), status=c.status)
    k, v = (torch.cat([x[n - m:] for x, m, n in zip(y, new, ctx)]) for y in (c.k, c.v))
    ops.paged_append(k, v, c.k_pages, c.v_pages, *c.index(), status=c.status)
    for b, n in enumerate(ctx):
        for p in {0, n // 2, n - 1}:
            pg, slot = c.rows[b][p // page], p % page
            assert torch.equal(c.k_pages[pg, :, slot], c.k[b][p]) and torch.equal(c.v_pages[pg, :, :, slot], c.v[b][p])
    many, c.table = crowded(c, q, how)
    for causal in (True, False):
        want, bound = attend(c, q, causal)
        within(ops.paged_attention(many, c.k_pages, c.v_pages, *c.index(), causal=causal, status=c.status)[:c.tokens], want, bound, 'causal %s' % causal)
    assert int(c.status) == 0


@pytest.mark.parametrize('dtype,how', FORMS)
@pytest.mark.parametrize('dh', [16, 56, 88, 104, 120, 136, 184, 200, 248])
def test_head_widths_between_the_kernels(dtype, how, dh):
    t, g = TYPES[dtype], gen(dh)
    c = pages_of(Paged(g, [65, 1, 40], [65, 300, 130], 2, dh, 16, t))      # unwritten slots hold NaN
    q = normal(g, c.tokens, 6, dh, dtype=t)
    many, c.table = crowded(c, q, how)
    for causal in (True, False):
        want, bound = attend(c, q, causal)
        within(ops.paged_attention(many, c.k_pages, c.v_pages, *c.index(), causal=causal, status=c.status)[:c.tokens], want, bound, 'causal %s' % causal)
    assert int(c.status) == 0


@pytest.mark.parametrize('B', [63, 64, 65, 300, 4097])
def test_many_sequences(B):
    """the search for a tile's sequence takes more than one round; most sequences bring one token or none"""
    t, g = torch.float32, gen(B)
    h, dh, page, wide = 1, 32, 16, 3
    rng = np.random.default_rng(B)
    new = rng.choice([0, 1, 1, 2, 20], B)
    new[0] = new[B - 1] = 1
    ctx = np.minimum(new + rng.integers(0, 28, B), wide * page)
    tokens = int(new.sum())
    cu = np.concatenate([[0], np.cumsum(new)])
    k_pages, v_pages = ops.paged_cache(B * wide, h, page, dh, t, DEV)
    k_pages.copy_(normal(g, *k_pages.shape)), v_pages.copy_(normal(g, *v_pages.shape))
    order = rng.permutation(B * wide).reshape(B, wide)
    table, status = i32(order.tolist()), torch.zeros(1, dtype=torch.int32, device=DEV)
    q, k, v = (normal(g, tokens + 2, h, dh) for _ in range(3))
    index = table, i32(cu.tolist()), i32(ctx.tolist())
    assert ops.paged_append(k, v, k_pages, v_pages, *index, q=q, q_out=q, status=status) is q
    # position p of sequence b in page order[b, p // page]
    dense = lambda pool: pool[index[0].long()].reshape(B, wide * page, dh)
    kd, vd = dense(k_pages[:, 0]), dense(v_pages[:, 0].transpose(1, 2))
    seq = torch.repeat_interleave(torch.arange(B), torch.from_numpy(new)).to(DEV)
    pos = torch.from_numpy(np.concatenate([np.arange(n - m, n) for m, n in zip(new, ctx)])).to(DEV)
    assert torch.equal(kd[seq, pos], k[:tokens, 0]) and torch.equal(vd[seq, pos], v[:tokens, 0])
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, k_pages, v_pages, *index, out=out, status=status)
    s = torch.einsum('nd,nkd->nk', q[:tokens, 0].double(), kd[seq].double()) * dh ** -0.5
    w = torch.softmax(s.masked_fill(torch.arange(wide * page, device=DEV)[None] > pos[:, None], float('-inf')), 1)
    want, size = torch.einsum('nk,nkd->nd', w, vd[seq].double()), torch.einsum('nk,nkd->nd', w, vd[seq].double().abs())
    dot = torch.einsum('nd,nkd->nk', q[:tokens, 0].double().abs(), kd[seq].double().abs()).amax() * dh ** -0.5
    rel = 2 * (dh + 8) * 2.0 ** -24 * dot + (wide * page + 64) * 2.0 ** -23
    within(out[:tokens, 0], want, size * rel * 1.01 + want.abs() * 2.0 ** -24 * 1.01 + 1e-30)
    assert int(status) == 0 and (out[tokens:] == 7.0).all()


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('rows,heads,dh,rot', [(5, 3, 7, 6), (3, 1, 1025, 64), (9, 2, 33, 2)])
def test_rotary_odd_heads_and_rows_that_begin_anywhere(dtype, rows, heads, dh, rot):
    t, g = TYPES[dtype], gen(dh)
    freq, _ = ops.rotary_frequencies(rot, device=DEV)
    pos = torch.randint(0, 5000, (rows,), generator=g, device=DEV, dtype=torch.int32)
    for lead in (0, 1, 3):
        x = normal(g, rows, lead + heads * dh + 1, dtype=t)[:, lead:lead + heads * dh].unflatten(1, (heads, dh))
        want, size = turn(x, freq, pos)
        within(ops.rotary(x, freq, pos), want, rot_bound(want, size, t))


NEAR = {'line': lambda V: torch.linspace(0, 1e-3, V), 'within a step': lambda V: 0.02 * torch.rand(V, generator=torch.Generator().manual_seed(V)),
        'two levels': lambda V: (torch.arange(V) % 3 == 0).float() * 2.0 ** -6, 'few steps': lambda V: 0.2 * torch.rand(V, generator=torch.Generator().manual_seed(V + 1)),
        'falling': lambda V: -torch.arange(V).float() * 2.0 ** -14}


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('V', [1500, 5000, 32003, 70001])
@pytest.mark.parametrize('how', list(NEAR))
def test_sample_rows_closer_than_a_step(dtype, V, how):
    """more words than a list or a step's candidates take, in few steps of the histogram: told apart by their keys"""
    x = NEAR[how](V)[None].repeat(3, 1)
    x[1] += 4.0
    x[2, V // 2:] = float('-inf')
    x = x.to(TYPES[dtype]).to(DEV)
    for u in (0.0, 0.37, 0.9):
        uu = torch.full((3,), u, device=DEV)
        for par in (dict(), dict(top_k=2), dict(top_k=300), dict(top_k=1400), dict(top_p=0.3), dict(top_k=700, top_p=0.5), dict(min_p=0.99),
                    dict(top_k=1000, top_p=0.9, min_p=0.9), dict(top_p=0.99, temperature=0.01), dict(top_k=299, top_p=0.6, temperature=0.004)):
            check_rows(x, uu, ops.sample(x, uu, **par), **par)


@pytest.mark.parametrize('V', [4999, 40001])
def test_sample_rows_that_begin_anywhere(V):
    g = gen(V)
    for t in (torch.bfloat16, torch.float32):
        wide = (3 * normal(g, 5, V + 20)).to(t)
        for lead in (1, 3, 7):
            x, u = wide[:, lead:lead + V], torch.rand(5, generator=g, device=DEV)
            check_rows(x, u, ops.sample(x, u, top_k=1500, top_p=0.9), top_k=1500, top_p=0.9)


def test_captured_draws_of_large_vocabularies():
    """rows in shared memory and rows beyond it, plain and with a step's books; the books are cleared between the replays"""
    g = gen(101)
    R = 6
    xs, u = [3 * normal(g, R, V) for V in (32003, 90001)], torch.rand(R, generator=g, device=DEV)
    preds = [torch.zeros(R, 2, dtype=torch.int32, device=DEV) for _ in xs]
    books = [[torch.zeros(n, dtype=torch.int32, device=DEV) for n in (R, R, R, 1)] + [torch.zeros(R, device=DEV)] for _ in xs]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def run():
        got = []
        for x, p, (tokens, fin, ln, left, scores) in zip(xs, preds, books):
            got.append(ops.sample(x, u, top_k=60, top_p=0.9))
            ops.sample_step(x, u, tokens, p, fin, ln, left, scores, 1, 5, top_k=60, top_p=0.9, status=status)
        return got
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for r in range(4):
        for x in xs:
            x.copy_(3 * normal(g, *x.shape))
        u.copy_(torch.rand(R, generator=g, device=DEV))
        if r == 2:
            xs[0][3] = float('nan')
        for p, b in zip(preds, books):
            for z in [p] + b:
                z.zero_()
        status.zero_()
        graph.replay()
        normal(g, 100)
        torch.cuda.synchronize()
        assert int(status) == (4 if r == 2 else 0)
        for x, o, p, (tokens, fin, ln, left, scores) in zip(xs, outs, preds, books):
            check_rows(x, u, o, top_k=60, top_p=0.9)
            ids = torch.where(o[0] < 0, 5, o[0])
            assert torch.equal(tokens, ids) and torch.equal(p[:, 1], ids) and not p[:, 0].any()
            assert torch.equal(fin, (ids == 5).int()) and int(left) == int((ids != 5).sum()) and torch.equal(ln, (ids != 5).int())
            assert torch.equal(scores, torch.where(o[0] < 0, 0.0, o[1]))


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_beam_search_with_rotary_positions(layout):
    """a hypothesis' score is the sum of its log-softmax under the teacher-forced decoder"""
    import test_gpu_sample_decode as D
    from neurst_amd.st.models import graph as G
    args, m, feats = D.make_model(6, D.ROTARY[layout], boost=0.05, beam_size=3, length_penalty_weight=0.0)
    m.infer(*feats)
    preds, scores, _ = m.last['beams']
    enc, len_enc = m.last['encoded'], m.last['len_encoded']
    for b in range(3):
        for j in range(3):
            toks = list(preds[b, j])
            if args.eos_idx in toks:
                toks = toks[:toks.index(args.eos_idx) + 1]
            inp = np.array([[args.token2idx['<sos>'], *toks[:-1]]], np.int32)
            with G.use_graph(m.graph), G.variable_scope(m.name):
                m.graph.begin_forward(None)
                with G.variable_scope('decoder'):
                    logits, _, _ = m.decoder.decode(enc[b:b + 1].contiguous(), len_enc[b:b + 1].contiguous(), torch.from_numpy(inp).to(DEV))
            lsm = torch.log_softmax(logits[0].double(), -1).cpu().numpy()
            want = sum(lsm[i, t] for i, t in enumerate(toks))
            # a dozen rounded layers of logits up to about 8, as for the drawn translations' scores
            assert abs(want - scores[b, j]) <= 12 * 8 * 2.0 ** -24 * 8 * len(toks), (b, j, want, scores[b, j], toks)
