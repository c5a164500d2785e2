"""Rotary positions inside the models and translations drawn over the paged cache (Transformer_Decoder.sample_decode), on the
tiny models of the other model tests."""
import numpy as np
import pytest
import torch

import __graft_entry__ as ge
from neurst_amd import lib, ops
from neurst_amd.synthetic import make_batch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
ROTARY = {None: None, 'half': dict(base=50.0), 'interleaved': dict(base=100.0, layout='interleaved', dims=6, scaling='parts', factor=4.0, original_length=32)}


def make_model(seed, rotary=None, shrink=False, compute_dtype='fp32', boost=0.2, **over):
    args = ge.tiny_args('ce_ctc' if shrink else 'ctc_kd_ce', compute_dtype, shrink)
    args.max_len = 20
    for k, v in over.items():
        args[k] = v
    if rotary:
        args.model.decoder.rotary = dict(rotary)
    from neurst_amd.st.models.TransformerTPE import GlobalStep
    m = args.Model(GlobalStep(0), encoder=args.model.encoder.type, decoder=args.model.decoder.type, is_train=False, args=args)
    rng = np.random.default_rng(seed)
    P = {k: (v + 0.05 * rng.standard_normal(v.shape)).astype(np.float32) for k, v in m.store.export().items()}
    fc = [k for k in P if k.endswith('decoder_fc/kernel')][0]
    for k in P:
        if '/decoder/block_' in k and k.endswith('layer_norm_bias'):
            P[k] = (P[k] + 0.5).astype(np.float32)
    P[fc] = (P[fc] + 0.3 * rng.standard_normal(P[fc].shape)).astype(np.float32)
    P[fc][:, args.eos_idx] += boost                       # hypotheses end at different steps
    m.store.load_params(P)
    batch = make_batch(B=3, Traw=30, V=11, L=5, U=3, dim_raw=4, ragged=True, seed=seed)
    return args, m, (batch['feature'], batch['len_fea'])


@pytest.mark.parametrize('layout', [None, 'half', 'interleaved'])
@pytest.mark.parametrize('shrink', [False, True])
@pytest.mark.parametrize('seed', [1, 2, 3])
def test_temperature_zero_is_the_greedy_search(layout, shrink, seed):
    """the dense cache's loop and the paged one: the same ids, lengths, and the same continuation of a forced prefix"""
    args, m, feats = make_model(seed, ROTARY[layout], shrink)
    greedy, am = m.infer(*feats)
    length = m.last['len_decoded']
    args.decode, args.sample = 'sample', dict(temperature=0.0, num=2)
    preds, am2 = m.infer(*feats)
    assert np.array_equal(preds, greedy) and np.array_equal(m.last['len_decoded'], length) and np.array_equal(am, am2)
    both, scores, lens = m.last['samples']
    assert np.array_equal(both[:, 0], both[:, 1]) and (scores == 0).all()
    # the first tokens forced, of several lengths, none for one utterance
    lp = np.minimum(np.array([2, 0, 4]), length)
    preds, _ = m.infer(*feats, prefix=greedy[:, :4], len_prefix=lp)
    for b in range(3):
        if lp[b] < length[b]:                             # else the prefix holds the whole translation
            rest = greedy[b, lp[b]:length[b]]             # a search cut off at max_len goes on here: as many new tokens again
            assert np.array_equal(preds[b, :rest.size], rest)
            assert m.last['len_decoded'][b] >= rest.size


@pytest.mark.parametrize('layout', [None, 'half', 'interleaved'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('page_size', [16, 32])
def test_scores_are_those_of_the_teacher_forced_decoder(layout, dtype, page_size):
    """temperature 1 and no filter: a translation's score is the sum of its log-softmax under `decode`, prefix left out"""
    args, m, feats = make_model(5, ROTARY[layout], compute_dtype=dtype, boost=0.05, decode='sample', sample=dict(num=4, seed=7, page_size=page_size))
    rng = np.random.default_rng(3)
    prefix, lp = rng.integers(4, 10, (3, 18)).astype(np.int32), np.array([18, 0, 5])
    m.infer(*feats, prefix=prefix, len_prefix=lp)
    preds, scores, lens = m.last['samples']
    assert (np.diff(scores, axis=1) <= 0).all() and len(np.unique(preds.reshape(12, -1), axis=0)) > 4
    from neurst_amd.st.models import graph as G
    enc, len_enc = m.last['encoded'], m.last['len_encoded']
    # a token's error: bf16 products of logits up to about 8 over a dozen rounded layers, 2^-8 of them each; fp32 as much of 2^-24
    tol = {'fp32': 12 * 8 * 2.0 ** -24 * 8, 'bf16': 12 * 8 * 2.0 ** -8}[dtype]
    for b in range(3):
        for j in range(4):
            n = int(lens[b, j])
            toks = list(preds[b, j, :n]) + ([args.eos_idx] if n < preds.shape[2] or n < args.max_len else [])
            toks = toks[:preds.shape[2]]
            inp = np.array([[args.token2idx['<sos>'], *prefix[b, :lp[b]], *toks[:-1]]], np.int32)
            with G.use_graph(m.graph), G.variable_scope(m.name):
                m.graph.begin_forward(None)
                with G.variable_scope('decoder'):
                    logits, _, _ = m.decoder.decode(enc[b:b + 1].contiguous(), len_enc[b:b + 1].contiguous(), torch.from_numpy(inp).to(DEV))
            lsm = torch.log_softmax(logits[0].double(), -1).cpu().numpy()[lp[b]:]
            want = sum(lsm[i, t] for i, t in enumerate(toks))
            assert abs(want - scores[b, j]) <= tol * len(toks), (b, j, want, scores[b, j], toks)


def test_draws_repeat_with_their_seed_and_differ_without():
    args, m, feats = make_model(8, ROTARY['half'], decode='sample', sample=dict(num=3, seed=11, temperature=1.5, top_k=8, top_p=0.95, min_p=0.01))
    one = m.infer(*feats)[0], m.last['samples']
    two = m.infer(*feats)[0], m.last['samples']
    assert np.array_equal(one[0], two[0]) and all(np.array_equal(a, b) for a, b in zip(one[1], two[1]))
    args.sample = dict(args.sample, seed=12)
    m.infer(*feats)
    assert not np.array_equal(one[1][0], m.last['samples'][0])
    assert (one[1][0] >= 0).all() and (one[1][0] < 11).all()


def test_calls_without_a_seed_draw_numbers_of_their_own():
    """two batches of a test set are not drawn with the same numbers; a new model repeats the run"""
    runs = []
    for _ in range(2):
        args, m, feats = make_model(8, decode='sample', sample=dict(num=3, temperature=1.5))
        runs.append([])
        for _ in range(2):
            m.infer(*feats)
            runs[-1].append(m.last['samples'])
    assert all(np.array_equal(x, y) for a, b in zip(*runs) for x, y in zip(a, b))
    assert not np.array_equal(runs[0][0][1], runs[0][1][1])
    args.sample = dict(args.sample, seed=5)
    m.infer(*feats)
    seeded = m.last['samples']
    m.infer(*feats)
    assert all(np.array_equal(x, y) for x, y in zip(seeded, m.last['samples']))


def test_logits_that_are_nan_are_not_a_translation():
    """a hypothesis that breaks off keeps the score it had, the best there is: the call raises instead of returning it"""
    args, m, feats = make_model(4, decode='sample', sample=dict(num=2, seed=3))
    m.infer(*feats)
    P = m.store.export()
    fc = [k for k in P if k.endswith('decoder_fc/kernel')][0]
    P[fc][:] = np.nan
    m.store.load_params(P)
    with pytest.raises(lib.NeurstLibError, match='nothing to draw'):
        m.infer(*feats)


def test_lengths_of_a_prefix_need_sampled_decoding():
    args, m, feats = make_model(9)
    with pytest.raises(NotImplementedError, match='prefix'):
        m.infer(*feats, len_prefix=np.array([0, 0, 0]))


def test_refusals():
    args, m, feats = make_model(9, decode='sample', sample=dict(nmu=3))
    with pytest.raises(ValueError, match='unknown keys'):
        m.infer(*feats)
    for sample in (dict(num=0), dict(page_size=24), dict(temperature=-1.0), dict(top_p=0.0), dict(min_p=2.0), dict(top_k=-1)):
        args.sample = sample
        with pytest.raises((ValueError, RuntimeError)):
            m.infer(*feats)
    args.sample = None
    with pytest.raises(ValueError, match='prefix'):
        m.infer(*feats, prefix=np.zeros((2, 3), np.int32))
    with pytest.raises(ValueError, match='prefix'):
        m.infer(*feats, prefix=np.zeros((3, 3), np.int32), len_prefix=np.array([1, 4, 0]))
    for prefix in (np.array([[1, 2, -1]] * 3), np.array([[1, 2, 10 ** 6]] * 3), np.zeros(3, np.int32), np.zeros((3, 3))):
        with pytest.raises(ValueError, match='prefix'):
            m.infer(*feats, prefix=prefix)
    m.infer(*feats, prefix=np.array([[1, 2, -1]] * 3), len_prefix=np.array([2, 0, 1]))       # what lies behind the length is not read
    with pytest.raises(ValueError, match='prefix'):
        m.infer(*feats, len_prefix=np.array([0, 0, 0]))
    args.sample = dict(page_size=0)
    with pytest.raises(ValueError, match='page_size'):
        m.infer(*feats)
    args.sample = None
    args.decode = 'search'
    with pytest.raises(NotImplementedError, match='prefix'):
        m.infer(*feats, prefix=np.zeros((3, 3), np.int32))
    args.decode = 'other'
    with pytest.raises(ValueError, match='decode'):
        m.infer(*feats)
    args.decode = None
    for rotary in (dict(dims=10), dict(layout='other'), dict(scaling='other'), dict(bse=3.0), dict(dims=3)):
        args.model.decoder.rotary = rotary
        with pytest.raises(ValueError, match='rotary'):
            m.infer(*feats)


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('causal', [True, False])
def test_rotary_self_attention_gradients(layout, causal):
    """multihead_attention with rotary positions against the same in fp64 with torch's gradients.  A result passes at most five
    sums of 64 terms or fewer, each within 64 2^-24 of its terms' magnitudes, taken as 8 times the largest result."""
    from neurst_amd.st.layers import common_attention_v1 as A
    from neurst_amd.st.models import graph as G
    from neurst_amd.st.models.tools.utils import Rotary, multihead_attention
    B, T, H, dh = 2, 21, 2, 16
    d = H * dh
    names = [('att/qkv_transform/kernel', (3 * d, d)), ('att/qkv_transform/bias', (3 * d,)), ('att/output_transform/kernel', (d, d)),
             ('att/output_transform/bias', (d,))]
    store = G.VariableStore([('m/' + n, s, 'glorot' if len(s) == 2 else 'zeros') for n, s in names], torch.device(DEV), ops.F32, seed=1)
    gen = torch.Generator().manual_seed(2)
    x, dy = torch.randn(B, T, d, generator=gen), torch.randn(B, T, d, generator=gen)
    cfg = dict(base=100.0, layout=layout, dims=12, scaling='parts', factor=4.0, original_length=64)
    lens = torch.tensor([T, 13], dtype=torch.int32)
    rot = Rotary.of(cfg, dh, DEV)
    g, tape = G.Graph(store, ops.F32), G.Tape()
    xd = x.to(DEV)
    with G.use_graph(g), G.variable_scope('m'):
        g.begin_forward(tape, step=0)
        bias = A.attention_bias_lower_triangle(T) if causal else A.attention_bias_ignore_padding(lens.to(DEV))
        out = multihead_attention(xd, None, bias, d, d, d, H, 0.0, name='att', rotary=rot)
        tape.set(out, dy.to(DEV))
        tape.backward()
        dx = tape.grad(xd)
        torch.cuda.synchronize()
    P = {k: torch.from_numpy(v).double().requires_grad_() for k, v in store.export().items()}
    xr = x.double().requires_grad_()
    qkv = xr @ P['m/att/qkv_transform/kernel'].t() + P['m/att/qkv_transform/bias']
    q, k, v = (t.view(B, T, H, dh).transpose(1, 2) for t in qkv.split(d, -1))
    a = torch.arange(T).double()[:, None] * rot.freq.cpu()
    c, s = torch.cos(a) * rot.mscale, torch.sin(a) * rot.mscale

    def turn(t):
        n = 6
        u, w = (t[..., :n], t[..., n:2 * n]) if layout == 'half' else (t[..., 0:2 * n:2], t[..., 1:2 * n:2])
        y = (u * c - w * s, w * c + u * s)
        y = torch.cat(y, -1) if layout == 'half' else torch.stack(y, -1).flatten(-2)
        return torch.cat([y, t[..., 2 * n:]], -1)
    w = turn(q) @ turn(k).transpose(-1, -2) * dh ** -0.5
    hide = torch.ones(T, T, dtype=torch.bool).triu(1)[None, None] if causal else (torch.arange(T) >= lens[:, None])[:, None, None]
    w = torch.softmax(w.masked_fill(hide, float('-inf')), -1)
    want = (w @ v).transpose(1, 2).reshape(B, T, d) @ P['m/att/output_transform/kernel'].t() + P['m/att/output_transform/bias']
    want.backward(dy.double())
    tol = 5 * 64 * 2.0 ** -24 * 8
    near = lambda got, ref, what: (got.double().cpu() - ref).abs().max() <= tol * ref.abs().max() or pytest.fail('%s: %g of %g' % (
        what, (got.double().cpu() - ref).abs().max(), ref.abs().max()))
    near(out, want.detach(), 'out')
    near(dx, xr.grad, 'dx')
    for n, gr in store.export_grads().items():
        ref = P[n].grad
        if n.endswith('qkv_transform/bias'):              # the key bias of unturned columns cancels in the softmax: against the largest
            near(torch.from_numpy(gr), ref, n)
        else:
            near(torch.from_numpy(gr), ref, n)


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_a_model_with_rotary_positions_trains(layout):
    """rotary positions in all three stacks: finite losses over a few steps, and every variable gets a gradient"""
    args = ge.tiny_args(compute_dtype='bf16')
    for part in ('encoder', 'encoder2', 'decoder'):
        getattr(args.model, part).rotary = dict(ROTARY[layout])
    from neurst_amd.st.models.TransformerTPE import GlobalStep
    m = args.Model(GlobalStep(3), encoder=args.model.encoder.type, decoder=args.model.decoder.type, is_train=True, args=args)
    batch = make_batch(B=2, Traw=24, V=11, L=5, U=3, Lb=4, bert_dim=16, dim_raw=4, ragged=True)
    for _ in range(3):
        assert np.isfinite(m.train_step(batch)[0])
    grads = m.store.export_grads()
    assert all(np.isfinite(v).all() for v in grads.values()) and all(np.abs(grads[k]).max() > 0 for k in grads if 'qkv_transform/kernel' in k)
