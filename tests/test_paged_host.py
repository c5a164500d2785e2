"""Rotary positions, the paged cache, attention over it and sampling, as far as they run without a GPU: the C ABI's and the
wrappers' refusals, the index arithmetic that keeps bad pages and lengths in range, and the frequencies."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from neurst_amd import lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20      # stands for an aligned device pointer: every call below is refused before it could be used
NAN, INF = float('nan'), float('inf')


def test_index_arithmetic_of_the_paged_cache(tmp_path):
    """ragged, empty and corrupted batches under the address and undefined-behaviour sanitizers (host code)"""
    exe = str(tmp_path / 'check')
    src = os.path.join(ROOT, 'tests', 'native', 'check_paged_index.cpp')
    subprocess.run(['g++', '-O2', '-std=c++17', '-fsanitize=address,undefined', src, '-o', exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == 'ok', r.stdout + r.stderr


def test_rows_and_positions_of_the_tiles_stay_with_their_sequences(tmp_path):
    """starts that do not grow, rows past the tensors: what a tile reads and writes lies inside its sequence's rows"""
    exe = str(tmp_path / 'check')
    src = os.path.join(ROOT, 'tests', 'native', 'check_paged_tiles.cpp')
    subprocess.run(['g++', '-O2', '-std=c++17', '-fsanitize=address,undefined', src, '-o', exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == 'ok', r.stdout + r.stderr


def _call(name, good, **change):
    args = dict(good, **change)
    return getattr(lib.load(), name)(*args.values())


ROTARY = dict(x=P, y=P, freq=P, positions=P, rows=4, heads=2, dh=16, pairs=8, ldx=32, ldy=32, pos0=0, period=0, layout=0, inverse=0,
              mscale=1.0, dtype=1, stream=None)


@pytest.mark.parametrize('change', [dict(x=None), dict(y=None), dict(freq=None), dict(dtype=2), dict(rows=-1), dict(heads=0), dict(dh=0),
                                    dict(pairs=0), dict(pairs=9), dict(ldx=31), dict(ldy=31), dict(layout=2), dict(y=P, ldy=40), dict(period=-1),
                                    dict(positions=None, pos0=2 ** 31 - 2), dict(positions=None, pos0=-2 ** 31 - 1), dict(layout=1, x=P + 2),
                                    dict(layout=1, ldx=33, y=2 * P)])
def test_rotary_refuses(change):
    assert _call('neurst_rotary', ROTARY, **change) == -1
    assert b'rotary' in lib.load().neurst_last_error()


APPEND = dict(k=P, v=P, q=P, k_pages=P, v_pages=P, q_out=P, page_table=P, cu_new=P, ctx_len=P, freq=P, status=None, tokens=4, batch=2, wide=3,
              ld_table=3, n_pages=6, page_size=16, kv_heads=2, q_heads=4, dh=16, ldk=32, ldv=32, ldq=64, ldqo=64, pairs=8, layout=0, mscale=1.0,
              dtype=1, stream=None)
BAD_INDEX = [dict(page_table=None), dict(cu_new=None), dict(ctx_len=None), dict(tokens=-1), dict(batch=-1), dict(batch=2 ** 21), dict(n_pages=0),
             dict(wide=0), dict(ld_table=2), dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(wide=2 ** 24, ld_table=2 ** 24, page_size=128),
             dict(dtype=3), dict(dh=12), dict(dh=0), dict(dh=264)]


@pytest.mark.parametrize('change', BAD_INDEX + [dict(k=None), dict(v=None), dict(k_pages=None), dict(v_pages=None), dict(q=None), dict(q_out=None),
                                                dict(kv_heads=0), dict(ldk=16), dict(ldv=16), dict(ldq=32), dict(ldqo=32), dict(ldqo=72),
                                                dict(pairs=0), dict(pairs=9), dict(freq=None), dict(layout=3), dict(k=P + 2), dict(v_pages=P + 8),
                                                dict(ldk=36), dict(ldq=68, ldqo=68)])
def test_paged_append_refuses(change):
    assert _call('neurst_paged_append', APPEND, **change) == -1
    assert b'paged_append' in lib.load().neurst_last_error()


ATTEND = dict(q=P, k_pages=P, v_pages=P, o=2 * P, page_table=P, cu_new=P, ctx_len=P, status=None, tokens=4, batch=2, wide=300, ld_table=300,
              n_pages=600, page_size=16, q_heads=4, kv_heads=2, dh=16, ldq=64, ldo=64, scale=0.25, causal=1, dtype=1, workspace=P,
              workspace_bytes=1 << 30, stream=None)


@pytest.mark.parametrize('change', BAD_INDEX[:12] + BAD_INDEX[13:] + [
    dict(q=None), dict(k_pages=None), dict(v_pages=None), dict(o=None), dict(q_heads=3), dict(q_heads=0), dict(kv_heads=0), dict(ldq=48), dict(ldo=48),
    dict(scale=NAN), dict(scale=INF), dict(q=P + 4), dict(ldo=68), dict(workspace=None), dict(workspace_bytes=16), dict(workspace=P + 4),
    dict(tokens=2 ** 31 - 1, q_heads=8)])
def test_paged_attention_refuses(change):
    assert _call('neurst_paged_attention', ATTEND, **change) == -1
    assert b'paged_attention' in lib.load().neurst_last_error()


def test_memory_that_is_written_must_be_apart():
    """in place and interleaved slices of one packed projection are fine (the GPU tests make those calls); what another part of the
    call reads is not"""
    M = 1 << 30
    refused = lambda name, good, **change: _call(name, good, **change) == -1 and b'apart' in lib.load().neurst_last_error()
    packed = dict(APPEND, k=M + 128, v=M + 192, q=M, q_out=M, k_pages=2 * M, v_pages=3 * M, ldk=128, ldv=128, ldq=128, ldqo=128)      # q | k | v, bf16
    for change in (dict(k=M), dict(v=M), dict(q_heads=2, q=M + 128, q_out=M + 128), dict(q_heads=2, q=M + 192, q_out=M + 192), dict(k=M + 112),
                   dict(q=4 * M, q_out=4 * M + 16), dict(q=4 * M, q_out=4 * M + 256 * 3 + 112), dict(q_out=M + 128), dict(q_out=M + 256),
                   dict(v_pages=2 * M), dict(v_pages=2 * M + 6 * 2 * 16 * 16 * 2 - 16), dict(k_pages=M + 256), dict(v_pages=M + 128), dict(k_pages=M - 16),
                   dict(q=5 * M, q_out=3 * M), dict(q=2 * M, q_out=2 * M), dict(ldk=136, k=M + 512)):
        assert refused('neurst_paged_append', packed, **change), change
    attend = dict(ATTEND, q=M, o=2 * M, k_pages=3 * M, v_pages=4 * M, workspace=5 * M)
    for change in (dict(o=M), dict(o=M + 128 * 3), dict(o=M + 64, ldq=128, ldo=128), dict(o=3 * M), dict(o=4 * M + 128), dict(workspace=M), dict(workspace=2 * M),
                   dict(workspace=3 * M + 16), dict(workspace=4 * M), dict(o=5 * M)):
        assert refused('neurst_paged_attention', attend, **change), change
    for change in (dict(y=P + 2), dict(y=P + 3 * 64), dict(y=P + 32, ldx=40, ldy=40), dict(y=P + 64, ldx=40, ldy=48)):
        assert refused('neurst_rotary', ROTARY, **change), change


SAMPLE = dict(logits=P, u=P, ids=P, logp=P, t=None, k=None, p=None, m=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, rows=2, V=10, ld=10,
              dtype=0, stream=None)


@pytest.mark.parametrize('change', [dict(logits=None), dict(u=None), dict(ids=None), dict(logp=None), dict(temperature=-1.0), dict(temperature=NAN),
                                    dict(temperature=INF), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=NAN), dict(min_p=-0.1),
                                    dict(min_p=1.1), dict(min_p=NAN), dict(rows=-1), dict(V=0), dict(V=2 ** 19 + 1, ld=2 ** 20), dict(ld=9), dict(dtype=2)])
def test_sample_refuses(change):
    assert _call('neurst_sample', SAMPLE, **change) == -1
    assert b'sample' in lib.load().neurst_last_error()


def test_sample_step_refuses():
    good = dict(logits=P, u=P, tokens=P, preds=P, finished=P, len_decoded=P, n_unfinished=P, scores=P, t=None, k=None, p=None, m=None, temperature=1.0,
                top_k=0, top_p=1.0, min_p=0.0, rows=2, V=10, ld=10, step=0, max_steps=4, eos=3, dtype=0, stream=None)
    for change in [{k: None} for k in ('tokens', 'preds', 'finished', 'len_decoded', 'n_unfinished', 'scores', 'u')] + [dict(step=4), dict(step=-1), dict(top_p=2.0)]:
        assert _call('neurst_sample_step', good, **change) == -1, change


def test_sizes_that_pass_64_bits_are_refused():
    """sums and products of the checks themselves"""
    for change in (dict(positions=None, pos0=2 ** 63 - 1), dict(positions=None, pos0=2 ** 63 - 1, period=7), dict(positions=None, rows=2 ** 62, pos0=-2 ** 31),
                   dict(heads=65536, dh=65536, pairs=1, ldx=2 ** 32, ldy=2 ** 32)):
        assert _call('neurst_rotary', ROTARY, **change) == -1, change
    for name, good in (('neurst_paged_append', APPEND), ('neurst_paged_attention', dict(ATTEND, workspace=None))):
        assert _call(name, good, wide=2 ** 60, ld_table=2 ** 60) == -1
        assert b'bad page counts' in lib.load().neurst_last_error()


def test_scales_and_head_counts_at_their_limits_are_refused():
    for scale in (3.3e38, -3.3e38, 2.4e38, NAN, -INF):      # times log2(e) beyond fp32
        assert _call('neurst_paged_attention', ATTEND, scale=scale) == -1
        assert b'scale' in lib.load().neurst_last_error()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    with pytest.raises(ValueError, match='heads'):
        ops.paged_attention(torch.zeros(3, 2, 8), torch.zeros(4, 0, 16, 8), torch.zeros(4, 0, 8, 16), torch.zeros(2, 1, dtype=torch.int32), i32(0, 1, 3), i32(1, 2))


def test_sample_step_checked_refuses():
    good = dict(logits=P, u=P, tokens=P, preds=P, finished=P, len_decoded=P, n_unfinished=P, scores=P, status=P, t=None, k=None, p=None, m=None,
                temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, rows=2, V=10, ld=10, step=0, max_steps=4, eos=3, dtype=0, stream=None)
    for change in [{k: None} for k in ('logits', 'tokens', 'preds', 'finished', 'len_decoded', 'n_unfinished', 'scores', 'u')] + [
            dict(step=4), dict(step=-1), dict(top_p=2.0), dict(ld=9), dict(dtype=2)]:
        assert _call('neurst_sample_step_checked', good, **change) == -1, change
    assert _call('neurst_sample_step_checked', good, rows=0) == 0


def test_calls_without_rows_do_nothing():
    assert _call('neurst_rotary', ROTARY, rows=0) == 0
    assert _call('neurst_paged_append', APPEND, tokens=0) == 0
    assert _call('neurst_paged_attention', ATTEND, tokens=0) == 0
    assert _call('neurst_sample', SAMPLE, rows=0) == 0


def test_wrappers_refuse_what_the_c_entry_cannot_see():
    f = torch.ones(4, dtype=torch.float64)
    x = torch.zeros(3, 2, 8)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    kp, vp = torch.zeros(4, 2, 16, 8), torch.zeros(4, 2, 8, 16)
    idx = (torch.zeros(2, 1, dtype=torch.int32), i32(0, 1, 3), i32(1, 2))
    bad = [lambda: ops.rotary(x, f),                                                            # not on a GPU
           lambda: ops.rotary(x.view(6, 8), f), lambda: ops.rotary(x.transpose(1, 2), f), lambda: ops.rotary(x.double(), f),
           lambda: ops.rotary(x, f.float()), lambda: ops.rotary(x, torch.ones(5, dtype=torch.float64)), lambda: ops.rotary(x, f, layout='other'),
           lambda: ops.rotary(x, f, positions=torch.zeros(3, dtype=torch.int64)), lambda: ops.rotary(x, f, positions=i32(1, 2)),
           lambda: ops.rotary(x, f, out=torch.zeros(3, 2, 7)), lambda: ops.rotary(x[:2], f, out=x[1:]), lambda: ops.rotary(x, f, mscale=NAN),
           lambda: ops.paged_append(x, x, kp, vp, *idx), lambda: ops.paged_append(x, x, kp, kp, *idx), lambda: ops.paged_append(x, x[:2], kp, vp, *idx),
           lambda: ops.paged_append(x, x, kp, vp, idx[0], idx[1].long(), idx[2]), lambda: ops.paged_append(x, x, kp, vp, idx[0], idx[1][:2], idx[2]),
           lambda: ops.paged_append(x, x, kp, vp, *idx, q=x.bfloat16()), lambda: ops.paged_append(x, x, kp, vp, *idx, q_out=x),
           lambda: ops.paged_append(x, x, kp, vp, *idx, q=torch.zeros(3, 2, 8), q_out=x),
           lambda: ops.paged_attention(x, kp, vp, *idx), lambda: ops.paged_attention(torch.zeros(3, 3, 8), kp, vp, *idx),
           lambda: ops.paged_attention(x, kp, vp, *idx, out=x), lambda: ops.paged_attention(x, kp, vp, *idx, scale=INF),
           lambda: ops.paged_attention(x.bfloat16(), kp, vp, *idx),
           lambda: ops.paged_append(x.view(6, 8), x.view(6, 8), kp, vp, *idx), lambda: ops.paged_append(x, x, kp, vp, *idx, q=x.flatten()),
           lambda: ops.sample(x[0], torch.zeros(2)), lambda: ops.sample(x[0], torch.zeros(3)), lambda: ops.sample(x, torch.zeros(3)),
           lambda: ops.sample(x[0], torch.zeros(2), top_k=torch.zeros(2)), lambda: ops.sample(x[0].t(), torch.zeros(8))]
    for k, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail('call %d was not refused' % k)


@pytest.mark.parametrize('scaling', [None, 'linear', 'base', 'parts'])
def test_frequencies(scaling):
    rot, base, s, L = 96, 10000.0, 8.0, 4096
    f, m = ops.rotary_frequencies(rot, base, scaling, 1.0 if scaling is None else s, L, device='cpu')
    assert f.dtype == torch.float64 and f.shape == (rot // 2,)
    plain = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if scaling is None:
        want = plain
    elif scaling == 'linear':
        want = [x / s for x in plain]
    elif scaling == 'base':
        want = [(base * s ** (rot / (rot - 2))) ** (-2 * i / rot) for i in range(rot // 2)]
        assert abs(want[-1] - plain[-1] / s) < 1e-12 * want[-1] and want[0] == plain[0]
    else:
        want = []
        for x in plain:
            turns = L * x / (2 * math.pi)
            a = min(1, max(0, (turns - 1) / 31))
            want.append(x if a == 1 else x / s if a == 0 else x * ((1 - a) / s + a))
        assert want[0] == plain[0] and want[-1] == plain[-1] / s
    # pow of two libraries: a few steps of fp64 each
    np.testing.assert_allclose(f.numpy(), want, rtol=16 * 2.0 ** -53)
    assert m == (0.1 * math.log(s) + 1 if scaling == 'parts' else 1.0)
    for bad in [dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=4, base=0.0), dict(rot_dim=4, factor=0.5), dict(rot_dim=4, scaling='other'),
                dict(rot_dim=2, scaling='base'), dict(rot_dim=4, scaling='parts', turns_fast=1.0), dict(rot_dim=4, factor=NAN)]:
        with pytest.raises(ValueError):
            ops.rotary_frequencies(device='cpu', **bad)
