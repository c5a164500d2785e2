"""The static checks of test_isa_invariants.py on the code as it is shipped: compiled with the compiler and the flags that the
Makefile builds libneurst_hip.so with, and an object for the Makefile to make again when they change."""
import os
import shutil
import subprocess

import pytest

import test_isa_invariants as checks

CSRC = checks.CSRC


def flags():
    return subprocess.run(['make', '-s', 'flags'], check=True, capture_output=True, text=True, cwd=CSRC).stdout.split()


@pytest.fixture(scope='module')
def shipped_isa(tmp_path_factory):
    compiler = flags()
    if not (shutil.which(compiler[0]) or os.path.exists(compiler[0])):
        pytest.skip('hipcc not available')
    out = tmp_path_factory.mktemp('isa') / 'layernorm.s'
    subprocess.run(compiler + ['-S', '--cuda-device-only', os.path.join(CSRC, 'layernorm.hip'), '-o', str(out)], check=True,
                   stdout=subprocess.PIPE, stderr=subprocess.PIPE)
    return open(out).read()


@pytest.mark.parametrize('which', ['fwd', 'bwd'])
def test_layernorm_line_kernels_as_shipped(shipped_isa, which):
    checks.test_layernorm_line_kernels_issue_exactly_the_operations_their_waits_count(shipped_isa, which)


def test_no_packed_fp32_arithmetic_is_shipped(shipped_isa):
    assert '-packed-fp32-ops' in flags()
    assert not any(op in shipped_isa for op in ('v_pk_add_f32', 'v_pk_mul_f32', 'v_pk_fma_f32'))


def test_objects_are_made_again_when_the_makefile_changes(tmp_path):
    """a dry run over empty objects that are newer than everything but the Makefile"""
    tree = tmp_path / 'neurst_amd' / 'csrc'
    shutil.copytree(CSRC, tree, ignore=shutil.ignore_patterns('build'))
    shutil.copytree(os.path.join(checks.ROOT, 'include'), tmp_path / 'include')
    names = [os.path.splitext(n)[0] for n in os.listdir(tree) if n.endswith(('.hip', '.cpp'))]
    (tree / 'build').mkdir()
    targets = [tree / 'build' / (n + '.o') for n in names]
    for p in [tree / n for n in os.listdir(tree) if n != 'build'] + [tmp_path / 'include' / 'neurst_hip.h']:
        os.utime(p, (1000, 1000))
    for i, p in enumerate(targets + [tree.parent / 'libneurst_hip.so']):
        p.write_bytes(b'')
        os.utime(p, (2000 + i, 2000 + i))
    assert subprocess.run(['make', '-q'], cwd=tree).returncode == 0
    os.utime(tree / 'Makefile', (9000, 9000))
    plan = subprocess.run(['make', '-n'], cwd=tree, check=True, capture_output=True, text=True).stdout
    assert all('-c %s' % n in plan for n in ('layernorm.hip', 'sample.hip', 'records.cpp')) and '-shared' in plan
