"""CPU: the 64-bit oracle of the sequence operators against differences, and what the entry points refuse."""
import ctypes as C

import pytest
import torch

from oracle import sequence_oracle as O

NULL_STREAM = None


def _differences(f, leaves, seeds, step=1e-5):
    """gradient of sum(seed * f) by central differences, one element at a time"""
    grads = []
    for t in leaves:
        g = torch.zeros_like(t)
        flat, gf = t.view(-1), g.view(-1)
        for i in range(flat.numel()):
            was = flat[i].item()
            vals = []
            for sign in (1, -1):
                flat[i] = was + sign * step
                vals.append(sum((s * o).sum() for s, o in zip(seeds, f())).item())
            flat[i] = was
            gf[i] = (vals[0] - vals[1]) / (2 * step)
        grads.append(g)
    return grads


def _rnd(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def test_norm_gradient_matches_differences():
    g = torch.Generator().manual_seed(1)
    t, gamma, dy = _rnd(g, 3, 5), _rnd(g, 5), _rnd(g, 3, 5)
    _, dt, dgamma = O.rms_norm(t, gamma, 1e-3, dy)
    a, b = _differences(lambda: [O.rms_norm(t, gamma, 1e-3)], [t, gamma], [dy])
    assert torch.allclose(a, dt, atol=1e-8) and torch.allclose(b, dgamma, atol=1e-8)


@pytest.mark.parametrize('silu', [True, False])
def test_conv_gradient_matches_differences(silu):
    g = torch.Generator().manual_seed(2)
    lengths = [3, 0, 1, 5]
    x, w, b, init = _rnd(g, 9, 2), _rnd(g, 4, 2), _rnd(g, 2), _rnd(g, 4, 3, 2)
    dy, df = _rnd(g, 9, 2), _rnd(g, 4, 3, 2)
    r = O.conv1d(x, w, b, init, lengths, silu, dy, df)

    def f():
        o = O.conv1d(x, w, b, init, lengths, silu)
        return o['y'], o['final']
    for got, want in zip(_differences(f, [x, w, b, init], [dy, df]), (r['dx'], r['dw'], r['dbias'], r['dinitial'])):
        assert torch.allclose(got, want, atol=1e-7)


@pytest.mark.parametrize('softplus', [True, False])
def test_scan_gradient_matches_differences(softplus):
    g = torch.Generator().manual_seed(3)
    lengths = [2, 0, 4]
    rows, cols, groups, n = 7, 4, 2, 3                      # one row behind the last utterance
    x, dt, z = (_rnd(g, rows, cols) for _ in range(3))
    if not softplus:
        dt = dt.abs()
    A, D, bias, init = -_rnd(g, cols, n).abs(), _rnd(g, cols), 0.1 * _rnd(g, cols), _rnd(g, 3, cols, n)
    B, Cm = _rnd(g, rows, groups, n), _rnd(g, rows, groups, n)
    dy, df = _rnd(g, rows, cols), _rnd(g, 3, cols, n)
    r = O.scan(x, dt, A, B, Cm, D, z, bias, init, lengths, softplus, dy, df)
    assert r['y'][6].abs().sum() == 0 and r['dx'][6].abs().sum() == 0

    def f():
        o = O.scan(x, dt, A, B, Cm, D, z, bias, init, lengths, softplus)
        return o['y'], o['final']
    leaves = dict(x=x, dt=dt, A=A, B=B, C=Cm, D=D, z=z, dt_bias=bias, initial=init)
    for (k, _), got in zip(leaves.items(), _differences(f, list(leaves.values()), [dy, df])):
        assert torch.allclose(got, r['d' + k], atol=1e-7), k


# ------------------------------------------------------------------------------------------------------------- refusals

@pytest.fixture(scope='module')
def L(built_lib):
    return built_lib


ONE = C.c_void_p(4096)           # an address that is never followed: every call below is refused before a launch


def test_revision(L):
    assert L.lib.vc_seq_version() == 1


def test_struct_layouts_match_the_header(L, tmp_path):
    import os
    import shutil
    import subprocess
    cc = shutil.which('gcc')
    if cc is None:
        pytest.skip('no host compiler')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ['#include "vc_cyclegan.h"', '#include <stdio.h>', 'int main(void) {']
    want = []
    for cls, name in ((L.ScanArgs, 'vc_scan_args'), (L.Conv1dArgs, 'vc_conv1d_args')):
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, f))
            want.append(getattr(cls, f).offset)
    src = tmp_path / 'l.c'
    src.write_text('\n'.join(lines + ['return 0; }']))
    subprocess.check_call([cc, '-I', os.path.join(root, 'include'), str(src), '-o', str(tmp_path / 'l')])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / 'l')], text=True).split()]
    assert got == want


def test_norm_refusals(L):
    f = L.lib.vc_rms_norm_fwd

    def call(x=ONE, gamma=ONE, y=ONE, res=None, total=None, eps=1e-6, rows=4, cols=8, kind=0, stream_kind=0):
        return f(x, 8, res, 8, gamma, y, 8, total, 8, None, eps, rows, cols, kind, stream_kind, NULL_STREAM)
    for bad in (dict(x=None), dict(gamma=None), dict(y=None), dict(eps=0.0), dict(eps=float('nan')), dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(kind=3), dict(kind=-1),
                dict(kind=1, stream_kind=2), dict(stream_kind=1), dict(res=ONE)):
        assert call(**bad) == -1, bad
        assert b'vc_rms_norm_fwd' in L.lib.vc_last_error()
    assert call(rows=0, x=None) == 0
    q = L.lib.vc_rms_norm_e4m3
    assert q(ONE, 96, None, 0, ONE, ONE, 96, ONE, None, 0, 1e-6, 4, 96, 48, 0, 0, NULL_STREAM) == -1       # a group that is not offered
    assert q(ONE, 96, None, 0, ONE, ONE, 96, ONE, None, 0, 1e-6, 4, 96, 64, 0, 0, NULL_STREAM) == -1       # ... or does not divide the columns
    assert q(ONE, 96, None, 0, ONE, ONE, 96, None, None, 0, 1e-6, 4, 96, 32, 0, 0, NULL_STREAM) == -1      # no place for the scales
    b = L.lib.vc_rms_norm_bwd
    assert b(ONE, 8, None, 0, ONE, 8, ONE, ONE, None, 8, None, 8, None, None, 0, 4, 8, 0, 0, NULL_STREAM) == -1     # nothing is wanted
    assert b(ONE, 8, None, 0, ONE, 8, None, ONE, ONE, 8, None, 8, None, None, 0, 4, 8, 0, 0, NULL_STREAM) == -1     # no statistics
    need = L.lib.vc_rms_norm_bwd_work(4, 8)
    if need:
        assert b(ONE, 8, None, 0, ONE, 8, ONE, ONE, ONE, 8, None, 8, ONE, ONE, need - 1, 4, 8, 0, 0, NULL_STREAM) == -2


def _conv(L, **kw):
    a = L.Conv1dArgs(x=4096, w=4096, y=4096, x_ld=8, y_ld=8, rows=12, cols=8, taps=4, n_seqs=3, type=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_conv_refusals(L):
    f = L.lib.vc_causal_conv1d_fwd
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(taps=1), dict(taps=9), dict(cols=0), dict(n_seqs=0), dict(rows=-1), dict(rows=1 << 31), dict(rows=13), dict(type=5),
                dict(initial=4096, final_state=4096)):
        assert f(C.byref(_conv(L, **bad)), NULL_STREAM) == -1, bad
    assert f(None, NULL_STREAM) == -1
    b = L.lib.vc_causal_conv1d_bwd
    for bad in (dict(dy=None), dict(dy=4096, taps=1), dict(dy=4096, w=None)):
        assert b(C.byref(_conv(L, **bad)), NULL_STREAM) == -1, bad
    a = _conv(L, dy=4096, dx=4096, dw=4096, dx_ld=8, dy_ld=8)
    need = L.lib.vc_causal_conv1d_bwd_work(C.byref(a))
    if need:
        a.work, a.work_floats = 4096, need - 1
        assert b(C.byref(a), NULL_STREAM) == -2
    s = L.lib.vc_causal_conv1d_step
    assert s(ONE, 8, ONE, ONE, ONE, None, ONE, 8, 4097, 5000, 8, 4, 0, 1, NULL_STREAM) == -1      # more rows with slots than a wave looks through
    args = [ONE, 8, ONE, None, ONE, None, ONE, 8, 2, 4, 8, 4, 0, 1, NULL_STREAM]
    for i, v in ((0, None), (2, None), (4, None), (6, None), (8, -1), (8, 65536), (9, 1), (9, 0), (10, 0), (11, 1), (11, 9), (12, 3)):
        bad = list(args)
        bad[i] = v
        assert s(*bad) == -1, (i, v)


def _scan(L, **kw):
    a = L.ScanArgs(x=4096, dt=4096, B=4096, C=4096, A=4096, y=4096, x_ld=8, dt_ld=8, b_ld=16, c_ld=16, y_ld=8, rows=12, cols=8, states=16, groups=1, n_seqs=3, type=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_scan_refusals(L):
    f = L.lib.vc_selective_scan_fwd
    for bad in (dict(x=None), dict(dt=None), dict(A=None), dict(B=None), dict(C=None), dict(y=None), dict(states=0), dict(states=65), dict(groups=3), dict(groups=0), dict(cols=0),
                dict(n_seqs=0), dict(rows=-1), dict(rows=1 << 31), dict(rows=13), dict(type=3), dict(initial=4096, final_state=4096),
                dict(x_ld=-1), dict(dt_ld=(1 << 24) + 1), dict(b_ld=1 << 25), dict(c_ld=-8), dict(y_ld=7), dict(y_ld=1 << 25), dict(z=4096, z_ld=1 << 25)):
        assert f(C.byref(_scan(L, **bad)), NULL_STREAM) == -1, bad
    assert f(None, NULL_STREAM) == -1
    a = _scan(L)
    need = L.lib.vc_selective_scan_saved(C.byref(a))
    assert need >= 3 * 8 * 16
    a.saved, a.saved_floats = 4096, need - 1
    assert f(C.byref(a), NULL_STREAM) == -2
    b = L.lib.vc_selective_scan_bwd
    full = dict(dy=4096, dx=4096, ddt=4096, dB=4096, dC=4096, dA=4096, saved=4096, saved_floats=need, dy_ld=8, dx_ld=8, ddt_ld=8, db_ld=16, dc_ld=16)
    a = _scan(L, **full)
    work = L.lib.vc_selective_scan_bwd_work(C.byref(a))
    assert work > 0
    full.update(work=4096, work_floats=work)
    for bad in (dict(dy=None), dict(dx=None), dict(ddt=None), dict(dB=None), dict(dC=None), dict(dA=None), dict(saved=None), dict(z=4096), dict(states=65),
                dict(dx_ld=7), dict(ddt_ld=1 << 25), dict(z=4096, dz=4096, dz_ld=7), dict(db_ld=15), dict(dc_ld=3), dict(dy_ld=-1)):
        assert b(C.byref(_scan(L, **{**full, **bad})), NULL_STREAM) == -1, bad
    for bad in (dict(saved_floats=need - 1), dict(work_floats=work - 1), dict(work=None)):
        assert b(C.byref(_scan(L, **{**full, **bad})), NULL_STREAM) == -2, bad
    assert L.lib.vc_selective_scan_saved(C.byref(_scan(L, states=70))) == -1
    s = L.lib.vc_selective_scan_step
    args = [ONE, 8, ONE, 8, None, 0, ONE, 16, ONE, 16, ONE, None, None, ONE, None, ONE, 8, 2, 4, 8, 16, 1, 0, 1, NULL_STREAM]
    assert s(*args[:14], ONE, ONE, 8, 4097, 5000, *args[19:]) == -1
    for i, v in ((0, None), (2, None), (6, None), (8, None), (10, None), (13, None), (15, None), (17, -1), (17, 65536), (18, 1), (18, 0), (19, 0), (20, 0), (20, 65), (21, 3), (22, 4)):
        bad = list(args)
        bad[i] = v
        assert s(*bad) == -1, (i, v)


def test_python_refuses_cpu_tensors(L):
    from voice_converter_cyclegan_amd import sequence as S
    x, w = torch.zeros(2, 3, 8), torch.zeros(4, 8)
    with pytest.raises(ValueError, match='no CPU path'):
        S.rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match='no CPU path'):
        S.rms_norm_e4m3(x, torch.ones(8))
    with pytest.raises(ValueError, match='no CPU path'):
        S.causal_conv1d(x, w)
    with pytest.raises(ValueError, match='no CPU path'):
        S.causal_conv1d_step(x[0], torch.zeros(3, 3, 8), w)
    with pytest.raises(ValueError, match='no CPU path'):
        S.selective_scan(x, x, torch.zeros(8, 4), x[..., :4], x[..., :4])
    with pytest.raises(ValueError, match='no CPU path'):
        S.selective_scan_step(x[0], x[0], torch.zeros(8, 4), x[0, :, :4], x[0, :, :4], torch.zeros(3, 8, 4))


def test_conv_refuses_strides_beyond_a_block(L):
    """a block of the convolution reaches its rows with 32-bit offsets, so a stride of 2^30 elements is refused, and a negative one"""
    f, b = L.lib.vc_causal_conv1d_fwd, L.lib.vc_causal_conv1d_bwd
    big = 1 << 30
    for bad in (dict(x_ld=big), dict(y_ld=big), dict(x_ld=-8), dict(y_ld=-8)):
        assert f(C.byref(_conv(L, **bad)), NULL_STREAM) == -1, bad
        assert b'row stride' in L.lib.vc_last_error()
    full = dict(dy=4096, dx=4096, dx_ld=8, dy_ld=8)
    for bad in (dict(x_ld=big), dict(dy_ld=big), dict(dx_ld=big), dict(dx_ld=-8)):
        assert b(C.byref(_conv(L, **{**full, **bad})), NULL_STREAM) == -1, bad
        assert b'row stride' in L.lib.vc_last_error()


def test_binding_is_built_from_these_sources(L):
    from voice_converter_cyclegan_amd import sequence as S
    assert S._seq.build_id == L._bmod.binding_id()


def test_more_channels_than_an_index_holds_are_refused(L):
    """column indexes are 31 bits with room for what a thread steps over"""
    for cols in ((1 << 28) + 1, (1 << 31) - 1):
        assert L.lib.vc_rms_norm_fwd(ONE, cols, None, 0, ONE, ONE, cols, None, 0, None, 1e-6, 1, cols, 0, 0, NULL_STREAM) == -1
        assert L.lib.vc_rms_norm_bwd_work(1, cols) == -1
    for cols in ((1 << 24) + 1, (1 << 31) - 1):
        assert L.lib.vc_causal_conv1d_fwd(C.byref(_conv(L, cols=cols)), NULL_STREAM) == -1
        assert L.lib.vc_causal_conv1d_bwd_work(C.byref(_conv(L, cols=cols))) == -1
        assert L.lib.vc_causal_conv1d_step(ONE, cols, ONE, None, ONE, None, ONE, cols, 1, 1, cols, 4, 0, 1, NULL_STREAM) == -1
        assert L.lib.vc_selective_scan_fwd(C.byref(_scan(L, cols=cols)), NULL_STREAM) == -1
        assert L.lib.vc_selective_scan_step(ONE, cols, ONE, cols, None, 0, ONE, 16, ONE, 16, ONE, None, None, ONE, None, ONE, cols, 1, 1, cols, 16, 1, 0, 1, NULL_STREAM) == -1


def test_output_rows_that_overlap_are_refused(L):
    """rows of an output closer than their width would be written by several threads in no order; one row has no stride"""
    f, q, b = L.lib.vc_rms_norm_fwd, L.lib.vc_rms_norm_e4m3, L.lib.vc_rms_norm_bwd

    def fwd(x_ld=8, res_ld=8, y_ld=8, sum_ld=8, y=ONE, rows=4):
        return f(C.c_void_p(1 << 20), x_ld, C.c_void_p(1 << 21), res_ld, ONE, y, y_ld, C.c_void_p(1 << 22), sum_ld, None, 1e-6, rows, 8, 0, 0, NULL_STREAM)
    for bad in (dict(x_ld=-8), dict(res_ld=-1), dict(y_ld=7), dict(y_ld=0), dict(y_ld=-8), dict(sum_ld=7), dict(y=C.c_void_p(1 << 20), x_ld=9)):
        assert fwd(**bad) == -1 and b'row stride' in L.lib.vc_last_error(), bad
    assert q(ONE, 96, None, 0, ONE, ONE, 95, ONE, None, 0, 1e-6, 4, 96, 32, 0, 0, NULL_STREAM) == -1 and b'row stride' in L.lib.vc_last_error()
    args = [ONE, 8, ONE, 8, ONE, 8, ONE, ONE, ONE, 8, ONE, 8, None, None, 0, 4, 8, 0, 0, NULL_STREAM]
    for i, v in ((1, -8), (3, -8), (5, -8), (9, 7), (9, -8), (11, 7), (11, 0)):
        bad = list(args)
        bad[i] = v
        assert b(*bad) == -1 and b'row stride' in L.lib.vc_last_error(), (i, v)
    f, b = L.lib.vc_causal_conv1d_fwd, L.lib.vc_causal_conv1d_bwd
    for v in (0, 7):
        assert f(C.byref(_conv(L, y_ld=v)), NULL_STREAM) == -1 and b'row stride' in L.lib.vc_last_error()
        assert b(C.byref(_conv(L, dy=8192, dx=16384, dx_ld=v, dy_ld=8)), NULL_STREAM) == -1 and b'row stride' in L.lib.vc_last_error()
    s = L.lib.vc_causal_conv1d_step
    args = [ONE, 8, ONE, None, ONE, None, ONE, 8, 2, 4, 8, 4, 0, 1, NULL_STREAM]
    for i, v in ((1, -8), (7, 7), (7, 0), (7, -8)):
        bad = list(args)
        bad[i] = v
        assert s(*bad) == -1 and b'row stride' in L.lib.vc_last_error(), (i, v)
    s = L.lib.vc_selective_scan_step
    args = [ONE, 8, ONE, 8, ONE, 8, ONE, 16, ONE, 16, ONE, None, None, ONE, None, ONE, 8, 2, 4, 8, 16, 1, 0, 1, NULL_STREAM]
    for i, v in ((1, -8), (3, -8), (5, -8), (7, -1), (9, -1), (16, 7), (16, 0)):
        bad = list(args)
        bad[i] = v
        assert s(*bad) == -1 and b'row stride' in L.lib.vc_last_error(), (i, v)


def test_convolution_in_place_is_refused(L):
    """a run of rows looks at frames that another one writes to: its output may not be its input, nor a gradient what it is taken from"""
    f, b = L.lib.vc_causal_conv1d_fwd, L.lib.vc_causal_conv1d_bwd
    assert f(C.byref(_conv(L, y=4096)), NULL_STREAM) == -1 and b'in place' in L.lib.vc_last_error()
    full = dict(dy=8192, dx=16384, dx_ld=8, dy_ld=8, initial=1 << 20, dfinal=1 << 21, dinitial=1 << 22)
    for bad in (dict(dx=4096), dict(dx=8192), dict(dinitial=1 << 20), dict(dinitial=1 << 21)):
        assert b(C.byref(_conv(L, **{**full, **bad})), NULL_STREAM) == -1 and b'in place' in L.lib.vc_last_error(), bad
    a = dict(dy=4096, dx=4096, ddt=4096, dB=4096, dC=4096, dA=4096, saved=4096, saved_floats=1 << 20, work=4096, work_floats=1 << 20, dy_ld=8, dx_ld=8, ddt_ld=8, db_ld=16, dc_ld=16)
    assert L.lib.vc_selective_scan_bwd(C.byref(_scan(L, dinitial=1 << 20, dfinal=1 << 20, **a)), NULL_STREAM) == -1 and b'in place' in L.lib.vc_last_error()


@pytest.mark.parametrize('lacks', ['nothing', 'torch', 'a compiler', 'headers'])
def test_the_library_is_built_first_and_without_torch(L, monkeypatch, capsys, lacks):
    """the binding comes behind the C-ABI library, and what only the binding needs does not stop the library"""
    import importlib.util
    import sys
    spec = importlib.util.spec_from_file_location('_vcb', L._bmod.__file__)
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    done = []
    monkeypatch.setattr(b, 'build_library', lambda force, verbose: done.append('library') or b.LIB)
    monkeypatch.setattr(b, 'build_binding', lambda force, verbose: done.append('binding'))
    if lacks == 'torch':
        monkeypatch.setitem(sys.modules, 'torch', None)
    elif lacks == 'a compiler':
        monkeypatch.setenv('CXX', 'no-such-compiler')
    elif lacks == 'headers':
        import sysconfig
        monkeypatch.setattr(sysconfig, 'get_paths', lambda: {'include': '/nonexistent'})
    assert b.build() == b.LIB
    assert done == (['library', 'binding'] if lacks == 'nothing' else ['library'])
    assert ('not built' in capsys.readouterr().out) == (lacks != 'nothing')


def test_norm_gradient_workspace_goes_by_the_layout(L):
    """a row of dgamma's sums for each block: four rows a block up to 128 vectors, at most 1024 blocks, 256 where a block has 1024 threads (from 1025 vectors of
    16 bytes on; the larger of what fp32 and 16-bit rows take)"""
    for cols, few, many in ((512, 25, 1024), (1024, 100, 1024), (4096, 100, 1024), (8192, 100, 1024), (8200, 100, 256), (16384, 100, 256), (40000, 100, 256)):
        assert L.lib.vc_rms_norm_bwd_work(100, cols) == few * cols, cols
        assert L.lib.vc_rms_norm_bwd_work(1 << 20, cols) == many * cols, cols
