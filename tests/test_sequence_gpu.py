"""GPU: the sequence operators against the 64-bit oracle, through their public entry points.

Tolerances.  A result of type t may be off by half a step of t (finfo(t).eps / 2 of its value) for its one rounding, and by K * 2^-24 of its magnitude --
the same sum over absolute values, which the oracle gives -- for the fp32 arithmetic behind it, K being the number of roundings a term passes:
  norm    each thread adds up to cols / 64 squares, then 6 + 4 steps across lanes and waves, and a few products: cols / 64 + 20
  conv    taps products and sums, the bias, a sigmoid (exponential, reciprocal): taps + 20; its parameter gradients add over the rows as well
  scan    a term is carried by exp(delta A) from frame to frame, 3 roundings each (the exponential's two and the product), for as many frames as it
          lasts -- delta |A| >= 0.02 in these inputs, so 2^-24 of it is left after 17 / 0.02 = 850 frames; the argument's own error (10 units of
          delta |A|, softplus and two products) adds 10 s e^-s < 4 in all; then the sums over the states.  Backwards the same twice, and the sums over rows
          and channels.
Nothing here is fitted to results."""
import numpy as np
import pytest
import torch

import vcgan_pkg  # noqa: F401
from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = 'cuda:0'


@pytest.fixture(scope='module')
def S(built_lib):
    assert torch.cuda.is_available()
    from voice_converter_cyclegan_amd import sequence
    return sequence


def close(got, ref, mag, k, name=''):
    got64, ref, mag = got.detach().cpu().double(), ref.double(), mag.double()
    assert got64.shape == ref.shape, (name, got64.shape, ref.shape)
    info = torch.finfo(got.dtype)
    half = 0.0 if got.dtype == F32 else info.eps / 2
    tol = half * ref.abs() + k * U * mag * (1 + half) + (info.smallest_normal * info.eps if got.dtype == F16 else 1e-37)
    bad = ~((got64 - ref).abs() <= tol)
    assert not bad.any(), '%s: %d of %d off, worst %.3g of its tolerance' % (name, int(bad.sum()), bad.numel(), float(((got64 - ref).abs() / tol).max()))


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------------------------------------ norm

NORM_SHAPES = [(1, 1), (1, 512), (3, 7), (5, 64), (2, 1001), (130, 1024), (7, 2048), (3, 2056), (4, 8192), (2, 8200), (2, 20001)]


@pytest.mark.parametrize('rows,cols', NORM_SHAPES)
@pytest.mark.parametrize('kind,stream', [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_norm_and_gradient(S, rows, cols, kind, stream):
    x, res = rnd(1, rows, cols, dtype=kind), rnd(2, rows, cols, dtype=stream, scale=3.0)
    gamma = 1 + rnd(3, cols, scale=0.1)
    dy, ds = rnd(4, rows, cols, dtype=kind), rnd(5, rows, cols, dtype=stream)
    for t in (x, res, gamma):
        t.requires_grad_(True)
    y, total = S.rms_norm(x, gamma, res, eps=1e-5)
    want_total = (x.detach().float() + res.detach().float()).to(stream)
    assert torch.equal(total.detach(), want_total)
    k = cols / 64 + 20
    ref, dt, dgamma = O.rms_norm(want_total, gamma, 1e-5, dy, ds)
    _, dt_m, dgamma_m = O.rms_norm(want_total, gamma, 1e-5, dy, ds, absolute=True)
    close(y, ref, ref.abs(), k, 'y')
    dx, dres, dg = torch.autograd.grad((y, total), (x, res, gamma), (dy, ds))
    close(dx, dt, dt_m, 3 * k, 'dx')
    close(dres, dt, dt_m, 3 * k, 'dres')
    close(dg, dgamma, dgamma_m, k + rows, 'dgamma')


@pytest.mark.parametrize('kind', [F32, BF16])
def test_norm_without_residual_and_partial_gradients(S, kind):
    x, gamma, dy = rnd(1, 4, 9, 100, dtype=kind), 1 + rnd(2, 100, scale=0.1), rnd(3, 4, 9, 100, dtype=kind)
    ref, dt, dgamma = O.rms_norm(x.view(36, 100), gamma, 1e-6, dy.view(36, 100))
    _, dt_m, dg_m = O.rms_norm(x.view(36, 100), gamma, 1e-6, dy.view(36, 100), absolute=True)
    with torch.no_grad():
        close(S.rms_norm(x, gamma).view(36, 100), ref, ref.abs(), 22)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(S.rms_norm(x, gamma), x, dy)
    close(dx.view(36, 100), dt, dt_m, 66)
    x.requires_grad_(False)
    gamma.requires_grad_(True)
    (dg,) = torch.autograd.grad(S.rms_norm(x, gamma), gamma, dy)
    close(dg, dgamma, dg_m, 60)


def test_norm_only_the_sum_has_a_gradient(S):
    x, res, gamma = rnd(1, 5, 64).requires_grad_(True), rnd(2, 5, 64).requires_grad_(True), torch.ones(64, device=DEV)
    _, total = S.rms_norm(x, gamma, res)
    d = rnd(3, 5, 64)
    dx, dr = torch.autograd.grad(total, (x, res), d)
    assert torch.equal(dx, d) and torch.equal(dr, d)


@pytest.mark.parametrize('kind,stream', [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize('rows,cols,group', [(1, 64, 0), (3, 1000, 0), (5, 96, 32), (130, 1024, 128), (4, 2048, 64), (9, 4224, 128), (2, 9000, 0), (2, 20032, 64), (2, 20001, 0)])
def test_norm_e4m3(S, kind, stream, rows, cols, group):
    x, res, gamma = rnd(1, rows, cols, dtype=kind), rnd(2, rows, cols, dtype=stream, scale=3.0), 1 + rnd(3, cols, scale=0.1)
    q, scale, total = S.rms_norm_e4m3(x, gamma, res, eps=1e-5, group=group)
    want_total = (x.float() + res.float()).to(stream)
    assert torch.equal(total, want_total) and q.dtype == torch.float8_e4m3fn and scale.shape == (rows, cols // group if group else 1)
    y = O.rms_norm(want_total, gamma, 1e-5)
    k = cols / 64 + 24
    top = y.view(rows, -1, group or cols).abs().amax(-1)
    close(scale, top / 448, top / 448, k, 'scale')
    # a value is off by half a step of e4m3 (2^-4 of it, 2^-10 scales below the normal range), and the y it rounds by the arithmetic before it
    wide = scale.double().cpu().repeat_interleave(group or cols, 1)
    err = (q.float().double().cpu() * wide - y).abs()
    assert (err <= y.abs() * (2.0 ** -4 + k * U) + wide * 2.0 ** -10).all(), float(err.max())
    assert q.float().abs().max() <= 448


def test_norm_e4m3_zeros_and_non_numbers(S):
    x = rnd(1, 4, 256)
    x[0] = 0
    x[1, 130] = float('nan')
    gamma = torch.ones(256, device=DEV)
    q, scale = S.rms_norm_e4m3(x, gamma, group=128)
    v = q.float().view(4, 2, 128) * scale[..., None]
    assert (v[0] == 0).all() and torch.isfinite(scale[0]).all()
    assert torch.isnan(v[1]).all()                                # the row's mean square is no number
    assert torch.isfinite(v[2:]).all()
    gamma2 = gamma.clone()
    gamma2[200] = float('inf')
    q, scale = S.rms_norm_e4m3(rnd(2, 1, 256), gamma2, group=128)
    assert torch.isfinite(scale[0, 0]) and not torch.isfinite(scale[0, 1])


def test_norm_zero_row_and_in_place_buffers(S):
    x = torch.zeros(2, 32, device=DEV, requires_grad=True)
    gamma = torch.ones(32, device=DEV, requires_grad=True)
    y = S.rms_norm(x, gamma, eps=1e-6)
    assert (y == 0).all()
    dx, dg = torch.autograd.grad(y, (x, gamma), torch.ones_like(y))
    assert torch.allclose(dx, torch.full_like(dx, 1e3)) and (dg == 0).all()


# ----------------------------------------------------------------------------------------------------------- convolution

LENGTHS = [[1], [5], [3, 3, 3], [0, 1, 2, 0, 7, 40], [17, 64, 65, 1], [150]]


def offsets_of(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32), device=DEV)


@pytest.mark.parametrize('lengths', LENGTHS)
@pytest.mark.parametrize('cols,taps,kind,silu', [(1, 2, F32, True), (24, 4, F32, False), (300, 4, BF16, True), (257, 3, F16, True), (64, 8, F32, True), (1030, 4, BF16, True)])
def test_conv_packed_with_states_and_a_tail(S, lengths, cols, taps, kind, silu):
    n, live = len(lengths), sum(lengths)
    rows = live + 3                                              # three rows behind the last utterance, which nothing may read
    x, w, b = rnd(1, rows, cols, dtype=kind), rnd(2, taps, cols, scale=taps ** -0.5), rnd(3, cols, scale=0.1)
    x[live:] = float('nan')
    init = rnd(4, n, taps - 1, cols, dtype=kind)
    dy, df = rnd(5, rows, cols, dtype=kind), rnd(6, n, taps - 1, cols, dtype=kind)
    dy[live:] = float('nan')
    leaves = [t.requires_grad_(True) for t in (x, w, b, init)]
    y, final = S.causal_conv1d(x, w, b, initial_state=init, seq_offsets=offsets_of(lengths), silu=silu, return_final_state=True)
    xc, dyc = x.detach().cpu(), dy.cpu().clone()
    xc[live:], dyc[live:] = 0, 0
    r = O.conv1d(xc, w, b, init, lengths, silu, dyc, df)
    m = O.conv1d(xc, w, b, init, lengths, silu, dyc, df, absolute=True)
    close(y, r['y'], m['p'], taps + 20, 'y')
    assert (y[live:] == 0).all()
    assert torch.equal(final.detach().double().cpu(), r['final'])
    dx, dw, db, di = torch.autograd.grad((y, final), leaves, (dy, df))
    close(dx, r['dx'], m['dx'], taps + 20, 'dx')
    assert (dx[live:] == 0).all()
    close(di, r['dinitial'], m['dinitial'], taps + 20, 'dinitial')
    close(dw, r['dw'], m['dw'], taps + 20 + live, 'dw')
    close(db, r['dbias'], m['dbias'], taps + 20 + live, 'dbias')


@pytest.mark.parametrize('kind', [F32, BF16])
def test_conv_batch_without_states(S, kind):
    x, w = rnd(1, 5, 33, 130, dtype=kind), rnd(2, 4, 130, scale=0.5)
    dy = rnd(3, 5, 33, 130, dtype=kind)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = S.causal_conv1d(x, w)
    flat = x.detach().view(-1, 130)
    r = O.conv1d(flat, w, None, None, [33] * 5, True, dy.view(-1, 130))
    m = O.conv1d(flat, w, None, None, [33] * 5, True, dy.view(-1, 130), absolute=True)
    close(y.view(-1, 130), r['y'], m['p'], 24, 'y')
    dx, dw = torch.autograd.grad(y, leaves, dy)
    close(dx.view(-1, 130), r['dx'], m['dx'], 24, 'dx')
    close(dw, r['dw'], m['dw'], 24 + 165, 'dw')


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('cols', [5, 264])
def test_conv_steps_equal_the_prompt(S, kind, cols):
    n, t, taps = 3, 9, 4
    x, w, b = rnd(1, n, t, cols, dtype=kind), rnd(2, taps, cols, scale=0.5), rnd(3, cols)
    init = rnd(4, n, taps - 1, cols, dtype=kind)
    y, final = S.causal_conv1d(x, w, b, initial_state=init, return_final_state=True)
    pool = rnd(5, 7, taps - 1, cols, dtype=kind)
    untouched = pool.clone()
    slots = torch.tensor([6, 0, 3], dtype=torch.int32, device=DEV)
    pool[slots.long()] = init
    m = O.conv1d(x.view(-1, cols), w, b, init, [t] * n, True, absolute=True)['p'].view(n, t, cols)
    for i in range(t):
        yi = S.causal_conv1d_step(x[:, i], pool, w, b, slots=slots)
        close(yi, y[:, i].cpu().double(), m[:, i] + (0 if kind == F32 else torch.finfo(kind).eps / U * y[:, i].cpu().double().abs()), 48, 'frame %d' % i)
    assert torch.equal(pool[slots.long()], final)
    for i in (1, 2, 4, 5):
        assert torch.equal(pool[i], untouched[i])


# ------------------------------------------------------------------------------------------------------------------ scan

def scan_inputs(rows, cols, states, groups, kind, seqs, seed=1):
    g = torch.Generator().manual_seed(seed)
    step = torch.exp(torch.rand(cols, generator=g) * 2.3 - 3.0)                  # 0.05 .. 0.5
    A = -(0.4 + torch.rand(cols, states, generator=g) * 4)
    v = dict(x=rnd(seed + 1, rows, cols, dtype=kind), dt=rnd(seed + 2, rows, cols, dtype=kind).clamp(-0.1, 0.5), A=A.to(DEV),
             B=rnd(seed + 3, rows, groups, states, dtype=kind), C=rnd(seed + 4, rows, groups, states, dtype=kind), D=rnd(seed + 5, cols),
             z=rnd(seed + 6, rows, cols, dtype=kind), dt_bias=(step + torch.log(-torch.expm1(-step))).to(DEV),
             initial=rnd(seed + 7, seqs, cols, states))
    return v


def lasts(r, A, rows):
    """frames a term of the recurrence lasts: until 2^-24 of it is left"""
    weakest = float(r['delta'].abs().min() * A.detach().abs().min())
    return min(rows, 17 / max(weakest, 1e-9))


SCAN_SHAPES = [(4, 1, 1), (5, 3, 1), (16, 16, 1), (100, 16, 2), (130, 16, 1), (24, 21, 3), (12, 32, 1), (7, 64, 1), (10, 50, 2), (64, 8, 1), (33, 12, 1)]


@pytest.mark.parametrize('lengths', LENGTHS)
@pytest.mark.parametrize('cols,states,groups', SCAN_SHAPES)
def test_scan_packed_with_states_and_a_tail(S, lengths, cols, states, groups):
    kind = [F32, BF16, F16][(cols + len(lengths)) % 3]
    n, live = len(lengths), sum(lengths)
    rows = live + 5
    v = scan_inputs(rows, cols, states, groups, kind, n)
    for k in ('x', 'dt', 'z', 'B', 'C'):
        v[k][live:] = float('nan')
    dy, df = rnd(20, rows, cols, dtype=kind), rnd(21, n, cols, states)
    dy[live:] = float('nan')
    leaves = [t.requires_grad_(True) for t in v.values()]
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of(lengths), return_final_state=True)
    clean = {k: t.detach().cpu().clone() for k, t in v.items()}
    dyc = dy.cpu().clone()
    for t in [clean[k] for k in ('x', 'dt', 'z', 'B', 'C')] + [dyc]:
        t[live:] = 0
    r = O.scan(**clean, lengths=lengths, dy=dyc, dfinal=df)
    m = O.scan(**clean, lengths=lengths, dy=dyc, dfinal=df, absolute=True)
    last = lasts(r, v['A'], max(lengths))
    k = 3 * last + states + 40
    close(y, r['y'], m['y'], k, 'y')
    assert (y[live:] == 0).all()
    close(final, r['final'], m['final'], k, 'final')
    grads = torch.autograd.grad((y, final), leaves, (dy, df))
    k = 6 * last + rows + cols + states + 60
    for (name, _), got in zip(v.items(), grads):
        close(got, r['d' + name], m['d' + name], k, 'd' + name)
    for name, got in zip(v, grads):
        if name in ('x', 'dt', 'z', 'B', 'C'):
            assert (got[live:] == 0).all(), name


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('softplus', [True, False])
def test_scan_batch_without_extras(S, kind, softplus):
    n, t, cols, states = 6, 37, 70, 16
    v = scan_inputs(n * t, cols, states, 1, kind, n)
    if not softplus:
        v['dt'] = v['dt'].abs() * 0.3 + 0.05
    dy = rnd(20, n, t, cols, dtype=kind)
    use = {k: v[k].view(n, t, -1) if k in ('x', 'dt') else v[k].view(n, t, states) if k in 'BC' else v[k] for k in ('x', 'dt', 'A', 'B', 'C')}
    leaves = [u.requires_grad_(True) for u in use.values()]
    y = S.selective_scan(*use.values(), softplus=softplus)
    plain = dict(x=v['x'], dt=v['dt'], A=v['A'], B=v['B'], C=v['C'], D=None, z=None, dt_bias=None, initial=None, lengths=[t] * n, softplus=softplus, dy=dy.view(-1, cols))
    r, m = O.scan(**plain), O.scan(**plain, absolute=True)
    last = lasts(r, v['A'], t)
    close(y.view(-1, cols), r['y'], m['y'], 3 * last + 56, 'y')
    for name, got in zip(use, torch.autograd.grad(y, leaves, dy)):
        close(got.reshape(r['d' + name].shape), r['d' + name], m['d' + name], 6 * last + n * t + cols + 76, 'd' + name)


@pytest.mark.parametrize('cols,states,kind', [(32, 16, F32), (20, 40, BF16)])
@pytest.mark.parametrize('lengths,hint', [([1500], None), ([700, 3, 0, 800, 16], None), ([700, 3, 0, 800, 16], 800), ([31] * 40, 31), ([31] * 40, None)])
def test_scan_long_and_many(S, cols, states, kind, lengths, hint):
    """long axes that are split, and many short utterances; with the longest one told and not"""
    n, rows = len(lengths), sum(lengths)
    v = scan_inputs(rows, cols, states, 1, kind, n)
    dy, df = rnd(20, rows, cols, dtype=kind), rnd(21, n, cols, states)
    leaves = [t.requires_grad_(True) for t in v.values()]
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of(lengths), max_len=hint, return_final_state=True)
    r = O.scan(**v, lengths=lengths, dy=dy, dfinal=df)
    m = O.scan(**v, lengths=lengths, dy=dy, dfinal=df, absolute=True)
    last = lasts(r, v['A'], max(lengths))
    close(y, r['y'], m['y'], 3 * last + states + 40, 'y')
    close(final, r['final'], m['final'], 3 * last + states + 40, 'final')
    for (name, _), got in zip(v.items(), torch.autograd.grad((y, final), leaves, (dy, df))):
        close(got, r['d' + name], m['d' + name], 6 * last + rows + cols + states + 60, 'd' + name)


def test_scan_of_many_short_utterances(S):
    """more utterances than any split has parts: runs that hold many of them, some of no frames, one long at the end"""
    g = torch.Generator().manual_seed(4)
    lengths = torch.randint(0, 4, (5000,), generator=g).tolist() + [90]
    n, rows, cols = len(lengths), sum(lengths), 5
    v = scan_inputs(rows, cols, 4, 1, F32, n)
    dy, df = rnd(20, rows, cols), rnd(21, n, cols, 4)
    leaves = [t.requires_grad_(True) for t in v.values()]
    for hint in (None, 90):
        y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                    seq_offsets=offsets_of(lengths), max_len=hint, return_final_state=True)
        r = O.scan(**v, lengths=lengths, dy=dy, dfinal=df)
        m = O.scan(**v, lengths=lengths, dy=dy, dfinal=df, absolute=True)
        close(y, r['y'], m['y'], 3 * 90 + 44, 'y')
        close(final, r['final'], m['final'], 3 * 90 + 44, 'final')
        for (name, _), got in zip(v.items(), torch.autograd.grad((y, final), leaves, (dy, df))):
            close(got, r['d' + name], m['d' + name], 6 * 90 + rows + cols + 64, 'd' + name)


def test_scan_that_grows(S):
    """A > 0: states grow by e^0.05 a frame, over 3000 frames further than fp32 reaches; while nothing has come in they stay zero, and what is small enough
    stays finite, also where a run's whole factor is not.  Errors relative to what has grown: 3 roundings a frame and 50 units of the exponent's sum."""
    t, cols = 3000, 8
    x = torch.zeros(1, t, cols, device=DEV)
    x[0, 1400:] = rnd(1, t - 1400, cols) * 1e-20
    dt = torch.full((1, t, cols), 0.05, device=DEV)
    A, bc = torch.ones(cols, 4, device=DEV), torch.ones(1, t, 4, device=DEV)
    y, final = S.selective_scan(x, dt, A, bc, bc, softplus=False, return_final_state=True)
    r = O.scan(x[0], dt[0], A, bc[0, :, None], bc[0, :, None], None, None, None, None, [t], softplus=False)
    m = O.scan(x[0], dt[0], A, bc[0, :, None], bc[0, :, None], None, None, None, None, [t], softplus=False, absolute=True)
    assert (y[0, :1400] == 0).all() and torch.isfinite(r['y'].float()).all()
    close(y[0], r['y'], m['y'], 3 * 1600 + 50 * 80, 'y')
    close(final, r['final'], m['final'], 3 * 1600 + 50 * 80, 'final')


@pytest.mark.parametrize('kind', [F32, BF16])
@pytest.mark.parametrize('cols,states,groups', [(6, 16, 1), (130, 16, 2), (9, 5, 3), (10, 64, 1)])
def test_scan_steps_equal_the_prompt(S, kind, cols, states, groups):
    n, t = 3, 11
    v = scan_inputs(n * t, cols, states, groups, kind, n)
    b = {k: v[k].view(n, t, *v[k].shape[1:]) for k in ('x', 'dt', 'z', 'B', 'C')}
    y, final = S.selective_scan(b['x'], b['dt'], v['A'], b['B'], b['C'], D=v['D'], z=b['z'], dt_bias=v['dt_bias'], initial_state=v['initial'], return_final_state=True)
    r = O.scan(**v, lengths=[t] * n)
    m = O.scan(**v, lengths=[t] * n, absolute=True)
    pool = rnd(30, 8, cols, states)
    was = pool.clone()
    slots = torch.tensor([5, 1, 7], dtype=torch.int32, device=DEV)
    pool[slots.long()] = v['initial']
    k = 3 * t + states + 40
    for i in range(t):
        yi = S.selective_scan_step(b['x'][:, i], b['dt'][:, i], v['A'], b['B'][:, i], b['C'][:, i], pool, D=v['D'], z=b['z'][:, i], dt_bias=v['dt_bias'], slots=slots)
        close(yi, r['y'].view(n, t, cols)[:, i], m['y'].view(n, t, cols)[:, i], k, 'frame %d' % i)
    close(pool[slots.long()], r['final'], m['final'], k, 'state')
    close(final, r['final'], m['final'], k, 'final')
    for i in (0, 2, 3, 4, 6):
        assert torch.equal(pool[i], was[i])


def test_steps_treat_strange_slots_as_padding(S):
    cols, states = 40, 16
    v = scan_inputs(6, cols, states, 1, F32, 1)
    slots = torch.tensor([2, -1, 2, 9, 0, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    pool = rnd(5, 4, cols, states)
    alone = pool.clone()
    args = [v[k] for k in ('x', 'dt', 'A')] + [v['B'][:, 0], v['C'][:, 0]]
    y = S.selective_scan_step(*args, pool, D=v['D'], z=v['z'], dt_bias=v['dt_bias'], slots=slots)
    keep = [0, 4]
    rows = [a[keep] if a.shape[0] == 6 else a for a in (args[0], args[1])] + [args[2], args[3][keep], args[4][keep]]
    y2 = S.selective_scan_step(*rows, alone, D=v['D'], z=v['z'][keep], dt_bias=v['dt_bias'], slots=slots[keep].contiguous())
    assert torch.equal(y[keep], y2) and torch.equal(pool, alone)
    assert (y[[1, 2, 3, 5]] == 0).all()
    w, cpool = rnd(6, 4, cols), rnd(7, 4, 3, cols)
    calone = cpool.clone()
    y = S.causal_conv1d_step(v['x'], cpool, w, slots=slots)
    y2 = S.causal_conv1d_step(v['x'][keep], calone, w, slots=slots[keep].contiguous())
    assert torch.equal(y[keep], y2) and torch.equal(cpool, calone) and (y[[1, 2, 3, 5]] == 0).all()


def test_a_non_number_stays_in_its_utterance(S):
    lengths, cols = [20, 9, 33], 24
    v = scan_inputs(62, cols, 16, 1, F32, 3)
    w = rnd(9, 4, cols)
    off = offsets_of(lengths)

    def go():
        leaves = [t.detach().clone().requires_grad_(True) for t in v.values()]
        u = dict(zip(v, leaves))
        c = S.causal_conv1d(u['x'], w, seq_offsets=off)
        y = S.selective_scan(c, u['dt'], u['A'], u['B'], u['C'], D=u['D'], z=u['z'], dt_bias=u['dt_bias'], initial_state=u['initial'], seq_offsets=off)
        g = torch.autograd.grad(y, [u[k] for k in ('x', 'dt', 'z', 'B', 'C', 'initial')], torch.ones_like(y))
        return y, g
    y0, g0 = go()
    v['x'][22] = float('nan')
    v['initial'][1, 3] = float('inf')
    y1, g1 = go()
    out = torch.cat([torch.arange(20), torch.arange(29, 62)]).to(DEV)
    assert torch.isnan(y1[22:29]).any()
    assert torch.equal(y0[out], y1[out])
    for a, b in zip(g0[:5], g1[:5]):
        assert torch.equal(a[out], b[out])
    assert torch.equal(g0[5][[0, 2]], g1[5][[0, 2]])


# ---------------------------------------------------------------------------------------------- how the calls may be made

def layer(S, p, stream, off=None, states=None):
    """a residual layer of the operators: norm -> product -> short convolution -> product -> scan (gated) -> product"""
    cols, n = p['A'].shape
    y, stream = S.rms_norm(p['x'] if stream is None else stream[0], p['gamma'], p['stream'] if stream is None else stream[1])
    xz = y @ p['Win']
    pack = dict(seq_offsets=off) if off is not None else {}
    u = S.causal_conv1d(xz[..., :cols], p['w'], p['bias'], **pack)
    s = u @ p['Wx']
    v = S.selective_scan(u, s[..., 2 * n:] @ p['Wdt'], p['A'], s[..., :n], s[..., n:2 * n], D=p['D'], z=xz[..., cols:], dt_bias=p['dt_bias'], **pack)
    return v @ p['Wout'], stream


def layer_parameters(width=40, cols=72, n=16, rank=6):
    v = scan_inputs(1, cols, n, 1, F32, 1)
    return dict(gamma=1 + rnd(1, width, scale=0.1), Win=rnd(2, width, 2 * cols, scale=width ** -0.5), w=rnd(3, 4, cols, scale=0.5), bias=rnd(4, cols, scale=0.1),
                Wx=rnd(5, cols, 2 * n + rank, scale=cols ** -0.5), Wdt=rnd(6, rank, cols, scale=0.3), A=v['A'], D=v['D'], dt_bias=v['dt_bias'],
                Wout=rnd(7, cols, width, scale=cols ** -0.5))


def plain_layer(p, x, stream, lengths):
    """the same in 64 bits on the CPU, with torch's autograd"""
    cols, n = p['A'].shape
    t = x + stream
    y = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * p['gamma']
    xz = y @ p['Win']
    outs, at = [], 0
    for m in lengths:
        axis = torch.cat([torch.zeros(3, cols, dtype=torch.float64), xz[at:at + m, :cols]])
        c = sum(axis[j:j + m] * p['w'][j] for j in range(4)) + p['bias']
        u = c * torch.sigmoid(c)
        s = u @ p['Wx']
        delta = torch.logaddexp(s[:, 2 * n:] @ p['Wdt'] + p['dt_bias'], torch.zeros((), dtype=torch.float64))
        h, ys = torch.zeros(cols, n, dtype=torch.float64), []
        for i in range(m):
            h = torch.exp(delta[i][:, None] * p['A']) * h + (delta[i] * u[i])[:, None] * s[i, :n]
            ys.append((h * s[i, n:2 * n]).sum(-1) + p['D'] * u[i])
        z = xz[at:at + m, cols:]
        outs.append(torch.stack(ys) * z * torch.sigmoid(z) if m else z)
        at += m
    return torch.cat(outs) @ p['Wout'], t


def test_a_layer_of_them_trains_like_its_definition(S):
    """norm, convolution and scan together, packed, with column slices of products as inputs: outputs and every gradient.  Tolerance: the three operators'
    and four products' roundings follow one another; each passes on the relative error of what it is given with a factor that the magnitudes here keep
    near one (norms of results and gradients are compared), so 200 roundings of 2^-24 a stage over 8 stages: 1e-4 of the largest element."""
    lengths = [19, 0, 40, 1]
    p = layer_parameters()
    p.update(x=rnd(20, 60, 40), stream=rnd(21, 60, 40))
    leaves = {k: t.requires_grad_(True) for k, t in p.items()}
    out, stream = layer(S, p, None, offsets_of(lengths))
    d1, d2 = rnd(22, 60, 40), rnd(23, 60, 40)
    got = torch.autograd.grad((out, stream), list(leaves.values()), (d1, d2))
    q = {k: t.detach().cpu().double().requires_grad_(True) for k, t in p.items()}
    ref, rs = plain_layer(q, q['x'], q['stream'], lengths)
    want = torch.autograd.grad((ref, rs), list(q.values()), (d1.cpu().double(), d2.cpu().double()))
    assert (out.detach().cpu().double() - ref.detach()).abs().max() <= 1e-4 * ref.detach().abs().max()
    for k, a, b in zip(leaves, got, want):
        assert (a.cpu().double() - b).abs().max() <= 1e-4 * b.abs().max(), k


def test_streaming_a_layer_frame_by_frame_equals_the_recording(S):
    """the same layer on a live stream: single-frame calls with carried states against one call over all frames (same stages, same tolerance)"""
    n, t, width = 2, 25, 40
    p = layer_parameters()
    cols, ns = p['A'].shape
    p.update(x=rnd(20, n, t, width), stream=rnd(21, n, t, width))
    out, _ = layer(S, p, None)
    conv, state = torch.zeros(n, 3, cols, device=DEV), torch.zeros(n, cols, ns, device=DEV)
    for i in range(t):
        y, _ = S.rms_norm(p['x'][:, i], p['gamma'], p['stream'][:, i])
        xz = y @ p['Win']
        u = S.causal_conv1d_step(xz[:, :cols], conv, p['w'], p['bias'])
        s = u @ p['Wx']
        v = S.selective_scan_step(u, s[:, 2 * ns:] @ p['Wdt'], p['A'], s[:, :ns], s[:, ns:2 * ns], state, D=p['D'], z=xz[:, cols:], dt_bias=p['dt_bias'])
        assert (v @ p['Wout'] - out[:, i]).abs().max() <= 1e-4 * out.abs().max(), i


def test_strided_transposed_and_repeated_inputs(S):
    """column slices, a time-contiguous tensor seen as frames, and one row for all: the same numbers as contiguous copies"""
    rows, cols = 50, 36
    wide = rnd(1, rows, 3 * cols + 5)
    x, dt, z = wide[:, 1:cols + 1], wide[:, cols + 2:2 * cols + 2], wide[:, 2 * cols + 4:3 * cols + 4]
    v = scan_inputs(rows, cols, 16, 1, F32, 1)
    bc = rnd(2, rows, 40)
    B, Cm = bc[:, 3:19], bc[:, 20:36]
    off = offsets_of([20, 30])
    a = S.selective_scan(x, dt, v['A'], B, Cm, D=v['D'], z=z, dt_bias=v['dt_bias'], seq_offsets=off)
    b = S.selective_scan(x.contiguous(), dt.contiguous(), v['A'], B.contiguous(), Cm.contiguous(), D=v['D'], z=z.contiguous(), dt_bias=v['dt_bias'], seq_offsets=off)
    assert torch.equal(a, b)
    w = rnd(3, 4, cols)
    assert torch.equal(S.causal_conv1d(x, w, seq_offsets=off), S.causal_conv1d(x.contiguous(), w, seq_offsets=off))
    frames = rnd(4, 2, cols, 25).transpose(1, 2)                  # [batch, frames, channels] of a [batch, channels, frames] tensor
    assert torch.equal(S.causal_conv1d(frames, w), S.causal_conv1d(frames.contiguous(), w))
    gamma = torch.ones(cols, device=DEV)
    assert torch.equal(S.rms_norm(frames, gamma), S.rms_norm(frames.contiguous(), gamma))
    one = rnd(5, 1, cols).expand(rows, cols)
    assert torch.equal(S.rms_norm(one, gamma, x)[0], S.rms_norm(one.contiguous(), gamma, x)[0])
    leaf = rnd(6, 1, cols).requires_grad_(True)                   # gradient of a row that all rows share
    (g,) = torch.autograd.grad(S.causal_conv1d(leaf.expand(rows, cols), w, seq_offsets=off).sum(), leaf)
    many = leaf.detach().repeat(rows, 1).requires_grad_(True)
    (h,) = torch.autograd.grad(S.causal_conv1d(many, w, seq_offsets=off).sum(), many)
    assert torch.allclose(g, h.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_two_runs_are_bitwise_equal(S):
    lengths = [300, 45, 200]
    v = scan_inputs(545, 150, 16, 1, BF16, 3)
    dy = rnd(20, 545, 150, dtype=BF16)

    def go():
        u = {k: t.detach().clone().requires_grad_(True) for k, t in v.items()}
        w = rnd(9, 4, 150).requires_grad_(True)
        gamma = torch.ones(150, device=DEV, requires_grad=True)
        c = S.causal_conv1d(S.rms_norm(u['x'], gamma), w, seq_offsets=offsets_of(lengths))
        y = S.selective_scan(c, u['dt'], u['A'], u['B'], u['C'], D=u['D'], z=u['z'], dt_bias=u['dt_bias'], initial_state=u['initial'], seq_offsets=offsets_of(lengths))
        return torch.autograd.grad(y, list(u.values()) + [w, gamma], dy)
    for a, b in zip(go(), go()):
        assert torch.equal(a, b)


def test_empty_calls(S):
    w, A = rnd(1, 4, 8), -torch.ones(8, 4, device=DEV)
    none = torch.empty(2, 0, 8, device=DEV)
    bc = torch.empty(2, 0, 4, device=DEV)
    init, h0 = rnd(2, 2, 3, 8), rnd(3, 2, 8, 4)
    y, f = S.causal_conv1d(none, w, initial_state=init, return_final_state=True)
    assert y.shape == none.shape and torch.equal(f, init)
    y, f = S.selective_scan(none, none, A, bc, bc, initial_state=h0, return_final_state=True)
    assert y.shape == none.shape and torch.equal(f, h0)
    assert S.rms_norm(none, torch.ones(8, device=DEV)).shape == none.shape
    assert S.rms_norm_e4m3(none, torch.ones(8, device=DEV))[1].shape == (2, 0, 1)
    row = torch.empty(0, 8, device=DEV)
    assert S.causal_conv1d_step(row, init, w).shape == (0, 8)
    assert S.selective_scan_step(row, row, A, row[:, :4], row[:, :4], h0).shape == (0, 8)
    leaves = [t.detach().clone().requires_grad_(True) for t in (none, w, A, init, h0)]
    y, f = S.selective_scan(S.causal_conv1d(leaves[0], leaves[1], initial_state=leaves[3]), leaves[0], leaves[2], bc, bc, initial_state=leaves[4], return_final_state=True)
    g = torch.autograd.grad((y, f), leaves, (y.detach(), torch.ones_like(f)))
    assert g[0].shape == none.shape and (g[1] == 0).all() and (g[2] == 0).all() and (g[3] == 0).all() and (g[4] == 1).all()
    x, gamma = none.clone().requires_grad_(True), torch.ones(8, device=DEV, requires_grad=True)
    assert (torch.autograd.grad(S.rms_norm(x, gamma).sum(), gamma)[0] == 0).all()


def test_refusals(S):
    x, w = rnd(1, 2, 5, 8), rnd(2, 4, 8)
    A, bc = -torch.ones(8, 4, device=DEV), rnd(3, 2, 5, 4)
    ok = dict(A=A, B=bc, C=bc)

    def no(f, *a, **k):
        with pytest.raises((ValueError, RuntimeError)):
            f(*a, **k)
    no(S.rms_norm, x.double(), torch.ones(8, device=DEV))
    no(S.rms_norm, x, torch.ones(7, device=DEV))
    no(S.rms_norm, x, torch.ones(8, device=DEV, dtype=BF16))
    no(S.rms_norm, x, torch.ones(8))
    no(S.rms_norm, x, torch.ones(8, device=DEV), x[:1])
    no(S.rms_norm, x, torch.ones(8, device=DEV), x.bfloat16())
    no(S.rms_norm, x, torch.ones(8, device=DEV), eps=0.0)
    no(S.rms_norm_e4m3, x, torch.ones(8, device=DEV), group=32)
    no(S.rms_norm_e4m3, x, torch.ones(8, device=DEV, requires_grad=True))
    no(S.causal_conv1d, x[0], w)                                  # rows without seq_offsets
    no(S.causal_conv1d, x, w[:1])
    no(S.causal_conv1d, x, rnd(4, 9, 8))
    no(S.causal_conv1d, x, w.bfloat16())
    no(S.causal_conv1d, x, w, initial_state=rnd(5, 2, 4, 8))
    no(S.causal_conv1d, x, w, seq_offsets=torch.tensor([0, 5], dtype=torch.int32, device=DEV))
    no(S.causal_conv1d, x[0], w, seq_offsets=torch.tensor([0, 5], device=DEV))
    no(S.causal_conv1d, x[0], w, seq_offsets=torch.tensor([0, 5], dtype=torch.int32))
    no(S.causal_conv1d, x[0], w, seq_offsets=torch.tensor([5], dtype=torch.int32, device=DEV))
    no(S.causal_conv1d_step, x[:, 0], rnd(6, 1, 3, 8), w)         # two streams, one state
    no(S.causal_conv1d_step, x[:, 0], rnd(6, 4, 3, 16)[..., ::2], w)
    no(S.causal_conv1d_step, x[:, 0].clone().requires_grad_(True), rnd(6, 4, 3, 8), w)
    no(S.causal_conv1d_step, x[:, 0], rnd(6, 4, 3, 8), w, slots=torch.tensor([0, 1], device=DEV))
    no(S.selective_scan, x, x[:, :4], **ok)
    no(S.selective_scan, x, x.bfloat16(), **ok)
    no(S.selective_scan, x, x, A[:7], bc, bc)
    no(S.selective_scan, x, x, A, bc[..., :3], bc)
    no(S.selective_scan, x, x, A, rnd(7, 2, 5, 3, 4), rnd(8, 2, 5, 3, 4))                # three groups, eight channels
    no(S.selective_scan, x, x, A, rnd(7, 2, 5, 2, 4), bc)
    no(S.selective_scan, x, x, -torch.ones(8, 65, device=DEV), rnd(7, 2, 5, 65), rnd(8, 2, 5, 65))
    no(S.selective_scan, x, x, z=x[..., :4], **ok)
    no(S.selective_scan, x, x, D=torch.ones(8, device=DEV, dtype=F16), **ok)
    no(S.selective_scan, x, x, initial_state=rnd(9, 2, 8, 5), **ok)
    no(S.selective_scan, x, x, initial_state=rnd(9, 2, 8, 4, dtype=BF16), **ok)
    no(S.selective_scan, x, x, max_len=-1, **ok)
    no(S.selective_scan_step, x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], rnd(9, 1, 8, 4))
    no(S.selective_scan_step, x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], rnd(9, 2, 8, 4).half())
    no(S.selective_scan_step, x[:, 0], x[:, 0], A.clone().requires_grad_(True), bc[:, 0], bc[:, 0], rnd(9, 2, 8, 4))


def test_another_stream(S):
    v = scan_inputs(400, 64, 16, 1, F32, 1)
    call = lambda: S.selective_scan(v['x'][None], v['dt'][None], v['A'], v['B'][None], v['C'][None], D=v['D'], z=v['z'][None], dt_bias=v['dt_bias'])  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_calls_replay(S):
    """two graphs of training passes and one of single frames, replayed in turn with eager work between, against eager results every time"""
    lengths = [130, 1, 60]
    off = offsets_of(lengths)
    v = scan_inputs(191, 80, 16, 1, F32, 3)
    w, gamma = rnd(9, 4, 80), 1 + rnd(10, 80, scale=0.1)
    dy = rnd(20, 191, 80)

    def train(u, w, gamma):
        y, s = S.rms_norm(u['x'], gamma, u['z'])
        c = S.causal_conv1d(y, w, seq_offsets=off)
        o, f = S.selective_scan(c, u['dt'], u['A'], u['B'], u['C'], D=u['D'], z=u['z'], dt_bias=u['dt_bias'], initial_state=u['initial'], seq_offsets=off, return_final_state=True)
        return [o, f] + list(torch.autograd.grad((o, f, s), list(u.values()) + [w, gamma], (dy, torch.ones_like(f), dy)))

    def leaves():
        return {k: t.detach().clone().requires_grad_(True) for k, t in v.items()}, w.clone().requires_grad_(True), gamma.clone().requires_grad_(True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(*leaves())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    sets, graphs, outs = [], [], []
    for _ in range(2):
        held = leaves()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = train(*held)
        sets.append(held); graphs.append(g); outs.append(out)
    pool, x1 = rnd(30, 5, 80, 16), rnd(31, 5, 80)
    start = pool.clone()
    gs = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gs):
        ys = S.selective_scan_step(x1, v['dt'][:5], v['A'], v['B'][:5], v['C'][:5], pool, D=v['D'], z=v['z'][:5], dt_bias=v['dt_bias'])
    eager_pool = start.clone()
    pool.copy_(start)
    for turn in range(4):
        for i in (0, 1):
            u = sets[i][0]
            with torch.no_grad():
                u['x'].copy_(rnd(100 + 10 * turn + i, 191, 80))
            graphs[i].replay()
            torch.cuda.synchronize()
            fresh = {k: t.detach().clone().requires_grad_(True) for k, t in u.items()}
            want = train(fresh, sets[i][1].detach().clone().requires_grad_(True), sets[i][2].detach().clone().requires_grad_(True))
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b), (turn, i)
        gs.replay()
        torch.cuda.synchronize()
        ye = S.selective_scan_step(x1, v['dt'][:5], v['A'], v['B'][:5], v['C'][:5], eager_pool, D=v['D'], z=v['z'][:5], dt_bias=v['dt_bias'])
        assert torch.equal(ys, ye) and torch.equal(pool, eager_pool), turn


def test_wrong_offsets_stay_inside_the_tensors(S):
    """offsets that fall, or reach outside: clamped on the device; what they give is not specified, that the guards around the outputs stay is"""
    v = scan_inputs(64, 40, 16, 1, F32, 3)
    from voice_converter_cyclegan_amd import _lib
    import ctypes as C
    for bad in ([0, 40, 20, 64], [-7, 10, 20, 1000], [50, 40, 30, 20], [0, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1]):
        off = torch.tensor(bad, dtype=torch.int32, device=DEV)
        guard = torch.full((64 + 32, 40), 7.0, device=DEV)
        y = guard[16:80]
        final = torch.zeros(3, 40, 16, device=DEV)
        a = _lib.ScanArgs(x=v['x'].data_ptr(), dt=v['dt'].data_ptr(), B=v['B'].data_ptr(), C=v['C'].data_ptr(), A=v['A'].data_ptr(), offsets=off.data_ptr(), y=y.data_ptr(),
                          final_state=final.data_ptr(), x_ld=40, dt_ld=40, b_ld=16, c_ld=16, y_ld=40, rows=64, cols=40, states=16, groups=1, n_seqs=3, type=0, softplus=1)
        a.work_floats = _lib.lib.vc_selective_scan_fwd_work(C.byref(a))
        work = torch.empty(max(1, a.work_floats), device=DEV)
        a.work = work.data_ptr()
        _lib.check(_lib.lib.vc_selective_scan_fwd(C.byref(a), torch.cuda.current_stream().cuda_stream))
        w = rnd(3, 4, 40)
        cy = torch.full((64 + 32, 40), 7.0, device=DEV)
        cf = torch.zeros(3, 3, 40, device=DEV)
        ca = _lib.Conv1dArgs(x=v['x'].data_ptr(), w=w.data_ptr(), offsets=off.data_ptr(), y=cy[16:80].data_ptr(), final_state=cf.data_ptr(), x_ld=40, y_ld=40, rows=64, cols=40,
                             taps=4, n_seqs=3, type=0, silu=1)
        _lib.check(_lib.lib.vc_causal_conv1d_fwd(C.byref(ca), torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        for g in (guard, cy):
            assert (g[:16] == 7).all() and (g[80:] == 7).all()


def test_rows_behind_the_last_utterance_are_left_without_zero_tail(S):
    from voice_converter_cyclegan_amd import _lib
    import ctypes as C
    v = scan_inputs(40, 24, 16, 1, F32, 2)
    off = offsets_of([10, 21])
    y = torch.full((40, 24), 7.0, device=DEV)
    a = _lib.ScanArgs(x=v['x'].data_ptr(), dt=v['dt'].data_ptr(), B=v['B'].data_ptr(), C=v['C'].data_ptr(), A=v['A'].data_ptr(), offsets=off.data_ptr(), y=y.data_ptr(),
                      x_ld=24, dt_ld=24, b_ld=16, c_ld=16, y_ld=24, rows=40, cols=24, states=16, groups=1, n_seqs=2, type=0, softplus=1)
    a.work_floats = _lib.lib.vc_selective_scan_fwd_work(C.byref(a))
    work = torch.empty(max(1, a.work_floats), device=DEV)
    a.work = work.data_ptr()
    _lib.check(_lib.lib.vc_selective_scan_fwd(C.byref(a), torch.cuda.current_stream().cuda_stream))
    assert (y[31:] == 7).all() and (y[:31] != 7).all()
    w = rnd(3, 4, 24)
    y.fill_(7)
    ca = _lib.Conv1dArgs(x=v['x'].data_ptr(), w=w.data_ptr(), offsets=off.data_ptr(), y=y.data_ptr(), x_ld=24, y_ld=24, rows=40, cols=24, taps=4, n_seqs=2, type=0, silu=1)
    _lib.check(_lib.lib.vc_causal_conv1d_fwd(C.byref(ca), torch.cuda.current_stream().cuda_stream))
    assert (y[31:] == 7).all() and (y[:31] != 7).all()


# ------------------------------------------------------------------------------------------------------- autograd's corners

def _three(S):
    """each operator on leaves of its own: (output, leaves)"""
    x, gamma, res = rnd(1, 12, 16).requires_grad_(True), (1 + rnd(2, 16, scale=0.1)).requires_grad_(True), rnd(3, 12, 16).requires_grad_(True)
    yield S.rms_norm(x, gamma, res)[0], [x, gamma, res]
    x, w = rnd(4, 3, 4, 16).requires_grad_(True), rnd(5, 4, 16).requires_grad_(True)
    yield S.causal_conv1d(x, w), [x, w]
    v = {k: t.detach().clone().requires_grad_(True) for k, t in scan_inputs(12, 16, 4, 1, F32, 1).items()}
    yield (S.selective_scan(v['x'][None], v['dt'][None], v['A'], v['B'][None], v['C'][None], D=v['D'], z=v['z'][None], dt_bias=v['dt_bias']),
           [v[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias')])


def test_gradients_kept_accumulated_and_not_differentiated_twice(S):
    for y, leaves in _three(S):
        dy = rnd(9, *y.shape)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        again = torch.autograd.grad(y, leaves, dy, create_graph=True)
        for a, b in zip(first, again):
            assert torch.equal(a, b.detach())
        with pytest.raises(RuntimeError, match='differentiated twice'):
            torch.autograd.grad(again[0].sum(), leaves, retain_graph=True)
        del again
        y.backward(dy, retain_graph=True)
        y.backward(dy)
        for t, a in zip(leaves, first):
            assert torch.equal(t.grad, a + a)
        with pytest.raises(RuntimeError):
            y.backward(dy)                                        # what was saved is gone


def test_changing_an_input_in_place_is_noticed(S):
    for y, leaves in _three(S):
        with torch.no_grad():
            leaves[1].mul_(2.0)
        with pytest.raises(RuntimeError, match='inplace'):
            y.backward(rnd(9, *y.shape))


def test_moving_a_state_on_is_noticed(S):
    state, w = rnd(1, 2, 3, 16), rnd(2, 4, 16)
    t = rnd(3, 2, 3, 16).requires_grad_(True)
    held = (t * state).sum()                                      # keeps the state for its gradient
    S.causal_conv1d_step(rnd(4, 2, 16), state, w)
    with pytest.raises(RuntimeError, match='inplace'):
        held.backward()
    v, pool = scan_inputs(2, 16, 4, 1, F32, 1), rnd(5, 2, 16, 4)
    t = rnd(6, 2, 16, 4).requires_grad_(True)
    held = (t * pool).sum()
    S.selective_scan_step(v['x'], v['dt'], v['A'], v['B'], v['C'], pool)
    with pytest.raises(RuntimeError, match='inplace'):
        held.backward()


def test_nothing_is_held_once_the_outputs_are_gone(S):
    import gc

    def use(backward):
        for y, leaves in _three(S):
            if backward:
                y.backward(rnd(9, *y.shape))
    use(True)
    for backward in (False, True):
        gc.collect(); torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        for _ in range(3):
            use(backward)
        gc.collect()
        assert torch.cuda.memory_allocated() == before


def test_what_memory_alone_does_not_tell_is_refused(S):
    gamma = torch.ones(8, device=DEV)
    negated = torch.view_as_complex(rnd(1, 6, 8, 2)).conj().imag
    assert negated.is_neg()
    with pytest.raises(ValueError, match='negated'):
        S.rms_norm(negated, gamma)
    assert torch.equal(S.rms_norm(negated.resolve_neg(), gamma), S.rms_norm(negated.clone(), gamma))
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = fw.make_dual(rnd(2, 6, 8), rnd(3, 6, 8))
        with pytest.raises(NotImplementedError, match='forward mode'):
            S.rms_norm(dual, gamma)
    with pytest.raises(ValueError):
        S.rms_norm(torch.ones((), device=DEV), gamma)
    x = rnd(4, 6, 8).requires_grad_(True)                         # a lazily negated gradient
    y = S.rms_norm(x, gamma)
    a, = torch.autograd.grad(y, x, negated, retain_graph=True)
    b, = torch.autograd.grad(y, x, negated.resolve_neg())
    assert torch.equal(a, b)


def test_rows_far_apart(S):
    """a few channels of very wide rows: copied where the kernel's 32-bit offsets would not reach"""
    wide = rnd(1, 9, (1 << 17) + 8)
    x, w, off = wide[:, 3:7], rnd(2, 4, 4), offsets_of([5, 4])
    assert torch.equal(S.causal_conv1d(x, w, seq_offsets=off), S.causal_conv1d(x.contiguous(), w, seq_offsets=off))
    leaf = wide.clone().requires_grad_(True)
    g, = torch.autograd.grad(S.causal_conv1d(leaf[:, 3:7], w, seq_offsets=off), leaf, x)
    leaf2 = x.contiguous().requires_grad_(True)
    g2, = torch.autograd.grad(S.causal_conv1d(leaf2, w, seq_offsets=off), leaf2, x.contiguous())
    assert torch.equal(g[:, 3:7], g2)


# --------------------------------------------------------------------------------------------------- more than 2^31 elements

def big(rows, cols, seed, **kw):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(rows, cols, device=DEV, dtype=BF16).normal_(generator=g, **kw)


def test_rows_beyond_32_bit_offsets(S):
    """2^21 + 70 rows of 1040 channels are more than 2^31 elements and 2^32 bytes: the last rows against the definition.  bf16, bounds as everywhere here."""
    rows, cols, tail = (1 << 21) + 70, 1040, 70
    lengths = [64] * (rows // 64 - 1) + [64 + rows % 64]
    off = offsets_of(lengths)
    x, dy = big(rows, cols, 1), big(rows, cols, 2)
    last = slice(rows - tail, rows)                               # the last utterance
    assert lengths[-1] == tail
    gamma = 1 + rnd(3, cols, scale=0.1)
    x.requires_grad_(True)
    y = S.rms_norm(x, gamma)
    dx, = torch.autograd.grad(y, x, dy)
    ref, dt, _ = O.rms_norm(x.detach()[last], gamma, 1e-6, dy[last])
    _, dt_m, _ = O.rms_norm(x.detach()[last], gamma, 1e-6, dy[last], absolute=True)
    close(y[last], ref, ref.abs(), 37, 'norm')
    close(dx[last], dt, dt_m, 111, 'norm dx')
    del y, dx
    w, b = rnd(4, 4, cols, scale=0.5), rnd(5, cols, scale=0.1)
    y = S.causal_conv1d(x, w, b, seq_offsets=off)
    dx, = torch.autograd.grad(y, x, dy)
    r = O.conv1d(x.detach()[last].cpu(), w, b, None, [tail], True, dy[last].cpu())
    m = O.conv1d(x.detach()[last].cpu(), w, b, None, [tail], True, dy[last].cpu(), absolute=True)
    close(y[last], r['y'], m['p'], 24, 'conv')
    close(dx[last], r['dx'], m['dx'], 24, 'conv dx')
    del y, dx
    v = scan_inputs(tail, cols, 4, 1, BF16, 1)
    dt = big(rows, cols, 6).clamp_(-0.1, 0.5)
    B, Cm = (big(rows, 4, s) for s in (7, 8))
    leaves = [t.requires_grad_(True) for t in (x, dt, B, Cm)]
    y = S.selective_scan(x, dt, v['A'], B, Cm, D=v['D'], dt_bias=v['dt_bias'], seq_offsets=off, max_len=70)
    got = torch.autograd.grad(y, leaves, dy)
    cut = dict(x=x.detach()[last], dt=dt.detach()[last], A=v['A'], B=B.detach()[last].view(tail, 1, 4), C=Cm.detach()[last].view(tail, 1, 4), D=v['D'], z=None,
               dt_bias=v['dt_bias'], initial=None, lengths=[tail], dy=dy[last])
    r, m = O.scan(**cut), O.scan(**cut, absolute=True)
    held = lasts(r, v['A'], tail)
    close(y[last], r['y'], m['y'], 3 * held + 44, 'scan')
    for name, g in zip(('x', 'dt', 'B', 'C'), got):
        close(g[last].reshape(r['d' + name].shape), r['d' + name], m['d' + name], 6 * held + tail + cols + 64, 'scan d' + name)


def test_slots_beyond_32_bit_offsets(S):
    """the last entry of a pool of more than 2^31 numbers moves on as the first one does"""
    n, cols, states = (1 << 17) + 5, 1024, 17
    pool = torch.zeros(n, cols, states, device=DEV)
    v = scan_inputs(1, cols, states, 1, BF16, 1)
    pool[0] = pool[n - 1] = v['initial'][0]
    assert pool.numel() > 1 << 31
    two = {k: v[k].repeat(2, *[1] * (v[k].dim() - 1)) for k in ('x', 'dt', 'z', 'B', 'C')}
    y = S.selective_scan_step(two['x'], two['dt'], v['A'], two['B'], two['C'], pool, D=v['D'], z=two['z'], dt_bias=v['dt_bias'],
                              slots=torch.tensor([0, n - 1], dtype=torch.int32, device=DEV))
    assert torch.equal(y[0], y[1]) and torch.equal(pool[0], pool[n - 1]) and not torch.equal(pool[0], v['initial'][0])
    assert (pool[1] == 0).all() and (pool[n - 2] == 0).all()
    del pool
    n, cols = (1 << 19) + 9, 1366
    state = torch.zeros(n, 3, cols, device=DEV, dtype=BF16)
    state[0] = state[n - 1] = rnd(1, 3, cols, dtype=BF16)
    assert state.numel() > 1 << 31
    x = rnd(2, 1, cols, dtype=BF16).repeat(2, 1)
    y = S.causal_conv1d_step(x, state, rnd(3, 4, cols), slots=torch.tensor([n - 1, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(y[0], y[1]) and torch.equal(state[0], state[n - 1]) and torch.equal(state[0, 2], x[0])
    assert (state[1] == 0).all() and (state[n - 2] == 0).all()


@pytest.mark.parametrize('cols,states,kind', [(16, 4, F32), (20, 16, BF16), (6, 21, F32)])
def test_scan_of_very_many_runs(S, cols, states, kind):
    """few channels and thousands of frames: hundreds of runs of a tile, what enters them worked out by a pass of its own, several runs a thread"""
    lengths = [7000, 0, 1500, 33, 700]
    n, rows = len(lengths), sum(lengths)
    v = scan_inputs(rows, cols, states, 1, kind, n)
    dy, df = rnd(20, rows, cols, dtype=kind), rnd(21, n, cols, states)
    leaves = [t.requires_grad_(True) for t in v.values()]
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of(lengths), return_final_state=True)
    r = O.scan(**v, lengths=lengths, dy=dy, dfinal=df)
    m = O.scan(**v, lengths=lengths, dy=dy, dfinal=df, absolute=True)
    last = lasts(r, v['A'], max(lengths))
    close(y, r['y'], m['y'], 3 * last + states + 40, 'y')
    close(final, r['final'], m['final'], 3 * last + states + 40, 'final')
    for (name, _), got in zip(v.items(), torch.autograd.grad((y, final), leaves, (dy, df))):
        close(got, r['d' + name], m['d' + name], 6 * last + rows + cols + states + 60, 'd' + name)


def test_a_state_that_grows_through_very_many_runs(S):
    """A > 0 over 640 runs: the factor of many runs together leaves the range of fp32, a state of zero stays one, and one that starts late stays finite"""
    rows, cols, n = 10240, 16, 4
    x = torch.zeros(1, rows, cols, device=DEV)
    x[0, rows - 300] = 1.0                                        # nothing before it
    dt = torch.full((1, rows, cols), 0.2, device=DEV)
    A = torch.full((cols, n), 0.5, device=DEV)
    one = torch.ones(1, rows, n, device=DEV)
    with torch.no_grad():
        y, final = S.selective_scan(x, dt, A, one, one, softplus=False, return_final_state=True)
    assert (y[0, :rows - 300] == 0).all() and torch.isfinite(y).all()
    steps = torch.arange(300, dtype=torch.float64)
    want = n * 0.2 * torch.exp(0.1 * steps)                       # e^30 at the end
    got = y[0, rows - 300:, 0].cpu().double()
    # a frame: two units for the exponential, one for the product, 0.3 for the exponent; over all: 0.2 and log2(e) as fp32 have them, and the exponents of
    # the runs' sums, which end at 43
    assert ((got - want).abs() <= want * U * (4 * 300 + 200)).all()
    assert torch.allclose(final, y[0, -1, 0] / n, rtol=1e-6)


@pytest.mark.parametrize('head', [5, 16, 100, 801])
@pytest.mark.parametrize('lengths', [[40, 3], [0, 700, 20], [0, 0, 9], [400]])
def test_utterances_that_begin_behind_row_zero(S, head, lengths):
    """offsets cut out of a longer list: rows ahead of the first utterance belong to none, are not read, and give zeros"""
    n, live, cols, taps = len(lengths), sum(lengths), 24, 4
    rows = head + live + 4
    v = scan_inputs(rows, cols, 16, 1, F32, n)
    dy, df = rnd(20, rows, cols), rnd(21, n, cols, 16)
    for t in [v[k] for k in ('x', 'dt', 'z', 'B', 'C')] + [dy]:
        t[:head] = float('nan')
        t[head + live:] = float('nan')
    off = offsets_of(lengths) + head
    w, init, dcf = rnd(2, taps, cols, scale=0.5), rnd(3, n, taps - 1, cols), rnd(4, n, taps - 1, cols)
    mid = slice(head, head + live)
    leaves = [v['x'].requires_grad_(True), w.requires_grad_(True), init.requires_grad_(True)]
    y, final = S.causal_conv1d(*leaves[:2], initial_state=init, seq_offsets=off, return_final_state=True)
    dx, dw, di = torch.autograd.grad((y, final), leaves, (dy, dcf))
    r = O.conv1d(v['x'][mid].detach(), w, None, init, lengths, True, dy[mid], dcf)
    m = O.conv1d(v['x'][mid].detach(), w, None, init, lengths, True, dy[mid], dcf, absolute=True)
    close(y[mid], r['y'], m['p'], taps + 20, 'conv')
    assert torch.equal(final.detach().double().cpu(), r['final'])
    close(dx[mid], r['dx'], m['dx'], taps + 20, 'conv dx')
    close(dw, r['dw'], m['dw'], taps + 20 + live, 'conv dw')
    close(di, r['dinitial'], m['dinitial'], taps + 20, 'conv dinitial')
    for t in (y, dx):
        assert (t[:head] == 0).all() and (t[head + live:] == 0).all()
    for hint in (None, max(lengths)):
        leaves = [t.detach().requires_grad_(True) for t in v.values()]
        u = dict(zip(v, leaves))
        y, final = S.selective_scan(u['x'], u['dt'], u['A'], u['B'], u['C'], D=u['D'], z=u['z'], dt_bias=u['dt_bias'], initial_state=u['initial'], seq_offsets=off,
                                    max_len=hint, return_final_state=True)
        grads = dict(zip(v, torch.autograd.grad((y, final), leaves, (dy, df))))
        cut = {k: t.detach()[mid] if k in ('x', 'dt', 'z', 'B', 'C') else t.detach() for k, t in v.items()}
        r, m = O.scan(**cut, lengths=lengths, dy=dy[mid], dfinal=df), O.scan(**cut, lengths=lengths, dy=dy[mid], dfinal=df, absolute=True)
        last = lasts(r, v['A'], max(lengths))
        close(y[mid], r['y'], m['y'], 3 * last + 56, 'y')
        close(final, r['final'], m['final'], 3 * last + 56, 'final')
        for k, got in grads.items():
            rowwise = k in ('x', 'dt', 'z', 'B', 'C')
            close(got[mid] if rowwise else got, r['d' + k], m['d' + k], 6 * last + rows + cols + 76, 'd' + k)
            if rowwise:
                assert (got[:head] == 0).all() and (got[head + live:] == 0).all(), k
        assert (y[:head] == 0).all() and (y[head + live:] == 0).all()


@pytest.mark.parametrize('kind,stream', [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_large_norms_equal_their_parts(S, kind, stream):
    """inputs of more than 32 MiB are loaded past the L2s as well"""
    rows, cols = 17000, 1024
    x, res, gamma = rnd(1, rows, cols, dtype=kind), rnd(2, rows, cols, dtype=stream), 1 + rnd(3, cols, scale=0.1)
    dy, ds = rnd(4, rows, cols, dtype=kind), rnd(5, rows, cols, dtype=stream)
    parts = [slice(i, min(i + 2000, rows)) for i in range(0, rows, 2000)]

    def norm(p):
        a, b = x[p].detach().requires_grad_(True), res[p].detach().requires_grad_(True)
        y, s = S.rms_norm(a, gamma, b)
        return [y, s] + list(torch.autograd.grad((y, s), (a, b), (dy[p], ds[p]))) + list(S.rms_norm_e4m3(x[p], gamma, res[p], group=128))
    for i, (a, *b) in enumerate(zip(norm(slice(0, rows)), *[norm(p) for p in parts])):
        assert torch.equal(a.float(), torch.cat(b).float()), i


@pytest.mark.parametrize('kind,stream', [(BF16, F32), (F32, F32), (F16, F16)])
def test_large_calls_equal_their_parts(S, kind, stream):
    """outputs of more than 8 MiB are stored past the L2s: the same bits as in parts that are not, odd channel counts and tails included"""
    rows, cols = 4300, 1001
    x, res, gamma = rnd(1, rows, cols, dtype=kind), rnd(2, rows, cols, dtype=stream), 1 + rnd(3, cols, scale=0.1)
    dy, ds = rnd(4, rows, cols, dtype=kind), rnd(5, rows, cols, dtype=stream)
    parts = [slice(0, 1000), slice(1000, 2000), slice(2000, 3000), slice(3000, rows)]
    assert rows * cols * x.element_size() >= 8 << 20 > 1300 * cols * x.element_size()

    def norm(p):
        a, b = x[p].detach().requires_grad_(True), res[p].detach().requires_grad_(True)
        y, s = S.rms_norm(a, gamma, b)
        return [y, s] + list(torch.autograd.grad((y, s), (a, b), (dy[p], ds[p]))) + list(S.rms_norm_e4m3(x[p], gamma, res[p]))
    for i, (a, *b) in enumerate(zip(norm(slice(0, rows)), *[norm(p) for p in parts])):
        assert torch.equal(a.float(), torch.cat(b).float()), i
    w, lengths = rnd(6, 4, cols, scale=0.5), [1000, 1000, 1000, 1300]

    def conv(p, lens):
        a = x[p].detach().requires_grad_(True)
        y = S.causal_conv1d(a, w, seq_offsets=offsets_of(lens))
        return [y] + list(torch.autograd.grad(y, a, dy[p]))
    for i, (a, *b) in enumerate(zip(conv(slice(0, rows), lengths), *[conv(p, [n]) for p, n in zip(parts, lengths)])):
        assert torch.equal(a, torch.cat(b)), i
    for states in (16, 13):
        v = scan_inputs(900, 200, states, 1, kind, 1)
        pool = rnd(7, 900, 200, states)
        halves = pool.clone()
        assert pool.numel() * 4 >= 8 << 20 > pool.numel() * 2

        def step(p, state):
            return S.selective_scan_step(v['x'][p], v['dt'][p], v['A'], v['B'][p], v['C'][p], state, D=v['D'], z=v['z'][p], dt_bias=v['dt_bias'])
        y = step(slice(0, 900), pool)
        assert torch.equal(y, torch.cat([step(slice(0, 450), halves[:450]), step(slice(450, 900), halves[450:])])) and torch.equal(pool, halves)


# ------------------------------------------------------------------------------------------- 8 bits: which side of a border

def e4m3_of(v):
    """64-bit v to the nearest e4m3 value, ties to even, as the numbers they stand for; and how far v lies from the next border, relative to v"""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    n = v / step
    return (torch.round(n) * step).clamp(-448, 448), ((n.abs() - torch.floor(n.abs()) - 0.5).abs() / n.abs().clamp_min(2.0 ** -60))


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('cols,group', [(1024, 0), (1024, 32), (1024, 128), (2048, 64), (8192, 0), (33280, 0), (33280, 128)])
def test_norm_e4m3_beside_a_border(S, kind, cols, group):
    """Quotients 448 t gamma / max|t gamma| that lie within 2^-24 of a border between two e4m3 values, in registers and in long rows: every one has to go to
    the side of it that the quotient in 64 bits lies on.  The kernel holds the quotient as a sum of two fp32 numbers: what it leaves out are products of two
    rounding errors, at most 8 of 2^-48 = 2^-45 of the value, so only what lies within 2^-40 of its border (64-bit arithmetic rounds too, by 2^-52) may differ."""
    g = torch.Generator().manual_seed(cols + group)
    wide = group or cols
    x = (1 + torch.rand(1, cols, generator=g)).to(kind)
    x64 = x.double()[0]
    top = x64.view(-1, wide)[:, :1].repeat_interleave(wide, 1).view(-1)                      # max|t gamma| of a group: its first column's, where gamma is 1
    e, m = torch.randint(-8, 6, (cols,), generator=g).double(), torch.randint(0, 8, (cols,), generator=g).double()
    border = torch.where(e == -8, (m + 0.5) * 2.0 ** -9, (8.5 + m) * torch.exp2(e) / 2)      # from half the least value to 248
    gamma = (border / 448 * top / x64).float()
    gamma.view(-1, wide)[:, 0] = 1.0
    sign = torch.where(torch.rand(cols, generator=g) < 0.5, -1.0, 1.0)
    q, scale = S.rms_norm_e4m3(x.to(DEV), (gamma * sign).to(DEV), group=group)
    p = x64 * (gamma * sign).double()
    v = p * 448 / p.view(-1, wide).abs().amax(-1, keepdim=True).repeat_interleave(wide, 1).view(-1)
    want, far = e4m3_of(v)
    assert (far < 2.0 ** -23).sum() > 0.9 * cols * (wide - 1) / wide
    clear = far > 2.0 ** -40
    assert clear.sum() > 0.9 * cols
    wrong = (q[0].float().cpu().double() != want) & clear
    assert not wrong.any(), '%d of %d on the wrong side' % (int(wrong.sum()), cols)


@pytest.mark.parametrize('kind,stream,group', [(BF16, F32, 128), (F32, F32, 0), (F16, F16, 32)])
def test_norm_e4m3_of_many_rows_is_the_nearest_value(S, kind, stream, group):
    """17 million ordinary values: nearest in 64 bits, apart from those within 2^-40 of a border; a quotient in fp32 gets several wrong"""
    rows, cols = 16384, 1024
    x, res, gamma = rnd(1, rows, cols, dtype=kind), rnd(2, rows, cols, dtype=stream, scale=3.0), 1 + rnd(3, cols, scale=0.1)
    q, scale, total = S.rms_norm_e4m3(x, gamma, res, group=group)
    p = total.double() * gamma.double()
    v = (p.view(rows, -1, group or cols) * 448 / p.view(rows, -1, group or cols).abs().amax(-1, keepdim=True)).view(rows, cols)
    want, far = e4m3_of(v)
    clear = far > 2.0 ** -40
    assert clear.float().mean() > 0.999
    assert int(((q.float().double() != want) & clear).sum()) == 0


@pytest.mark.parametrize('cols', [256, 33280])
def test_norm_e4m3_of_tiny_rows(S, cols):
    """Groups under the least scale (max|y| below 2^-100) that are not zero, and products t gamma so small that 448 over the largest leaves fp32 while the norm
    itself is above the least scale (a tiny eps): the values and scales of the definition.  rstd is off by cols / 64 + 8 roundings (a sum of squares of a
    thread's columns, steps across lanes and waves, a root and a quotient), and two products follow."""
    u = rnd(1, 2, cols)
    k = cols / 64 + 12
    for size, eps in ((1e-30, 1e-6), (3e-34, 1e-6), (3e-37, 1e-14), (1e-39, 1e-18)):
        x, gamma = u * size, torch.ones(cols, device=DEV)
        q, scale = S.rms_norm_e4m3(x, gamma, eps=eps, group=128)
        y = O.rms_norm(x, gamma, eps).view(2, -1, 128)
        want = y.abs().amax(-1).clamp_min(2.0 ** -100) / 448
        close(scale, want, want, k, 'scale %g %g' % (size, eps))
        v = q.float().double().cpu().view(2, -1, 128)
        assert torch.isfinite(v).all(), (size, eps)
        ideal = y / want[..., None]
        assert ((v - ideal).abs() <= ideal.abs() * (2.0 ** -4 + k * U) + 2.0 ** -10 + k * U).all(), (size, eps, float((v - ideal).abs().max()))


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [20, 1500])
def test_scan_from_an_infinite_state(S, kind, rows):
    """an infinite state wears off by no factor above zero: infinite with its sign to the end, frame by frame and over runs whose whole factor leaves fp32; the
    gradient that an infinite one of the final state leaves behind is infinite back to the first frame"""
    cols, states = 12, 8
    v = scan_inputs(rows, cols, states, 1, kind, 1)
    v['C'], v['z'] = v['C'].abs() + 0.5, v['z'].abs() + 0.5
    sign = torch.tensor([1.0, -1.0, 1.0], device=DEV).repeat(4)
    sick = torch.tensor([True, True, False], device=DEV).repeat(4)
    v['initial'][:, sick] = float('inf') * sign[sick, None]
    call = lambda u: S.selective_scan(u['x'], u['dt'], u['A'], u['B'], u['C'], D=u['D'], z=u['z'], dt_bias=u['dt_bias'], initial_state=u['initial'],  # noqa: E731
                                      seq_offsets=offsets_of([rows]), return_final_state=True)
    y, final = call(v)
    assert (y[:, sick] == float('inf') * sign[sick]).all() and (final[:, sick] == float('inf') * sign[sick, None]).all()
    assert torch.isfinite(y[:, ~sick]).all() and torch.isfinite(final[:, ~sick]).all()
    v['initial'] = torch.zeros_like(v['initial']).requires_grad_(True)
    df = torch.zeros(1, cols, states, device=DEV)
    df[:, sick] = float('inf') * sign[sick, None]
    d, = torch.autograd.grad(call(v)[1], v['initial'], df)
    assert torch.equal(d, df)


# ------------------------------------------------------------------------------------------------- steps of zero and beyond

def masked_scan(kind, lengths, cols, states, fill, seed=1):
    """scan_inputs with frames whose dt is `fill`: the first two of every utterance, a stretch in it, the last one, and all of the second utterance"""
    rows = sum(lengths)
    v = scan_inputs(rows, cols, states, 1, kind, len(lengths), seed)
    mask = torch.zeros(rows, dtype=torch.bool)
    at = 0
    for i, m in enumerate(lengths):
        mask[at:at + 2] = True
        mask[at + m // 3:at + m // 2] = True
        mask[at + m - 1:at + m] = True
        if i == 1:
            mask[at:at + m] = True
        at += m
    v['dt'][mask.to(DEV)] = fill
    return v, mask


def least_of(kind):
    return [float('-inf'), torch.finfo(kind).min]


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('which', [0, 1])
@pytest.mark.parametrize('lengths,hint', [([23, 18, 40], 40), ([700, 20, 900], None), ([2000], None)])
def test_scan_of_masked_frames(S, kind, which, lengths, hint):
    """dt = -inf or the type's lowest value is a step of zero (softplus is 0 in 64 bits, and in fp32): the state stays as it is, y = C h + D x, dt has no
    gradient there, and nothing else of the utterance notices; walked and in runs"""
    cols, states = 24, 16
    v, mask = masked_scan(kind, lengths, cols, states, least_of(kind)[which])
    rows = sum(lengths)
    dy, df = rnd(20, rows, cols, dtype=kind), rnd(21, len(lengths), cols, states)
    leaves = [t.requires_grad_(True) for t in v.values()]
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of(lengths), max_len=hint, return_final_state=True)
    r = O.scan(**v, lengths=lengths, dy=dy, dfinal=df)
    m = O.scan(**v, lengths=lengths, dy=dy, dfinal=df, absolute=True)
    assert all(torch.isfinite(t).all() for t in r.values())
    steps = r['delta'][~mask]                                     # masked frames carry a term by a factor of exactly 1: they do not wear it
    last = min(max(lengths), 17 / float(steps.min() * v['A'].detach().abs().min()))
    close(y, r['y'], m['y'], 3 * last + states + 40, 'y')
    close(final, r['final'], m['final'], 3 * last + states + 40, 'final')
    if len(lengths) > 1:
        assert torch.equal(final[1], v['initial'][1])
    grads = dict(zip(v, torch.autograd.grad((y, final), leaves, (dy, df))))
    assert (grads['dt'][mask.to(DEV)] == 0).all()
    for name, got in grads.items():
        over = rows if name in ('A', 'D', 'dt_bias') else cols if name in ('B', 'C') else 0
        close(got, r['d' + name], m['d' + name], 6 * last + over + states + 60, 'd' + name)


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('which', [0, 1])
def test_single_frames_of_masked_streams(S, kind, which):
    """a masked frame of a live stream leaves its state as it is"""
    v = scan_inputs(6, 40, 16, 1, kind, 6)
    v['dt'][1::2] = least_of(kind)[which]
    pool = v['initial'].clone()
    y = S.selective_scan_step(v['x'], v['dt'], v['A'], v['B'][:, 0], v['C'][:, 0], pool, D=v['D'], z=v['z'], dt_bias=v['dt_bias'])
    r, m = O.scan(**v, lengths=[1] * 6), O.scan(**v, lengths=[1] * 6, absolute=True)
    close(y, r['y'], m['y'], 59, 'y')
    close(pool, r['final'], m['final'], 59, 'state')
    assert torch.equal(pool[1::2], v['initial'][1::2])


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [40, 1500])
def test_scan_of_the_largest_steps(S, kind, rows):
    """dt = the type's largest value: softplus is dt itself, the state forgets everything and takes delta x B.  x is small there (2^-30, in fp16 2^-8) and dy
    (2^-20), so that neither h nor a gradient leaves its type; what is 1e29 large wears off over the frames behind, and so do the bounds"""
    cols, states, big = 24, 4, torch.finfo(kind).max
    v = scan_inputs(rows, cols, states, 1, kind, 1)
    at = [5, rows // 2]
    v['dt'][at] = big
    v['x'][at] *= 2.0 ** (-8 if kind == F16 else -30)
    v['C'] *= 2.0 ** -8                                           # y within fp16
    v['z'] = v['z'].clamp(-2, 2)
    dy = (rnd(20, rows, cols) * 2.0 ** -20).to(kind) if kind != F16 else rnd(20, rows, cols, dtype=kind) * 2.0 ** -10
    leaves = [t.requires_grad_(True) for t in v.values()]
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of([rows]), return_final_state=True)
    r, m = O.scan(**v, lengths=[rows], dy=dy), O.scan(**v, lengths=[rows], dy=dy, absolute=True)
    assert all(torch.isfinite(t.to(kind)).all() for k, t in r.items() if k in ('y', 'dx', 'ddt', 'dz', 'dB', 'dC')), 'inputs out of range'
    last = lasts(r, v['A'], rows)
    close(y, r['y'], m['y'], 3 * last + states + 40, 'y')
    close(final, r['final'], m['final'], 3 * last + states + 40, 'final')
    for name, got in zip(v, torch.autograd.grad(y, leaves, dy)):
        over = rows if name in ('A', 'D', 'dt_bias') else cols if name in ('B', 'C') else 0
        close(got, r['d' + name], m['d' + name], 6 * last + over + states + 60, 'd' + name)
    pool = v['initial'].detach().repeat(2, 1, 1)
    w = {k: t.detach()[at] if k in ('x', 'dt', 'z', 'B', 'C') else t.detach() for k, t in v.items()}
    y = S.selective_scan_step(w['x'], w['dt'], w['A'], w['B'][:, 0], w['C'][:, 0], pool, D=w['D'], z=w['z'], dt_bias=w['dt_bias'])
    w['initial'] = v['initial'].detach().repeat(2, 1, 1)
    r, m = O.scan(**w, lengths=[1, 1]), O.scan(**w, lengths=[1, 1], absolute=True)
    close(y, r['y'], m['y'], 59, 'step')
    close(pool, r['final'], m['final'], 59, 'state')


@pytest.mark.parametrize('kind', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [9, 1500])
def test_scan_of_infinite_and_undefined_steps(S, kind, rows):
    """dt = inf: softplus is infinite, and so are a channel's states from there on, with the sign of x B; dt = NaN is NaN from there on.  One sign a channel"""
    cols, states = 12, 8
    v = scan_inputs(rows, cols, states, 1, kind, 1)
    v['x'] = (v['x'].abs() + 0.5) * torch.tensor([1.0, -1.0, -1.0], device=DEV, dtype=kind).repeat(4)
    v['B'], v['C'], v['z'] = v['B'].abs() + 0.5, v['C'].abs() + 0.5, v['z'].abs() + 0.5
    v['dt'][4, 1::2] = float('inf')
    v['dt'][4, 2::4] = float('nan')
    r = O.scan(**v, lengths=[rows])
    assert torch.isinf(r['y'][4:, 1::2]).all() and torch.isnan(r['y'][4:, 2::4]).all() and torch.isfinite(r['y'][:, ::4]).all()
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of([rows]), return_final_state=True)
    pool = v['initial'].clone()
    one = torch.stack([S.selective_scan_step(v['x'][i:i + 1], v['dt'][i:i + 1], v['A'], v['B'][i:i + 1, 0], v['C'][i:i + 1, 0], pool, D=v['D'], z=v['z'][i:i + 1],
                                             dt_bias=v['dt_bias'])[0] for i in range(rows)])
    for got, ref in ((y, r['y']), (one, r['y']), (final, r['final']), (pool, r['final'])):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.where(torch.isinf(got), got.sign(), torch.zeros_like(got)), torch.where(torch.isinf(ref), ref.sign(), torch.zeros_like(ref)))


def test_one_row_of_any_stride(S):
    """a call of a single row takes no stride from its arguments: 0 (or any other) means the same as its width, in outputs too"""
    from voice_converter_cyclegan_amd import _lib
    import ctypes as C
    cols, states = 24, 16
    v = scan_inputs(1, cols, states, 1, F32, 1)
    dy = rnd(20, 1, cols)
    leaves = [v[k].requires_grad_(True) for k in ('x', 'dt', 'A', 'B', 'C', 'z')]
    y0 = S.selective_scan(v['x'][None], v['dt'][None], v['A'], v['B'][None], v['C'][None], z=v['z'][None])
    want = torch.autograd.grad(y0, leaves, dy[None])
    for ld in (0, 5, cols, 1 << 28):
        out = {k: torch.full((cols, states) if k == 'dA' else (1, states) if k in ('dB', 'dC') else (1, cols), 7.0, device=DEV) for k in ('y', 'dx', 'ddt', 'dz', 'dA', 'dB', 'dC')}
        a = _lib.ScanArgs(x=v['x'].data_ptr(), dt=v['dt'].data_ptr(), z=v['z'].data_ptr(), B=v['B'].data_ptr(), C=v['C'].data_ptr(), A=v['A'].data_ptr(), dy=dy.data_ptr(),
                          x_ld=cols, dt_ld=cols, z_ld=cols, b_ld=states, c_ld=states, dy_ld=cols, y_ld=ld, dx_ld=ld, ddt_ld=ld, dz_ld=ld, db_ld=ld, dc_ld=ld,
                          rows=1, cols=cols, states=states, groups=1, n_seqs=1, type=0, softplus=1, **{k: t.data_ptr() for k, t in out.items()})
        a.saved_floats = _lib.lib.vc_selective_scan_saved(C.byref(a))
        assert a.saved_floats > 0, _lib.lib.vc_last_error()
        a.work_floats = max(_lib.lib.vc_selective_scan_fwd_work(C.byref(a)), _lib.lib.vc_selective_scan_bwd_work(C.byref(a)))
        saved, work = torch.empty(a.saved_floats, device=DEV), torch.empty(a.work_floats, device=DEV)
        a.saved, a.work = saved.data_ptr(), work.data_ptr()
        stream = torch.cuda.current_stream().cuda_stream
        _lib.check(_lib.lib.vc_selective_scan_fwd(C.byref(a), stream))
        _lib.check(_lib.lib.vc_selective_scan_bwd(C.byref(a), stream))
        torch.cuda.synchronize()
        assert torch.equal(out['y'], y0[0].detach()), ld
        for k, w in zip(('dx', 'ddt', 'dA', 'dB', 'dC', 'dz'), want):
            assert torch.equal(out[k].view(w.shape), w), (k, ld)


# -------------------------------------------------------------------------------------------------- far out on the sigmoid

def test_gates_and_activations_of_large_magnitude(S):
    """p sigmoid(p) and its slope relative to themselves, in fp32 and far to both sides (rounding the exponential's argument alone would cost |p| 2^-24).
    Roundings of 2^-24: the exponential 2 (one unit in the last place) and its correction 1, 1 + e 1, the reciprocal 2, e times it 1, p times it 1 = 8; slope
    s (1 + p (1 - s)), relative to s (1 + |p|): s 7, 1 - s 2, the multiply-add and the product 1 each = 11; the scan multiplies once more."""
    n = 512
    p = torch.cat([-torch.linspace(2.0, 80.0, n), torch.linspace(2.0, 80.0, n)]) + 0.3 * torch.rand(2 * n, generator=torch.Generator().manual_seed(1))
    p = p.to(DEV)
    s64 = 1 / (1 + torch.exp(-p.cpu().double()))
    y64, d64 = O.silu(p.cpu().double()), O.dsilu(p.cpu().double())
    dmag = s64 * (1 + p.cpu().double().abs())
    w = torch.tensor([0.0, 1.0], device=DEV)[:, None].repeat(1, 2 * n)
    x = p[None, None].clone().requires_grad_(True)
    y = S.causal_conv1d(x, w)
    close(y[0, 0], y64, y64.abs(), 8, 'convolution')
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    close(dx[0, 0], d64, dmag, 11, 'convolution, slope')
    close(S.causal_conv1d_step(p[None], torch.zeros(1, 1, 2 * n, device=DEV), w)[0], y64, y64.abs(), 8, 'convolution, single frame')
    one, bc = torch.ones(1, 1, 2 * n, device=DEV), torch.zeros(1, 1, 4, device=DEV)
    A, D = -torch.ones(2 * n, 4, device=DEV), torch.ones(2 * n, device=DEV)
    z = p[None, None].clone().requires_grad_(True)
    y = S.selective_scan(one, one, A, bc, bc, D=D, z=z)
    close(y[0, 0], y64, y64.abs(), 9, 'gate')
    dz, = torch.autograd.grad(y, z, torch.ones_like(y))
    close(dz[0, 0], d64, dmag, 13, 'gate, slope')
    pool = torch.zeros(1, 2 * n, 4, device=DEV)
    close(S.selective_scan_step(one[0], one[0], A, bc[0], bc[0], pool, D=D, z=p[None])[0], y64, y64.abs(), 9, 'gate, single frame')


@pytest.mark.parametrize('kind', [F32, BF16, F16])
def test_gates_and_activations_at_the_ends_of_a_type(S, kind):
    """the lowest value gates to zero with a slope of zero, the largest to itself with a slope of one"""
    ends = torch.tensor([torch.finfo(kind).min, torch.finfo(kind).max, -200.0, 200.0], device=DEV, dtype=kind)
    y0, d0 = ends.clamp_min(0), torch.tensor([0.0, 1.0, 0.0, 1.0], device=DEV, dtype=kind)
    w = torch.tensor([0.0, 1.0], device=DEV)[:, None].repeat(1, 4)
    x = ends[None, None].clone().requires_grad_(True)
    y = S.causal_conv1d(x, w)
    assert torch.equal(y[0, 0], y0) and torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0][0, 0], d0)
    assert torch.equal(S.causal_conv1d_step(ends[None], torch.zeros(1, 1, 4, device=DEV, dtype=kind), w)[0], y0)
    one, bc = torch.ones(1, 1, 4, device=DEV, dtype=kind), torch.zeros(1, 1, 4, device=DEV, dtype=kind)
    A, D = -torch.ones(4, 4, device=DEV), torch.ones(4, device=DEV)
    z = ends[None, None].clone().requires_grad_(True)
    y = S.selective_scan(one, one, A, bc, bc, D=D, z=z)
    assert torch.equal(y[0, 0], y0) and torch.equal(torch.autograd.grad(y, z, torch.ones_like(y))[0][0, 0], d0)
    assert torch.equal(S.selective_scan_step(one[0], one[0], A, bc[0], bc[0], torch.zeros(1, 4, 4, device=DEV), D=D, z=ends[None])[0], y0)


@pytest.mark.parametrize('kind,stream,rows,cols', [(BF16, BF16, 24000, 1024), (F16, F16, 6000, 4096), (F32, F32, 12000, 1024), (BF16, None, 50000, 1024), (F32, None, 24000, 1024)])
def test_norms_that_read_past_the_l2s_equal_their_parts(S, kind, stream, rows, cols):
    """from 88 MiB of inputs on every pass loads past the L2s: the same bits as in parts that do not; with and without a residual, and a gradient of the sum"""
    x, gamma, dy = rnd(1, rows, cols, dtype=kind), 1 + rnd(3, cols, scale=0.1), rnd(4, rows, cols, dtype=kind)
    res, ds = (None, None) if stream is None else (rnd(2, rows, cols, dtype=stream), rnd(5, rows, cols, dtype=stream))
    assert x.numel() * x.element_size() * (1 if res is None else 2) >= 88 << 20
    step = rows // 8

    def norm(p):
        a = x[p].detach().requires_grad_(True)
        if res is None:
            y = S.rms_norm(a, gamma)
            return [y] + list(torch.autograd.grad(y, a, dy[p])) + list(S.rms_norm_e4m3(x[p], gamma, group=64))
        b = res[p].detach().requires_grad_(True)
        y, s = S.rms_norm(a, gamma, b)
        return [y, s] + list(torch.autograd.grad((y, s), (a, b), (dy[p], ds[p]), retain_graph=True)) + list(torch.autograd.grad(y, a, dy[p])) \
            + list(S.rms_norm_e4m3(x[p], gamma, res[p], group=64))
    whole, parts = norm(slice(0, rows)), [norm(slice(i, min(i + step, rows))) for i in range(0, rows, step)]
    for i, (a, *b) in enumerate(zip(whole, *parts)):
        assert torch.equal(a.float(), torch.cat(b).float()), i


# ------------------------------------------------------------------------------------------ gradients by what they add over

@pytest.mark.parametrize('lengths,hint', [([4000], None), ([900, 7, 0, 1500], None), ([70] * 40, 70)])
@pytest.mark.parametrize('cols,states,groups,kind', [(48, 16, 1, F32), (26, 12, 2, F32), (40, 16, 1, BF16)])
def test_scan_gradients_add_over_what_their_bounds_count(S, lengths, hint, cols, states, groups, kind):
    """dx, ddt, dz and dinitial add over states only, dB and dC over a group's channels as well, dA, dD and ddt_bias over the rows: bounds that count no more.
    States forget fast here (delta |A| >= 0.5: 2^-24 is left after 34 frames), so the recurrence's own share is small."""
    rows, n = sum(lengths), len(lengths)
    v = scan_inputs(rows, cols, states, groups, kind, n)
    v['A'] = v['A'] - 10.0
    dy, df = rnd(20, rows, cols, dtype=kind), rnd(21, n, cols, states)
    leaves = [t.requires_grad_(True) for t in v.values()]
    y, final = S.selective_scan(v['x'], v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], initial_state=v['initial'],
                                seq_offsets=offsets_of(lengths), max_len=hint, return_final_state=True)
    r = O.scan(**v, lengths=lengths, dy=dy, dfinal=df)
    m = O.scan(**v, lengths=lengths, dy=dy, dfinal=df, absolute=True)
    last = lasts(r, v['A'], max(lengths))
    assert last < 50
    close(y, r['y'], m['y'], 3 * last + states + 40, 'y')
    close(final, r['final'], m['final'], 3 * last + states + 40, 'final')
    for (name, _), got in zip(v.items(), torch.autograd.grad((y, final), leaves, (dy, df))):
        over = rows if name in ('A', 'D', 'dt_bias') else cols // groups if name in ('B', 'C') else 0
        close(got, r['d' + name], m['d' + name], 6 * last + over + states + 60, 'd' + name)
