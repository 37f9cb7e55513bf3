"""Sequence operators on torch GPU tensors: what a causal model of frames is built of, beside the utterance-wide blocks of module.py.

The reference's generator looks ahead (SAME convolutions, module.py:32-40) and normalises over a whole utterance (module.py:135-146).  These
operators look back only: a model of them trains on packed utterances and converts a live stream frame by frame, with the same results.

    y, stream = rms_norm(x, gamma, stream)            # stream + x, and its norm
    u = causal_conv1d(y @ W, w, bias)                 # a few earlier frames, channel by channel
    v = selective_scan(u, dt, A, B, C, D=D, z=z)      # all earlier frames, through a state of `states` numbers a channel

Frames are rows: tensors are [batch, frames, channels], or [rows, channels] with `seq_offsets` (int32, [n + 1], rising, on the same device) where
utterances of different lengths lie one behind the other; lengths of zero are fine, and rows behind the last utterance give zeros.  Any row
stride is taken in place (column slices of a product, for one).  Activations are fp32, bf16 or fp16 (one type in a call); parameters, recurrent
states and parameter gradients are fp32, and every sum is.  The kernels are those of include/vc_cyclegan.h; gradients are deterministic.

A backward pass that is captured into a graph must not meet an eager autograd graph of the same leaves that is still alive: torch's gradient
accumulators belong to the stream they were made on.  Drop the eager outputs first."""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import lib, check

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = torch._C._cuda_getCurrentRawStream


def _refuse(text, *args):
    raise ValueError(text % args)


def _p(t):
    return None if t is None else t.data_ptr()


def _launch(f, name, ref, *args):
    """f(*args, stream) on ref's device and that device's current stream."""
    index = ref.get_device()
    if torch.cuda.current_device() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        check(rc, name)


def _activation(t, name):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        _refuse('%s must be a tensor on a GPU (there is no CPU path)', name)
    if t.dtype not in _TYPES:
        _refuse('%s must be float32, bfloat16 or float16, got %s', name, t.dtype)
    return t


def _like(t, ref, name, shape=None, dtype=None):
    """t on ref's device, with this shape and type."""
    dtype = dtype or ref.dtype
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == ref.get_device() and (shape is None or t.shape == shape):
        return t
    if not (isinstance(t, torch.Tensor) and t.device == ref.device and t.dtype is dtype):
        _refuse('%s must be a %s tensor on %s', name, dtype, ref.device)
    raise ValueError('%s must have shape %s, got %s' % (name, tuple(shape), tuple(t.shape)))


def _parameter(t, ref, name, shape):
    return None if t is None else _like(t, ref, name, shape, torch.float32).contiguous()


def _rows(t, tail=1):
    """[..., channels] (or [..., groups, states] with tail = 2) as rows with one stride between them: (tensor, stride).  Copies only what cannot be seen so."""
    if t.is_contiguous():
        return t, t.shape[-1] if tail == 1 else t.shape[-1] * t.shape[-2]
    if tail == 1 and t.dim() == 2 and t.stride(1) == 1:
        return t, t.stride(0)
    inner = t.shape[t.dim() - tail:]
    width = 1
    for n in inner:
        width *= n
    flat = t if t.dim() == tail + 1 else t.reshape(-1, *inner)
    if flat.stride(-1) != 1 and inner[-1] > 1 or tail == 2 and inner[0] > 1 and flat.stride(1) != inner[1] or flat.stride(0) < 0:
        flat = flat.contiguous()
    return flat, flat.stride(0) if flat.shape[0] > 1 else width


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_grad(what, *tensors):
    if _wants_grad(*tensors):
        _refuse('%s has no gradient: call it under torch.no_grad() or on detached tensors', what)


def _fresh(shape, ref, dtype=None):
    return ref.new_empty(shape, dtype=dtype)


def _fresh_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _once(grad):
    """The backward of a Function that cannot be differentiated again: refuses that where a graph of the backward is built, costs nothing where none is."""
    guarded = once_differentiable(grad)

    def backward(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else grad)(ctx, *grads)
    return backward


# ------------------------------------------------------------------------------------------------------------------ norm

def _norm_inputs(x, gamma, residual, eps):
    _activation(x, 'x')
    if not (x.dim() >= 1 and x.shape[-1] > 0):
        _refuse('x must be [..., channels]')
    if not eps > 0:
        _refuse('eps must be positive')
    gamma = _parameter(gamma, x, 'gamma', (x.shape[-1],))
    if gamma is None:
        _refuse('gamma is missing')
    if residual is not None:
        if not (isinstance(residual, torch.Tensor) and residual.dtype in (x.dtype, torch.float32)):
            _refuse('residual must be a tensor of %s or float32', x.dtype)
        _like(residual, x, 'residual', x.shape, residual.dtype)
    return gamma


def _norm_forward(x, gamma, residual, eps, keep):
    cols = x.shape[-1]
    rows = x.numel() // cols
    x2, x_ld = _rows(x)
    y = _fresh_like(x)
    kind = stream_kind = _TYPES[x.dtype]
    total, r2, r_ld = None, None, 0
    if residual is not None:
        total = _fresh_like(residual)
        r2, r_ld = _rows(residual)
        stream_kind = _TYPES[residual.dtype]
    rstd = _fresh((rows,), gamma) if keep else None
    _launch(lib.vc_rms_norm_fwd, 'vc_rms_norm_fwd', x, _p(x2), x_ld, _p(r2), r_ld, _p(gamma), _p(y), cols, _p(total), cols, _p(rstd), eps, rows, cols,
            kind, stream_kind)
    return y, total, rstd, (kind, stream_kind)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, residual, eps):
        y, total, rstd, ctx.kinds = _norm_forward(x, gamma, residual, eps, True)
        ctx.x_dtype = x.dtype
        ctx.has_residual = residual is not None
        ctx.save_for_backward(x if total is None else total, gamma, rstd)
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @_once
    def backward(ctx, dy, dtotal=None):
        total, gamma, rstd = ctx.saved_tensors
        cols = total.shape[-1]
        if dy is None:
            dy = torch.zeros(total.shape, dtype=ctx.x_dtype, device=total.device)
        t2, t_ld = _rows(total)
        dy2, dy_ld = _rows(dy)
        ds2, ds_ld = _rows(dtotal) if dtotal is not None else (None, 0)
        rows = total.numel() // cols
        need_x, need_g, need_r = ctx.needs_input_grad[:3]
        need_r = need_r and ctx.has_residual
        one = ctx.kinds[0] == ctx.kinds[1]                       # one gradient serves both summands where they have one type
        dx = _fresh(total.shape, total, ctx.x_dtype) if need_x or (one and need_r) else None
        dres = _fresh(total.shape, total) if need_r and not one else None
        dgamma = torch.zeros_like(gamma) if need_g and rows == 0 else _fresh(gamma.shape, gamma) if need_g else None
        floats = lib.vc_rms_norm_bwd_work(rows, cols) if need_g else 0
        work = _fresh((floats,), gamma) if floats else None
        if rows:
            _launch(lib.vc_rms_norm_bwd, 'vc_rms_norm_bwd', total, _p(dy2), dy_ld, _p(ds2), ds_ld, _p(t2), t_ld, _p(rstd), _p(gamma), _p(dx), cols,
                    _p(dres), cols, _p(dgamma), _p(work), floats, rows, cols, *ctx.kinds)
        return dx if need_x else None, dgamma, (dx if one else dres) if need_r else None, None


def rms_norm(x, gamma, residual=None, eps=1e-6):
    """x [..., channels] (+ residual, the same shape, x's type or float32) -> its RMS norm times gamma; with a residual (norm, sum).

    The sum has the residual's type and is what the norm sees: y = gamma * sum / sqrt(mean(sum^2) + eps)."""
    gamma = _norm_inputs(x, gamma, residual, eps)
    if _wants_grad(x, gamma, residual):
        return _RmsNorm.apply(x, gamma, residual, eps)
    y, total, _, _ = _norm_forward(x, gamma, residual, eps, False)
    return y if total is None else (y, total)


def rms_norm_e4m3(x, gamma, residual=None, eps=1e-6, group=0):
    """rms_norm with its result in 8 bits: (q float8_e4m3fn, scale float32 [..., channels / group or 1]), with a residual (q, scale, sum).

    q * scale stands for the norm.  group: columns that share a scale, 32, 64 or 128; 0: the whole row.  It has no gradient."""
    gamma = _norm_inputs(x, gamma, residual, eps)
    cols = x.shape[-1]
    if not (group in (0, 32, 64, 128) and (group == 0 or cols % group == 0)):
        _refuse('group must be 0, 32, 64 or 128 and divide the channels')
    _no_grad('rms_norm_e4m3', x, gamma, residual)
    rows = x.numel() // cols
    x2, x_ld = _rows(x)
    q = _fresh(x.shape, x, torch.float8_e4m3fn)
    scale = _fresh((*x.shape[:-1], cols // group if group else 1), x, torch.float32)
    total = _fresh_like(residual) if residual is not None else None
    r2, r_ld = _rows(residual) if residual is not None else (None, 0)
    kind = _TYPES[x.dtype]
    _launch(lib.vc_rms_norm_e4m3, 'vc_rms_norm_e4m3', x, _p(x2), x_ld, _p(r2), r_ld, _p(gamma), _p(q), cols, _p(scale), _p(total), cols,
            eps, rows, cols, group, kind, _TYPES[residual.dtype] if residual is not None else kind)
    return (q, scale) if residual is None else (q, scale, total)


# ------------------------------------------------------------------------------------------------------------ utterances

def _utterances(x, seq_offsets):
    """(utterances, rows) of [batch, frames, ...] or of packed [rows, ...]."""
    if seq_offsets is None:
        if x.dim() != 3:
            _refuse('x must be [batch, frames, channels], or [rows, channels] with seq_offsets; got %s', tuple(x.shape))
        if x.shape[0] == 0:
            _refuse('x holds no utterance')
        return x.shape[0], x.shape[0] * x.shape[1]
    if x.dim() != 2:
        _refuse('with seq_offsets x must be [rows, channels], got %s', tuple(x.shape))
    if not (isinstance(seq_offsets, torch.Tensor) and seq_offsets.dtype == torch.int32 and seq_offsets.device == x.device and seq_offsets.dim() == 1 and
            seq_offsets.numel() >= 2):
        _refuse('seq_offsets must be an int32 tensor [utterances + 1] on %s', x.device)
    return seq_offsets.numel() - 1, x.shape[0]


def _slots(slots, rows, pool, ref):
    if slots is None:
        if rows > pool:
            _refuse('%d frames without slots, and a state of %d', rows, pool)
        return None
    _like(slots, ref, 'slots', (rows,), torch.int32)
    return slots.contiguous()


# ----------------------------------------------------------------------------------------------------------- convolution

def _conv_args(x, w, bias, initial, offsets, seqs, rows, silu):
    x2, x_ld = _rows(x)
    a = _lib.Conv1dArgs(x=_p(x2), w=_p(w), bias=_p(bias), initial=_p(initial), offsets=_p(offsets), x_ld=x_ld, rows=rows, cols=w.shape[1], taps=w.shape[0],
                        n_seqs=seqs, type=_TYPES[x.dtype], silu=int(silu), zero_tail=1)
    return a, x2


def _conv_forward(x, w, bias, initial, offsets, plan, want_final):
    seqs, rows, silu = plan
    a, x2 = _conv_args(x, w, bias, initial, offsets, seqs, rows, silu)
    y = _fresh_like(x)
    final = _fresh((seqs, a.taps - 1, a.cols), x) if want_final else None
    a.y, a.y_ld, a.final_state = _p(y), a.cols, _p(final)
    _launch(lib.vc_causal_conv1d_fwd, 'vc_causal_conv1d_fwd', x, C.byref(a))
    return (y, final) if want_final else y


class _CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, initial, offsets, plan, want_final):
        ctx.save_for_backward(x, w, bias, initial, offsets)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        return _conv_forward(x, w, bias, initial, offsets, plan, want_final)

    @staticmethod
    @_once
    def backward(ctx, dy, dfinal=None):
        x, w, bias, initial, offsets = ctx.saved_tensors
        seqs, rows, silu = ctx.plan
        a, x2 = _conv_args(x, w, bias, initial, offsets, seqs, rows, silu)
        if dy is None:
            dy = torch.zeros_like(x)
        dy2, a.dy_ld = _rows(dy)
        if dfinal is not None:
            dfinal = dfinal.contiguous()
        need = ctx.needs_input_grad
        dx = _fresh_like(x) if need[0] else None
        dw = _fresh_like(w) if need[1] else None
        dbias = _fresh(bias.shape, bias) if bias is not None and need[2] else None
        dinitial = _fresh(initial.shape, initial) if initial is not None and need[3] else None
        a.dy, a.dfinal, a.dx, a.dx_ld, a.dw, a.dbias, a.dinitial = _p(dy2), _p(dfinal), _p(dx), a.cols, _p(dw), _p(dbias), _p(dinitial)
        a.work_floats = lib.vc_causal_conv1d_bwd_work(C.byref(a))
        work = _fresh((a.work_floats,), w) if a.work_floats else None
        a.work = _p(work)
        _launch(lib.vc_causal_conv1d_bwd, 'vc_causal_conv1d_bwd', x, C.byref(a))
        return dx, dw, dbias, dinitial, None, None, None


def _conv_weights(x, w, bias, cols):
    if not (isinstance(w, torch.Tensor) and w.dim() == 2 and 2 <= w.shape[0] <= 8 and w.shape[1] == cols):
        _refuse('w must be [taps, %d] with 2 to 8 taps', cols)
    return _parameter(w, x, 'w', w.shape), _parameter(bias, x, 'bias', (cols,))


def causal_conv1d(x, w, bias=None, initial_state=None, seq_offsets=None, silu=True, return_final_state=False):
    """Convolution of each channel with its own `taps` filter weights, over its current and earlier frames: x, w [taps, channels] -> y like x.

    silu: y = p * sigmoid(p) of the convolution p.  initial_state [utterances, taps - 1, channels] (x's type, oldest first): the frames before
    each utterance, zeros otherwise.  return_final_state: (y, the same for what comes next)."""
    _activation(x, 'x')
    seqs, rows = _utterances(x, seq_offsets)
    w, bias = _conv_weights(x, w, bias, x.shape[-1])
    if initial_state is not None:
        initial_state = _like(initial_state, x, 'initial_state', (seqs, w.shape[0] - 1, x.shape[-1])).contiguous()
    if seq_offsets is not None:
        seq_offsets = seq_offsets.contiguous()
    args = x, w, bias, initial_state, seq_offsets, (seqs, rows, bool(silu)), bool(return_final_state)
    return (_CausalConv1d.apply if _wants_grad(x, w, bias, initial_state) else _conv_forward)(*args)


def causal_conv1d_step(x, state, w, bias=None, slots=None, silu=True):
    """One frame of each of x's [streams, channels]: y, and `state` [pool, taps - 1, channels] moved on by a frame in place.

    slots (int32 [streams]): the stream's entry in the pool; without them stream i has entry i.  A stream whose slot lies outside the pool, or is
    named by an earlier stream of the call, is padding: its y is zero and no state moves.  At most 4096 streams a call with slots."""
    _activation(x, 'x')
    if not (x.dim() == 2 and x.shape[1] > 0):
        _refuse('x must be [streams, channels], got %s', tuple(x.shape))
    rows, cols = x.shape
    w, bias = _conv_weights(x, w, bias, cols)
    if not (isinstance(state, torch.Tensor) and state.dim() == 3):
        _refuse('state must be [pool, taps - 1, channels]')
    _like(state, x, 'state', (state.shape[0], w.shape[0] - 1, cols))
    if not state.is_contiguous():
        _refuse('state must be contiguous: it is moved on in place')
    _no_grad('causal_conv1d_step', x, state, w, bias)
    slots = _slots(slots, rows, state.shape[0], x)
    x2, x_ld = _rows(x)
    y = _fresh_like(x)
    _launch(lib.vc_causal_conv1d_step, 'vc_causal_conv1d_step', x, _p(x2), x_ld, _p(state), _p(slots), _p(w), _p(bias), _p(y), cols, rows,
            state.shape[0], cols, w.shape[0], _TYPES[x.dtype], int(silu))
    return y


# ------------------------------------------------------------------------------------------------------------------ scan

def _grouped(t, lead, states, ref, name):
    """B or C as [..., groups, states]."""
    if not (isinstance(t, torch.Tensor) and t.dtype is ref.dtype and t.get_device() == ref.get_device()):
        _refuse('%s must be a %s tensor on %s', name, ref.dtype, ref.device)
    if t.dim() == len(lead) + 1:
        t = t.unsqueeze(-2)
    if not (t.dim() == len(lead) + 2 and t.shape[:-2] == lead and t.shape[-1] == states and t.shape[-2] > 0):
        _refuse('%s must be %s + [groups, %d] or + [%d], got %s', name, tuple(lead), states, states, tuple(t.shape))
    return t


def _scan_inputs(x, dt, A, B, C_, D, z, dt_bias):
    cols = x.shape[-1]
    _like(dt, x, 'dt', x.shape)
    if z is not None:
        _like(z, x, 'z', x.shape)
    if not (isinstance(A, torch.Tensor) and A.dim() == 2 and A.shape[0] == cols and 1 <= A.shape[1] <= 64):
        _refuse('A must be [%d, states] with 1 to 64 states', cols)
    A = _parameter(A, x, 'A', A.shape)
    B = _grouped(B, x.shape[:-1], A.shape[1], x, 'B')
    C_ = _grouped(C_, x.shape[:-1], A.shape[1], x, 'C')
    if not (B.shape[-2] == C_.shape[-2] and cols % B.shape[-2] == 0):
        _refuse('B and C must have the same groups, and these divide the channels')
    return A, B, C_, _parameter(D, x, 'D', (cols,)), _parameter(dt_bias, x, 'dt_bias', (cols,))


def _scan_args(x, dt, A, B, C_, D, z, dt_bias, initial, offsets, plan):
    seqs, rows, max_len, softplus = plan
    held = [_rows(x), _rows(dt), _rows(z) if z is not None else (None, 0), _rows(B, 2), _rows(C_, 2)]
    (x2, x_ld), (t2, t_ld), (z2, z_ld), (b2, b_ld), (c2, c_ld) = held
    a = _lib.ScanArgs(x=_p(x2), dt=_p(t2), z=_p(z2), B=_p(b2), C=_p(c2), A=_p(A), D=_p(D), dt_bias=_p(dt_bias), initial=_p(initial), offsets=_p(offsets),
                      x_ld=x_ld, dt_ld=t_ld, z_ld=z_ld, b_ld=b_ld, c_ld=c_ld, rows=rows, cols=A.shape[0], states=A.shape[1], groups=B.shape[-2],
                      n_seqs=seqs, type=_TYPES[x.dtype], softplus=int(softplus), zero_tail=1, max_len=max_len)
    return a, held


def _scan_forward(x, dt, A, B, C_, D, z, dt_bias, initial, offsets, plan, want_final, keep=False):
    a, held = _scan_args(x, dt, A, B, C_, D, z, dt_bias, initial, offsets, plan)
    y = _fresh_like(x)
    final = _fresh((plan[0], a.cols, a.states), A) if want_final else None
    a.y, a.y_ld, a.final_state = _p(y), a.cols, _p(final)
    saved = None
    if keep:
        a.saved_floats = lib.vc_selective_scan_saved(C.byref(a))
        saved = _fresh((a.saved_floats,), A)
        a.saved = _p(saved)
    a.work_floats = lib.vc_selective_scan_fwd_work(C.byref(a))
    work = _fresh((a.work_floats,), A) if a.work_floats > 0 else None
    a.work = _p(work)
    _launch(lib.vc_selective_scan_fwd, 'vc_selective_scan_fwd', x, C.byref(a))
    out = (y, final) if want_final else y
    return (out, saved) if keep else out


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C_, D, z, dt_bias, initial, offsets, plan, want_final):
        out, saved = _scan_forward(x, dt, A, B, C_, D, z, dt_bias, initial, offsets, plan, want_final, True)
        ctx.save_for_backward(x, dt, A, B, C_, D, z, dt_bias, initial, offsets, saved)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @_once
    def backward(ctx, dy, dfinal=None):
        x, dt, A, B, C_, D, z, dt_bias, initial, offsets, saved = ctx.saved_tensors
        a, held = _scan_args(x, dt, A, B, C_, D, z, dt_bias, initial, offsets, ctx.plan)
        if dy is None:
            dy = torch.zeros_like(x)
        dy2, a.dy_ld = _rows(dy)
        if dfinal is not None:
            dfinal = dfinal.contiguous()
        need = ctx.needs_input_grad
        dx, ddt, dB, dC, dA = _fresh_like(x), _fresh_like(x), _fresh_like(B), _fresh_like(C_), _fresh_like(A)
        dz = _fresh_like(x) if z is not None else None
        dD = _fresh(D.shape, A) if D is not None else None
        dbias = _fresh(dt_bias.shape, A) if dt_bias is not None else None
        dinitial = _fresh(initial.shape, A) if initial is not None and need[8] else None
        wide = a.groups * a.states
        a.dy, a.dfinal, a.dx, a.ddt, a.dz, a.dB, a.dC, a.dA = _p(dy2), _p(dfinal), _p(dx), _p(ddt), _p(dz), _p(dB), _p(dC), _p(dA)
        a.dD, a.ddt_bias, a.dinitial = _p(dD), _p(dbias), _p(dinitial)
        a.dx_ld = a.ddt_ld = a.dz_ld = a.cols
        a.db_ld = a.dc_ld = wide
        a.saved, a.saved_floats = _p(saved), saved.numel()
        a.work_floats = lib.vc_selective_scan_bwd_work(C.byref(a))
        work = _fresh((a.work_floats,), A)
        a.work = _p(work)
        _launch(lib.vc_selective_scan_bwd, 'vc_selective_scan_bwd', x, C.byref(a))
        grads = (dx, ddt, dA, dB, dC, dD, dz, dbias, dinitial)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None,) * 3


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, initial_state=None, seq_offsets=None, max_len=None, softplus=True, return_final_state=False):
    """Selective state space scan over the frames of each utterance:

        delta = softplus(dt + dt_bias);  h[t] = exp(delta[t] A) h[t-1] + delta[t] x[t] B[t];  y[t] = (C[t] h[t] + D x[t]) * z[t] sigmoid(z[t])

    x, dt, z: [batch, frames, channels] or packed [rows, channels]; A [channels, states] (finite, 1 to 64 states); B, C: [..., states] shared by all
    channels, or [..., groups, states], the channels of a group next to each other; D, dt_bias [channels].  softplus=False: delta = dt + dt_bias.
    initial_state [utterances, channels, states] (float32; zeros otherwise); return_final_state: (y, the state behind each utterance's last frame).
    max_len: the longest utterance where the program knows it: how a packed call is split, never what it gives."""
    _activation(x, 'x')
    seqs, rows = _utterances(x, seq_offsets)
    if x.shape[-1] == 0:
        _refuse('x has no channels')
    A, B, C, D, dt_bias = _scan_inputs(x, dt, A, B, C, D, z, dt_bias)
    if initial_state is not None:
        initial_state = _like(initial_state, x, 'initial_state', (seqs, *A.shape), torch.float32).contiguous()
    if not (max_len is None or max_len >= 0):
        _refuse('max_len must not be negative')
    tensors = (x, dt, A, B, C, D, z, dt_bias, initial_state)
    if seq_offsets is not None:
        seq_offsets = seq_offsets.contiguous()
    plan = seqs, rows, int(max_len or 0), bool(softplus)
    return (_SelectiveScan.apply if _wants_grad(*tensors) else _scan_forward)(*tensors, seq_offsets, plan, bool(return_final_state))


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, slots=None, softplus=True):
    """One frame of each of x's [streams, channels] (dt, z alike; B, C [streams, states] or [streams, groups, states]): y, and `state`
    [pool, channels, states] (float32) moved on in place.  slots as in causal_conv1d_step."""
    _activation(x, 'x')
    if not (x.dim() == 2 and x.shape[1] > 0):
        _refuse('x must be [streams, channels], got %s', tuple(x.shape))
    rows, cols = x.shape
    A, B, C, D, dt_bias = _scan_inputs(x, dt, A, B, C, D, z, dt_bias)
    if not (isinstance(state, torch.Tensor) and state.dim() == 3):
        _refuse('state must be [pool, channels, states]')
    _like(state, x, 'state', (state.shape[0], *A.shape), torch.float32)
    if not state.is_contiguous():
        _refuse('state must be contiguous: it is moved on in place')
    _no_grad('selective_scan_step', x, dt, A, B, C, state, D, z, dt_bias)
    slots = _slots(slots, rows, state.shape[0], x)
    (x2, x_ld), (t2, t_ld), (b2, b_ld), (c2, c_ld) = _rows(x), _rows(dt), _rows(B, 2), _rows(C, 2)
    z2, z_ld = _rows(z) if z is not None else (None, 0)
    y = _fresh_like(x)
    _launch(lib.vc_selective_scan_step, 'vc_selective_scan_step', x, _p(x2), x_ld, _p(t2), t_ld, _p(z2), z_ld, _p(b2), b_ld, _p(c2), c_ld,
            _p(A), _p(D), _p(dt_bias), _p(state), _p(slots), _p(y), cols, rows, state.shape[0], cols, A.shape[1], B.shape[-2], _TYPES[x.dtype], int(softplus))
    return y
