"""Sequence operators on torch GPU tensors: what a causal model of frames is built of, beside the utterance-wide blocks of module.py.

The reference's generator looks ahead (SAME convolutions, module.py:32-40) and normalises over a whole utterance (module.py:135-146).  These
operators look back only: a model of them trains on packed utterances and converts a live stream frame by frame, with the same results.

    y, stream = rms_norm(x, gamma, stream)            # stream + x, and its norm
    u = causal_conv1d(y @ W, w, bias)                 # a few earlier frames, channel by channel
    v = selective_scan(u, dt, A, B, C, D=D, z=z)      # all earlier frames, through a state of `states` numbers a channel

Frames are rows: tensors are [batch, frames, channels], or [rows, channels] with `seq_offsets` (int32, [n + 1], rising, on the same device) where
utterances of different lengths lie one behind the other; lengths of zero are fine, and rows ahead of the first utterance or behind the last give
zeros.  Rows are taken in place (column slices of a product, for one) unless they lie very far apart, more than 2^15 elements for the convolution (2^20 from
256 channels on) and 2^24 for the scan: those are copied.  Activations are fp32, bf16 or fp16 (one type in a call); parameters, recurrent states and
parameter gradients are fp32, and every sum is.  The kernels are those of include/vc_cyclegan.h; gradients are deterministic.

A backward pass that is captured into a graph must not meet an eager autograd graph of the same leaves that is still alive: torch's gradient
accumulators belong to the stream they were made on.  Drop the eager outputs first."""
import torch

from . import _lib


def _load_binding():
    """csrc/vc_seq_torch.cpp, built for this torch and these sources, and bound to the library that _lib loaded."""
    import ctypes
    import importlib
    import os
    want = _lib._bmod.binding_id()
    if not os.path.exists(_lib._bmod.BINDING):
        raise ImportError('_seq.so not built: run `python -c "import __graft_entry__ as g; g.build()"`')
    seq = importlib.import_module('._seq', __package__)
    if seq.build_id != want and not os.environ.get('VC_ALLOW_STALE_LIB'):
        raise ImportError('_seq.so was built from other sources or for another torch (build id %s, tree %s): run '
                          '`python -c "import __graft_entry__ as g; g.build()"`' % (seq.build_id, want))
    entries = [n for n, _, _ in _lib.SIGNATURES if n.startswith(('vc_rms_norm', 'vc_causal_conv1d', 'vc_selective_scan', 'vc_last_error'))]
    seq.bind({n: ctypes.cast(getattr(_lib.lib, n), ctypes.c_void_p).value for n in entries}, _lib.VcError, torch._C._cuda_getCurrentRawStream)
    return seq


_seq = _load_binding()


def rms_norm(x, gamma, residual=None, eps=1e-6):
    """x [..., channels] (+ residual, the same shape, x's type or float32) -> its RMS norm times gamma; with a residual (norm, sum).

    The sum has the residual's type and is what the norm sees: y = gamma * sum / sqrt(mean(sum^2) + eps)."""
    return _seq.rms_norm(x, gamma, residual, eps)


def rms_norm_e4m3(x, gamma, residual=None, eps=1e-6, group=0):
    """rms_norm with its result in 8 bits: (q float8_e4m3fn, scale float32 [..., channels / group or 1]), with a residual (q, scale, sum).

    q * scale stands for the norm.  group: columns that share a scale, 32, 64 or 128; 0: the whole row.  It has no gradient."""
    return _seq.rms_norm_e4m3(x, gamma, residual, eps, group)


def causal_conv1d(x, w, bias=None, initial_state=None, seq_offsets=None, silu=True, return_final_state=False):
    """Convolution of each channel with its own `taps` filter weights, over its current and earlier frames: x, w [taps, channels] -> y like x.

    silu: y = p * sigmoid(p) of the convolution p.  initial_state [utterances, taps - 1, channels] (x's type, oldest first): the frames before
    each utterance, zeros otherwise.  return_final_state: (y, the same for what comes next)."""
    return _seq.causal_conv1d(x, w, bias, initial_state, seq_offsets, bool(silu), bool(return_final_state))


def causal_conv1d_step(x, state, w, bias=None, slots=None, silu=True):
    """One frame of each of x's [streams, channels]: y, and `state` [pool, taps - 1, channels] moved on by a frame in place.

    slots (int32 [streams]): the stream's entry in the pool; without them stream i has entry i.  A stream whose slot lies outside the pool, or is
    named by an earlier stream of the call, is padding: its y is zero and no state moves.  At most 4096 streams a call with slots, 65535 without."""
    return _seq.causal_conv1d_step(x, state, w, bias, slots, bool(silu))


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, initial_state=None, seq_offsets=None, max_len=None, softplus=True, return_final_state=False):
    """Selective state space scan over the frames of each utterance:

        delta = softplus(dt + dt_bias);  h[t] = exp(delta[t] A) h[t-1] + delta[t] x[t] B[t];  y[t] = (C[t] h[t] + D x[t]) * z[t] sigmoid(z[t])

    x, dt, z: [batch, frames, channels] or packed [rows, channels]; A [channels, states] (finite, 1 to 64 states); B, C: [..., states] shared by all
    channels, or [..., groups, states], the channels of a group next to each other; D, dt_bias [channels].  softplus=False: delta = dt + dt_bias.
    A frame masked by dt = -inf or its type's lowest value leaves the state as it is.
    initial_state [utterances, channels, states] (float32; zeros otherwise); return_final_state: (y, the state behind each utterance's last frame).
    max_len: the longest utterance where the program knows it: how a packed call is split, never what it gives."""
    return _seq.selective_scan(x, dt, A, B, C, D, z, dt_bias, initial_state, seq_offsets, max_len or 0, bool(softplus), bool(return_final_state))


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, slots=None, softplus=True):
    """One frame of each of x's [streams, channels] (dt, z alike; B, C [streams, states] or [streams, groups, states]): y, and `state`
    [pool, channels, states] (float32) moved on in place.  slots as in causal_conv1d_step."""
    return _seq.selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, slots, bool(softplus))
