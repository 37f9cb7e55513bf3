"""The sequence operators in 64 bits on the CPU, from their definitions, utterance by utterance and frame by frame (test infrastructure).

Every function takes tensors of any floating type and returns float64.  absolute=True gives the same sums over absolute values: the magnitude that
rounding errors of the terms are relative to."""
import torch


def _d(t):
    return None if t is None else t.detach().cpu().double()


def _abs(t, on):
    return t.abs() if on and t is not None else t


def silu(p):
    return p / (1 + torch.exp(-p))


def dsilu(p, absolute=False):
    s = 1 / (1 + torch.exp(-p))
    return s * (1 + (p.abs() if absolute else p) * (1 - s))


def rms_norm(t, gamma, eps, dy=None, dsum=None, absolute=False):
    """t: the stored sum.  -> y, and with dy (dt, dgamma)."""
    t, gamma, dy, dsum = _d(t), _d(gamma), _d(dy), _d(dsum)
    rstd = 1 / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps)
    that = t * rstd
    if dy is None:
        return that * gamma
    that, gamma, dy, dsum = (_abs(v, absolute) for v in (that, gamma, dy, dsum))
    g = dy * gamma
    m = that * (g * that).mean(-1, keepdim=True)
    dt = rstd * (g + m if absolute else g - m)
    return that * gamma, dt if dsum is None else dt + dsum, (dy * that).reshape(-1, t.shape[-1]).sum(0)


def conv1d(x, w, bias, initial, lengths, silu_on, dy=None, dfinal=None, absolute=False):
    """x [rows, cols] packed.  -> dict with p, y, final and (with dy) dx, dw, dbias, dinitial.  Rows behind the last utterance are zero.
    absolute: p is the sum of absolute values; the factor silu'(p) of the gradients is s (1 + |p| (1 - s)) at the true p, and half that sum more: an
    error of p moves it by at most half as much (|silu''| <= 1/2)."""
    x, w, bias, initial, dy, dfinal = (_d(v) for v in (x, w, bias, initial, dy, dfinal))
    k, cols = w.shape
    n = len(lengths)
    out = dict(p=torch.zeros_like(x), y=torch.zeros_like(x), final=torch.zeros(n, k - 1, cols, dtype=torch.float64))
    if dy is not None:
        out.update(dx=torch.zeros_like(x), dw=torch.zeros_like(w), dbias=torch.zeros(cols, dtype=torch.float64), dinitial=torch.zeros_like(out['final']))
    at = 0
    for i, m in enumerate(lengths):
        ahead = torch.zeros(k - 1, cols, dtype=torch.float64) if initial is None else initial[i]
        axis = torch.cat([ahead, x[at:at + m]])
        true = sum(axis[j:j + m] * w[j] for j in range(k)) + (0 if bias is None else bias)
        axis = _abs(axis, absolute)
        wa = _abs(w, absolute)
        p = sum(axis[j:j + m] * wa[j] for j in range(k)) + (0 if bias is None else _abs(bias, absolute))
        out['p'][at:at + m] = p
        out['y'][at:at + m] = silu(true) if silu_on else true
        out['final'][i] = axis[m:m + k - 1]
        if dy is not None:
            factor = dsilu(true, absolute) if silu_on else torch.ones_like(true)
            if absolute and silu_on:
                factor = factor + 0.5 * p
            g = _abs(dy[at:at + m], absolute) * factor
            daxis = torch.zeros_like(axis)
            for j in range(k):
                daxis[j:j + m] += g * wa[j]
                out['dw'][j] += (g * axis[j:j + m]).sum(0)
            if dfinal is not None:
                daxis[m:m + k - 1] += _abs(dfinal[i], absolute)
            out['dbias'] += g.sum(0)
            out['dx'][at:at + m] = daxis[k - 1:]
            out['dinitial'][i] = daxis[:k - 1]
        at += m
    return out


def scan(x, dt, A, B, C, D, z, dt_bias, initial, lengths, softplus=True, dy=None, dfinal=None, absolute=False):
    """x [rows, cols] packed; B, C [rows, groups, states].  -> dict with y, final and (with dy) dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dinitial."""
    x, dt, A, B, C, D, z, dt_bias, initial, dy, dfinal = (_d(v) for v in (x, dt, A, B, C, D, z, dt_bias, initial, dy, dfinal))
    rows, cols = x.shape
    groups, n = B.shape[1:]
    wide = cols // groups
    v = dt if dt_bias is None else dt + dt_bias
    delta = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
    slope = torch.sigmoid(v) if softplus else torch.ones_like(v)
    gate = torch.ones_like(x) if z is None else silu(z)
    dgate = torch.zeros_like(x) if z is None else dsilu(z, absolute)
    D = torch.zeros(cols, dtype=torch.float64) if D is None else D
    a = torch.exp(delta[..., None] * A)
    x, B, C, D, initial, gate, dgate, dy, dfinal = (_abs(t, absolute) for t in (x, B, C, D, initial, gate, dgate, dy, dfinal))
    size, Aw = _abs(delta, absolute), _abs(A, absolute)
    B, C = B.repeat_interleave(wide, 1), C.repeat_interleave(wide, 1)
    h = torch.zeros(rows, cols, n, dtype=torch.float64)
    before = torch.zeros_like(h)
    out = dict(y=torch.zeros_like(x), final=torch.zeros(len(lengths), cols, n, dtype=torch.float64), delta=delta)
    at, spans = 0, []
    for i, m in enumerate(lengths):
        s = out['final'][i] if initial is None else initial[i].clone()
        for t in range(at, at + m):
            before[t] = s
            s = a[t] * s + (size[t] * x[t])[:, None] * B[t]
            h[t] = s
        out['final'][i] = s
        spans.append((at, at + m))
        at += m
    pre = (h * C).sum(-1) + D * x
    out['y'][:at] = (pre * gate)[:at]
    if dy is None:
        return out
    dp = dy * gate
    dp[at:] = 0
    dh = torch.zeros_like(h)
    out['dinitial'] = torch.zeros_like(out['final'])
    for i, (lo, hi) in enumerate(spans):
        s = torch.zeros(cols, n, dtype=torch.float64) if dfinal is None else dfinal[i].clone()
        for t in reversed(range(lo, hi)):
            dh[t] = s + dp[t][:, None] * C[t]
            s = a[t] * dh[t]
        out['dinitial'][i] = s
    q = dh * a * before
    into = (dh * B).sum(-1)
    ddelta = ((q * Aw).sum(-1) + x * into) * slope
    ddelta[at:] = 0
    dx = dp * D + size * into
    dx[at:] = 0
    out.update(dx=dx, ddt=ddelta, dA=(q * size[..., None])[:at].sum(0), dD=(dp * x)[:at].sum(0), ddt_bias=ddelta[:at].sum(0),
               dB=(dh * (size * x)[..., None]).view(rows, groups, wide, n).sum(2), dC=(dp[..., None] * h).view(rows, groups, wide, n).sum(2))
    out['dz'] = dy * pre * dgate
    for k in ('dB', 'dC', 'dz'):
        out[k][at:] = 0
    return out
