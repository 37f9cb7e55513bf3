"""The sequence operators (RMS norm, short causal convolution, selective state space scan): what is measured of them.

`listed()` names the cases, `draw()` makes more of the same ranges, `prepare()` makes the inputs that a program has in hand, `run()` is one pass:
in elementary torch operations, or through the framework where `own` is set.  `exact()` gives the same results from the definitions in 64 bits.

Rows are frames, columns are channels.  Utterances of different lengths lie one behind the other (`offsets`)."""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}
E4M3_MAX = 448.0
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one frame of a live stream through a norm: the smallest call, all latency
        dict(name='norm-frame', op='norm', rows=1, cols=512, type='f32', stream='f32', train=False),
        # a training batch of 128 crops of 128 frames, 16-bit activations on a 16-bit residual stream
        dict(name='norm-train', op='norm', rows=16384, cols=1024, type='bf16', stream='bf16', train=True),
        # four utterances of 2208 frames on their way into an 8-bit product, a scale for each 128 columns, fp32 residual stream
        dict(name='norm-e4m3', op='norm8', rows=8832, cols=2048, type='bf16', stream='f32', group=128),
        # eight live streams, one frame each
        dict(name='conv-frame', op='conv_step', streams=8, pool=16, cols=1024, taps=4, type='bf16'),
        # utterances of different lengths, packed, in the framework's own precision; the state goes on to the next call
        dict(name='conv-packed', op='conv', seqs=13, rows=9001, cols=1000, taps=4, type='f32', packed=True, states=True, train=False),
        # a training batch of 64 crops of 128 frames, wide
        dict(name='conv-train', op='conv', seqs=64, rows=8192, cols=2048, taps=4, type='bf16', packed=False, states=False, train=True),
        # one live stream, one frame
        dict(name='scan-frame', op='scan_step', streams=1, pool=1, cols=1024, states=16, groups=1, type='f32'),
        # 256 live streams out of a pool of 512, one frame each
        dict(name='scan-streams', op='scan_step', streams=256, pool=512, cols=2048, states=16, groups=1, type='bf16'),
        # one long recording: few channels beside a long axis
        dict(name='scan-long', op='scan', seqs=1, rows=8192, cols=1024, states=16, groups=1, type='bf16', packed=False, carry=True, train=False),
        # utterances of different lengths, packed
        dict(name='scan-packed', op='scan', seqs=23, rows=16001, cols=1024, states=16, groups=1, type='bf16', packed=True, carry=False, train=False),
        # a training batch of 64 crops of 128 frames
        dict(name='scan-train', op='scan', seqs=64, rows=8192, cols=1024, states=16, groups=1, type='bf16', packed=False, carry=False, train=True),
        # training on one utterance of 2208 frames in fp32, odd sizes, two groups, the state carried in and out
        dict(name='scan-train-long', op='scan', seqs=1, rows=2208, cols=1002, states=12, groups=2, type='f32', packed=False, carry=True, train=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'norm8', 'conv', 'conv_step', 'scan', 'scan', 'scan_step'])
    t = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'norm':
        cols = _spread(rng, 64, 8192)
        rows = _spread(rng, 1, min(16384, (1 << 24) // cols))
        return dict(op=op, rows=rows, cols=cols, type=t, stream=rng.choice([t, 'f32']), train=rng.random() < 0.5)
    if op == 'norm8':
        group = rng.choice([0, 32, 64, 128])
        cols = _spread(rng, 64, 8192) if group == 0 else group * rng.randint(1, 8192 // group)
        return dict(op=op, rows=_spread(rng, 1, min(16384, (1 << 24) // cols)), cols=cols, type=t, stream=rng.choice([t, 'f32']), group=group)
    if op == 'conv':
        cols = _spread(rng, 24, 4096)
        seqs = _spread(rng, 1, 64)
        packed = rng.random() < 0.5
        rows = _spread(rng, seqs, min(16384, (1 << 24) // cols))
        return dict(op=op, seqs=seqs, rows=rows if packed else max(1, rows // seqs) * seqs, cols=cols, taps=rng.choice([2, 3, 4, 4]), type=t, packed=packed,
                    states=rng.random() < 0.5, train=rng.random() < 0.5)
    if op == 'conv_step':
        streams = _spread(rng, 1, 512)
        return dict(op=op, streams=streams, pool=streams + rng.randint(0, 64), cols=_spread(rng, 24, 4096), taps=rng.choice([2, 3, 4, 4]), type=t)
    states = rng.choice([4, 8, 12, 16, 16, 16, 16, 21, 32])
    groups = rng.choice([1, 1, 2, 4])
    if op == 'scan_step':
        streams = _spread(rng, 1, 512)
        cols = groups * _spread(rng, 8, min(1024, (1 << 23) // (states * streams * groups)))
        return dict(op=op, streams=streams, pool=streams + rng.randint(0, 64), cols=cols, states=states, groups=groups, type=t)
    train = rng.random() < 0.5
    cols = groups * _spread(rng, 16, 512)
    seqs = _spread(rng, 1, 64)
    packed = rng.random() < 0.5
    rows = _spread(rng, seqs, min(16384, (1 << (27 if train else 28)) // (16 * ((states + 15) // 16) * cols)))
    return dict(op=op, seqs=seqs, rows=rows if packed else max(1, rows // seqs) * seqs, cols=cols, states=states, groups=groups, type=t, packed=packed,
                carry=rng.random() < 0.5, train=train)


# --------------------------------------------------------------------------------------------------------------- inputs

def _lengths(case, seed):
    """The utterances' lengths: equal ones, or drawn ones that add up to the case's rows (a short one among them now and then)."""
    n, rows = case['seqs'], case['rows']
    if not case['packed']:
        return [rows // n] * n
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(n, generator=g) ** 2 + 0.01
    cuts = (torch.cumsum(w, 0) / w.sum() * rows).round().long().tolist()
    cuts[-1] = rows
    return [b - a for a, b in zip([0] + cuts[:-1], cuts)]


def prepare(case, seed):
    dev = 'cuda'
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case['type']]
    op, cols = case['op'], case['cols']

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    s = dict(op=op, train=case.get('train', False), type=t)
    if op in ('norm', 'norm8'):
        st = TYPES[case['stream']]
        s.update(x=normal(case['rows'], cols), residual=normal(case['rows'], cols, scale=3.0, dtype=st),
                 gamma=1.0 + normal(cols, scale=0.1, dtype=torch.float32), group=case.get('group'))
        if s['train']:
            s.update(dy=normal(case['rows'], cols), dtotal=normal(case['rows'], cols, dtype=st))
        leaves = ('x', 'residual', 'gamma')
    elif op in ('conv', 'conv_step'):
        k = case['taps']
        s.update(w=normal(k, cols, scale=k ** -0.5, dtype=torch.float32), bias=normal(cols, scale=0.1, dtype=torch.float32))
        if op == 'conv_step':
            s.update(x=normal(case['streams'], cols), state=normal(case['pool'], k - 1, cols),
                     slots=torch.randperm(case['pool'], generator=g, device=dev)[:case['streams']].int())
        leaves = ('x', 'w', 'bias', 'initial')
    else:
        n, gr = case['states'], case['groups']
        step = torch.exp(torch.rand(cols, generator=g, device=dev) * math.log(100.0) + math.log(0.001))        # steps between 0.001 and 0.1
        s.update(A=-(torch.arange(1, n + 1, device=dev, dtype=torch.float32) * torch.exp(normal(cols, n, scale=0.1, dtype=torch.float32))),
                 D=normal(cols, dtype=torch.float32), dt_bias=step + torch.log(-torch.expm1(-step)))
        if op == 'scan_step':
            rows = case['streams']
            s.update(state=normal(case['pool'], cols, n, scale=0.3, dtype=torch.float32),
                     slots=torch.randperm(case['pool'], generator=g, device=dev)[:rows].int())
        else:
            rows = case['rows']
        s.update(x=normal(rows, cols), dt=normal(rows, cols, scale=0.5), z=normal(rows, cols), B=normal(rows, gr, n), C=normal(rows, gr, n))
        leaves = ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'initial')
    if op in ('conv', 'scan'):
        lengths = _lengths(case, seed)
        edges = [0]
        for n_ in lengths:
            edges.append(edges[-1] + n_)
        live = [i for i, n_ in enumerate(lengths) if n_]
        s.update(packed=case['packed'], seqs=case['seqs'], max_len=max(lengths), offsets=torch.tensor(edges, dtype=torch.int32, device=dev),
                 live=torch.tensor(live, device=dev), first=torch.tensor([edges[i] for i in live], device=dev),
                 last=torch.tensor([edges[i + 1] - 1 for i in live], device=dev))
        if op == 'conv':
            s['x'] = normal(case['rows'], cols)
            s['initial'] = normal(case['seqs'], case['taps'] - 1, cols) if case['states'] else None
        else:
            s['initial'] = normal(case['seqs'], cols, case['states'], scale=0.3, dtype=torch.float32) if case['carry'] else None
        if s['train']:
            s['dy'] = normal(case['rows'], cols)
            if s['initial'] is not None:
                s['dfinal'] = torch.randn(s['initial'].shape, generator=g, device=dev).to(s['initial'].dtype)
    if s['train']:
        s['leaves'] = [k for k in leaves if s.get(k) is not None]
        for k in s['leaves']:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------- through the framework

def _sequence():
    import vcgan_pkg  # noqa: F401
    from voice_converter_cyclegan_amd import sequence
    return sequence


def _shaped(s, v):
    """Rows as [utterances, frames, ...] where the lengths are equal: the unpacked calling form."""
    return v if s['packed'] or v is None else v.view(s['seqs'], -1, *v.shape[1:])


def _own(s):
    S = _sequence()
    op = s['op']
    if op == 'norm8':
        return S.rms_norm_e4m3(s['x'], s['gamma'], s['residual'], eps=EPS, group=s['group'])
    if op == 'conv_step':
        y = S.causal_conv1d_step(s['x'], s['state'], s['w'], s['bias'], slots=s['slots'])
        return y, s['state']
    if op == 'scan_step':
        y = S.selective_scan_step(s['x'], s['dt'], s['A'], s['B'], s['C'], s['state'], D=s['D'], z=s['z'], dt_bias=s['dt_bias'], slots=s['slots'])
        return y, s['state']
    if op == 'norm':
        out = S.rms_norm(s['x'], s['gamma'], s['residual'], eps=EPS)
        seeds = (s['dy'], s['dtotal']) if s['train'] else None
    else:
        carry = s['initial'] is not None
        off = dict(seq_offsets=s['offsets']) if s['packed'] else {}
        if op == 'conv':
            out = S.causal_conv1d(_shaped(s, s['x']), s['w'], s['bias'], initial_state=s['initial'], return_final_state=carry, **off)
        else:
            if s['packed']:
                off['max_len'] = s['max_len']
            out = S.selective_scan(_shaped(s, s['x']), _shaped(s, s['dt']), s['A'], _shaped(s, s['B']), _shaped(s, s['C']), D=s['D'], z=_shaped(s, s['z']),
                                   dt_bias=s['dt_bias'], initial_state=s['initial'], return_final_state=carry, **off)
        out = out if carry else (out,)
        seeds = ((_shaped(s, s['dy']), s['dfinal']) if carry else (_shaped(s, s['dy']),)) if s['train'] else None
    grads = torch.autograd.grad(out, [s[k] for k in s['leaves']], seeds) if s['train'] else ()
    return [o.detach().reshape(s['x'].shape) if i == 0 else o.detach() for i, o in enumerate(out)], list(grads)


# ----------------------------------------------------------------------------------------- in elementary torch operations

def _plain_norm(s):
    st = s['residual'].dtype
    total = (s['x'].float() + s['residual'].float()).to(st)
    t = total.float()
    rstd = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    that = t * rstd
    y = that * s['gamma']
    if s['op'] == 'norm8':
        v = y.view(y.shape[0], -1, s['group'] or y.shape[1])
        scale = v.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100) / E4M3_MAX
        return (v / scale).view_as(y).to(torch.float8_e4m3fn), scale.squeeze(-1), total
    if not s['train']:
        return [y.to(s['type']), total], []
    dy = s['dy'].float()
    gy = dy * s['gamma']
    dt = s['dtotal'].float() + rstd * (gy - that * (gy * that).mean(-1, keepdim=True))
    return [y.to(s['type']), total], [dt.to(s['type']), dt.to(st), (dy * that).sum(0)]


def _windows(s, x):
    """[rows, taps, cols]: what each row's taps look at, and which row of the padded sequence axis that is.  Every utterance has its taps - 1 earlier
    frames (its initial state or zeros) laid before it."""
    k = s['w'].shape[0]
    rows, cols = x.shape
    ahead = torch.zeros(s['seqs'], k - 1, cols, device=x.device) if s['initial'] is None else s['initial'].float()
    sizes = (s['offsets'][1:] - s['offsets'][:-1]).long()
    of = torch.repeat_interleave(torch.arange(s['seqs'], device=x.device), sizes, output_size=rows)
    at = torch.arange(rows, device=x.device) + (of + 1) * (k - 1)                       # a row's place on the axis with the earlier frames in it
    heads = s['offsets'][:-1].long() + torch.arange(s['seqs'], device=x.device) * (k - 1)
    head = (heads[:, None] + torch.arange(k - 1, device=x.device)).reshape(-1)
    axis = torch.empty(rows + s['seqs'] * (k - 1), cols, device=x.device)
    axis[at] = x
    axis[head] = ahead.reshape(-1, cols)
    look = at[:, None] + torch.arange(1 - k, 1, device=x.device)
    ends = heads + sizes                                                                # the last taps - 1 frames of every utterance
    tail = ends[:, None] + torch.arange(k - 1, device=x.device)
    return axis, look, at, head, tail


def _plain_conv(s):
    x = s['x'].float()
    axis, look, at, head, tail = _windows(s, x)
    seen = axis[look]
    p = (seen * s['w']).sum(1) + s['bias']
    sig = torch.sigmoid(p)
    out = [(p * sig).to(s['type'])]
    if s['initial'] is not None:
        out.append(axis[tail].to(s['type']))
    if not s['train']:
        return out, []
    gr = s['dy'].float() * sig * (1 + p * (1 - sig))
    daxis = torch.zeros_like(axis)
    if s['initial'] is not None:
        daxis.index_add_(0, tail.reshape(-1), s['dfinal'].float().reshape(-1, axis.shape[1]))
    k = s['w'].shape[0]
    spread = torch.zeros(axis.shape[0] + k - 1, axis.shape[1], device=axis.device)       # g on the padded axis, zeros where no row is
    spread[at] = gr
    after = torch.arange(axis.shape[0], device=axis.device)[:, None] + torch.arange(k - 1, -1, -1, device=axis.device)
    daxis += (spread[after] * s['w']).sum(1)
    grads = [daxis[at].to(s['type']), (gr[:, None] * seen).sum(0), gr.sum(0)]
    if s['initial'] is not None:
        grads.append(daxis[head].view_as(s['initial']).to(s['type']))
    return out, grads


def _plain_conv_step(s):
    slots = s['slots'].long()
    seen = torch.cat([s['state'][slots], s['x'][:, None]], 1)
    p = (seen.float() * s['w']).sum(1) + s['bias']
    s['state'][slots] = seen[:, 1:]
    return (p * torch.sigmoid(p)).to(s['type']), s['state']


def _recur(a, b, longest):
    """h[t] = a[t] h[t-1] + b[t] along the first axis, by doubling: after the step of size n every row holds what its last 2 n rows bring."""
    n = 1
    while n < longest:
        b = torch.cat([b[:n], torch.addcmul(b[n:], a[n:], b[:-n])])
        a = torch.cat([a[:n], a[n:] * a[:-n]])
        n *= 2
    return b


def _per_channel(v, cols):
    """[rows, groups, states] -> [rows, groups, channels of a group, states], broadcast over the channels."""
    return v.float()[:, :, None].expand(-1, -1, cols // v.shape[1], -1)


def _plain_scan(s):
    x, z = s['x'].float(), s['z'].float()
    rows, cols = x.shape
    groups, n = s['B'].shape[1:]
    v = s['dt'].float() + s['dt_bias']
    delta = v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))
    a = torch.exp(delta[..., None] * s['A'])
    dx_ = (delta * x).view(rows, groups, -1, 1)
    b = (dx_ * _per_channel(s['B'], cols)).reshape(rows, cols, n)
    c = _per_channel(s['C'], cols)
    h0 = torch.zeros(s['seqs'], cols, n, device=x.device) if s['initial'] is None else s['initial']
    first, last, live = s['first'], s['last'], s['live']
    b[first] += a[first] * h0[live]
    inner = a.clone()
    inner[first] = 0
    h = _recur(inner, b, s['max_len'])
    y = (h.view(rows, groups, -1, n) * c).sum(-1).view(rows, cols) + s['D'] * x
    sig = torch.sigmoid(z)
    out = [(y * z * sig).to(s['type'])]
    if s['initial'] is not None:
        out.append(h0.clone())
        out[1][live] = h[last]
    if not s['train']:
        return out, []
    dy = s['dy'].float()
    dz = dy * y * sig * (1 + z * (1 - sig))
    dp = dy * z * sig
    seed = (dp.view(rows, groups, -1, 1) * c).reshape(rows, cols, n)
    if s['initial'] is not None:
        seed[last] += s['dfinal'][live]
    behind = torch.cat([inner[1:], torch.zeros_like(inner[:1])])
    dh = _recur(behind.flip(0), seed.flip(0), s['max_len']).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = h0[live]
    through = dh * before * a
    into = (dh.view(rows, groups, -1, n) * _per_channel(s['B'], cols)).sum(-1).view(rows, cols)
    ddelta = (through * s['A']).sum(-1) + into * x
    dv = ddelta * torch.sigmoid(v)
    t = s['type']
    grads = [(dp * s['D'] + delta * into).to(t), dv.to(t), (through * delta[..., None]).sum(0), (dh.view(rows, groups, -1, n) * dx_).sum(2).to(t),
             (dp.view(rows, groups, -1, 1) * h.view(rows, groups, -1, n)).sum(2).to(t), (dp * x).sum(0), dz.to(t), dv.sum(0)]
    if s['initial'] is not None:
        dh0 = s['dfinal'].clone()
        dh0[live] = dh[first] * a[first]
        grads.append(dh0)
    return out, grads


def _plain_scan_step(s):
    x, z = s['x'].float(), s['z'].float()
    rows, cols = x.shape
    groups, n = s['B'].shape[1:]
    slots = s['slots'].long()
    v = s['dt'].float() + s['dt_bias']
    delta = v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))
    b = (delta * x).view(rows, groups, -1, 1) * _per_channel(s['B'], cols)
    h = torch.exp(delta[..., None] * s['A']) * s['state'][slots] + b.reshape(rows, cols, n)
    s['state'][slots] = h
    y = (h.view(rows, groups, -1, n) * _per_channel(s['C'], cols)).sum(-1).view(rows, cols) + s['D'] * x
    return (y * z * torch.sigmoid(z)).to(s['type']), s['state']


PLAIN = {'norm': _plain_norm, 'norm8': _plain_norm, 'conv': _plain_conv, 'conv_step': _plain_conv_step, 'scan': _plain_scan, 'scan_step': _plain_scan_step}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state['op']](state)


# ------------------------------------------------------------------------------------------------------------------ work

def work(case):
    """Every input read once, every output written once; one multiply-add counts two, an exponential one."""
    op, e, cols = case['op'], SIZE[case['type']], case['cols']
    train = case.get('train', False)
    if op in ('norm', 'norm8'):
        n, es = case['rows'] * cols, SIZE[case['stream']]
        out = 1 if op == 'norm8' else e
        moved = n * (e + es) + n * (out + es) + 4 * cols
        if op == 'norm8':
            moved += 4 * case['rows'] * (cols // case['group'] if case['group'] else 1)
        if train:
            moved += n * (e + es) + n * e + (n * es if es != e else 0) + 4 * cols
        return dict(bytes=moved, flops=n * (6 + (10 if train else 0)))
    if op == 'conv':
        n, k = case['rows'] * cols, case['taps']
        moved = 2 * n * e + 4 * (k + 1) * cols + (2 * case['seqs'] * (k - 1) * cols * e if case['states'] else 0)
        if train:
            moved += 2 * n * e + 4 * (k + 1) * cols + (2 * case['seqs'] * (k - 1) * cols * e if case['states'] else 0)
        return dict(bytes=moved, flops=n * (2 * k + 4) * (3 if train else 1))
    if op == 'conv_step':
        n, k = case['streams'] * cols, case['taps']
        return dict(bytes=2 * n * e + 2 * n * (k - 1) * e + 4 * (k + 1) * cols + 4 * case['streams'], flops=n * (2 * k + 4))
    n = case['states']
    weights = 4 * cols * (n + 2)
    if op == 'scan_step':
        r = case['streams']
        return dict(bytes=4 * r * cols * e + 2 * r * case['groups'] * n * e + 8 * r * cols * n + weights + 4 * r, flops=r * cols * (7 * n + 12))
    r = case['rows']
    moved = 4 * r * cols * e + 2 * r * case['groups'] * n * e + weights + (8 * case['seqs'] * cols * n if case['carry'] else 0)
    flops = r * cols * (7 * n + 12)
    if train:
        moved += 4 * r * cols * e + 2 * r * case['groups'] * n * e + weights + (8 * case['seqs'] * cols * n if case['carry'] else 0)
        flops += r * cols * (17 * n + 30)
    return dict(bytes=moved, flops=flops)


# -------------------------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = s['op']
    f = {}
    for k, v in s.items():
        f[k] = v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
    for k in s.get('leaves', ()):
        f[k].requires_grad_(True)
    with torch.set_grad_enabled(s['train']):
        if op in ('norm', 'norm8'):
            total = f['x'] + f['residual']
            rounded = total.detach().to(s['residual'].dtype).double()
            total = total + (rounded - total.detach())                      # the stream as it is stored; its rounding passes gradients through
            y = total / torch.sqrt(total.pow(2).sum(-1, keepdim=True) / case['cols'] + EPS) * f['gamma']
            if op == 'norm8':
                v = y.unflatten(-1, (-1, s['group'] or case['cols']))
                scale = v.abs().amax(-1).clamp_min(2.0 ** -100) / E4M3_MAX
                q = v / scale[..., None]
                ulp = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)      # e4m3: three bits behind the leading one, steps of 2^-9 at least
                return (torch.round(q / ulp) * ulp).view_as(y).to(torch.float8_e4m3fn), scale, total
            outs, seeds = [y, total], [f.get('dy'), f.get('dtotal')]
        elif op == 'conv_step':
            at = s['slots'].long()
            p = f['bias'] + f['x'] * f['w'][-1]
            for k in range(case['taps'] - 1):
                p = p + f['state'][at, k] * f['w'][k]
            f['state'][at] = torch.cat([f['state'][at, 1:], f['x'][:, None]], 1)
            return p / (1 + torch.exp(-p)), f['state']
        elif op == 'scan_step':
            at = s['slots'].long()
            h, y = _exact_step(f, f['state'][at], f['x'], f['dt'], f['B'], f['C'], f['z'], case['groups'])
            f['state'][at] = h
            return y, f['state']
        else:
            edges = s['offsets'].tolist()
            longest = max(b - a for a, b in zip(edges, edges[1:]))
            place = torch.zeros(case['seqs'], longest, dtype=torch.long, device='cuda')          # rows of the padded batch, -1 behind an utterance's end
            for i, (a, b) in enumerate(zip(edges, edges[1:])):
                place[i, :b - a] = torch.arange(a, b, device='cuda')
                place[i, b - a:] = -1
            inside = place >= 0

            def padded(k):
                return f[k][place.clamp_min(0)]

            sizes = inside.sum(1)
            if op == 'conv':
                k = case['taps']
                ahead = f['initial'] if f['initial'] is not None else torch.zeros(case['seqs'], k - 1, case['cols'], dtype=torch.float64, device='cuda')
                axis = torch.cat([ahead, padded('x')], 1)
                p = f['bias'] + sum(f['w'][j] * axis[:, j:j + longest] for j in range(k))
                y = p / (1 + torch.exp(-p))
                final = torch.stack([axis[i, n:n + k - 1] for i, n in enumerate(sizes.tolist())])
            else:
                h = f['initial'] if f['initial'] is not None else torch.zeros(case['seqs'], case['cols'], case['states'], dtype=torch.float64, device='cuda')
                xs, dts, Bs, Cs, zs = (padded(k) for k in ('x', 'dt', 'B', 'C', 'z'))
                ys = []
                for t in range(longest):
                    new, y = _exact_step(f, h, xs[:, t], dts[:, t], Bs[:, t], Cs[:, t], zs[:, t], case['groups'])
                    h = torch.where(inside[:, t, None, None], new, h)
                    ys.append(y)
                y, final = torch.stack(ys, 1), h
            y = y[inside]
            outs, seeds = [y], [f.get('dy')]
            if s['initial'] is not None:
                outs.append(final)
                seeds.append(f.get('dfinal'))
        grads = torch.autograd.grad(outs, [f[k] for k in s['leaves']], seeds) if s['train'] else ()
    return [o.detach() for o in outs], list(grads)


def _exact_step(f, h, x, dt, B, C, z, groups):
    """One frame of the recurrence for a batch of utterances: h, x, ... [utterances, ...] -> the new h, and y."""
    wide = h.shape[1] // groups
    delta = torch.logaddexp(dt + f['dt_bias'], torch.zeros_like(dt))
    h = torch.exp(delta[..., None] * f['A']) * h + (delta * x)[..., None] * B.repeat_interleave(wide, 1)
    y = (h * C.repeat_interleave(wide, 1)).sum(-1) + f['D'] * x
    return h, y * z / (1 + torch.exp(-z))
