"""The sequence operators as they are measured: layer norm, the short causal convolution and the selective state space
scan (whole sequences, their gradients, and single tokens).  `own` chooses between the framework's calls
(vqa_amd.sequence) and plain torch arithmetic in 32 bits; `exact` restates each operator in 64 bits.

Formulas (x_t is the row of token t):
  layer norm      y = (x - mean) / sqrt(var + eps) * weight + bias, over the last axis
  causal conv     y_t = silu(bias + sum_k weight[:, k] * x_{t - W + 1 + k}), rows before the first from `state`, else 0
  selective scan  dt_t = softplus(dt_t + dt_bias);  h_t = exp(dt_t a) h_{t-1} + (dt_t x_t) b_t;
                  y_t = (sum_n c_t[n] h_t[n] + skip x_t) * silu(gate_t)
  tokens at or past a sequence's length give zero rows, take no part in the state and get zero gradients."""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one question's word vectors (14 tokens, 300 wide) normalised at inference: latency
        dict(name='norm one question', op='norm', rows=14, width=300, dtype='f32', train=False),
        # the question batch of the default training step, hidden size 1024
        dict(name='norm question batch', op='norm', rows=256 * 14, width=1024, dtype='bf16', train=True),
        # long sequences at the large hidden size
        dict(name='norm long', op='norm', rows=65536, width=2048, dtype='bf16', train=True),
        # a padded batch of 30-token questions read into a cache, inner width twice the hidden size 1024
        dict(name='conv padded prompt', op='conv', batch=64, length=30, width=2048, taps=4, dtype='bf16', train=False,
             ragged=True, carry=True),
        # training on long sequences
        dict(name='conv long training', op='conv', batch=8, length=4096, width=2048, taps=4, dtype='bf16', train=True,
             ragged=False, carry=False),
        # one new token for each of 256 sequences
        dict(name='conv token x256', op='conv_token', batch=256, width=2048, taps=4, dtype='bf16'),
        # an odd shape in 32 bits: shared b / c in two groups, odd length, state carried in and out, padded
        dict(name='scan odd training', op='scan', batch=3, length=577, width=600, state=16, groups=2, dtype='f32',
             train=True, ragged=True, carry=True),
        # the question batch of the default training step
        dict(name='scan question training', op='scan', batch=256, length=14, width=2048, state=16, groups=1,
             dtype='bf16', train=True, ragged=False, carry=False),
        # training on long sequences
        dict(name='scan long training', op='scan', batch=4, length=2048, width=2048, state=16, groups=1, dtype='bf16',
             train=True, ragged=False, carry=False),
        # one long prompt read into a cache: few rows, a long axis
        dict(name='scan long prompt', op='scan', batch=1, length=16383, width=2048, state=16, groups=1, dtype='bf16',
             train=False, ragged=False, carry=True),
        # one new token of one sequence: latency
        dict(name='scan token x1', op='scan_token', batch=1, width=2048, state=16, groups=1, dtype='bf16'),
        # one new token for each of 256 sequences: the state's bytes
        dict(name='scan token x256', op='scan_token', batch=256, width=2048, state=16, groups=1, dtype='bf16'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'conv', 'scan', 'scan', 'conv_token', 'scan_token'])
    dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    if op == 'norm':
        width = _log(rng, 33, 8192)
        return dict(op=op, rows=_log(rng, 1, min(65536, 65536 * 2048 // width)), width=width, dtype=dtype,
                    train=rng.random() < 0.6)
    if op == 'conv':
        width = _log(rng, 64, 4096)
        batch = _log(rng, 1, 256)
        length = _log(rng, 1, min(16384, 8 * 4096 * 2048 // (width * batch)))
        return dict(op=op, batch=batch, length=length, width=width, taps=rng.choice([2, 3, 4]), dtype=dtype,
                    train=rng.random() < 0.6, ragged=rng.random() < 0.4, carry=rng.random() < 0.4)
    if op == 'conv_token':
        return dict(op=op, batch=_log(rng, 1, 1024), width=_log(rng, 64, 4096), taps=rng.choice([2, 3, 4]), dtype=dtype)
    groups = rng.choice([1, 1, 1, 2, 4])
    state = rng.choice([16, 16, 16, 8, 32, 64, _log(rng, 3, 64)])
    width = groups * _log(rng, 64 // groups, 4096 // groups)
    if op == 'scan_token':
        return dict(op=op, batch=_log(rng, 1, max(1, min(1024, 256 * 2048 * 16 // (width * state)))), width=width,
                    state=state, groups=groups, dtype=dtype)
    train = rng.random() < 0.6
    most = (4 * 2048 * 2048 * 16) // (width * state)
    batch = _log(rng, 1, min(256, most))
    length = _log(rng, 1, min(16384, most // batch))
    return dict(op=op, batch=batch, length=length, width=width, state=state, groups=groups, dtype=dtype, train=train,
                ragged=rng.random() < 0.4, carry=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------------------ inputs

def _inputs(case, seed, device):
    """What a user's program has in hand: activations in the case's type, parameters and states in 32 bits."""
    g = torch.Generator(device=device).manual_seed(int(seed) * 2 + 1)
    t = DTYPES[case['dtype']]
    rand = lambda *s: torch.rand(*s, device=device, generator=g)                    # noqa: E731
    randn = lambda *s: torch.randn(*s, device=device, generator=g)                  # noqa: E731
    s, op = {}, case['op']
    if op == 'norm':
        rows, width = case['rows'], case['width']
        s['x'] = (randn(rows, width) * (0.5 + rand(rows, 1)) + 0.3 * randn(rows, 1)).to(t)
        s['weight'], s['bias'] = 1 + 0.1 * randn(width), 0.1 * randn(width)
        if case['train']:
            s['dy'] = randn(rows, width).to(t)
        return s
    batch, width = case['batch'], case['width']
    if op in ('conv', 'conv_token'):
        taps = case['taps']
        s['weight'], s['bias'] = randn(width, taps) / math.sqrt(taps), 0.1 * randn(width)
        if op == 'conv_token':
            s['x'], s['state'] = randn(batch, width).to(t), randn(batch, taps - 1, width).to(t)
            return s
        s['x'] = randn(batch, case['length'], width).to(t)
        if case['carry']:
            s['state'] = randn(batch, taps - 1, width).to(t)
        if case['train']:
            s['dy'] = randn(batch, case['length'], width).to(t)
            if case['carry']:
                s['dlast'] = randn(batch, taps - 1, width).to(t)
    else:
        n, groups = case['state'], case['groups']
        lead = (batch,) if op == 'scan_token' else (batch, case['length'])
        s['x'], s['gate'] = randn(*lead, width).to(t), randn(*lead, width).to(t)
        s['dt'] = (0.5 * randn(*lead, width)).to(t)
        s['b'], s['c'] = randn(*lead, groups, n).to(t), randn(*lead, groups, n).to(t)
        s['a'] = -(torch.arange(1, n + 1, device=device).float() * (0.9 + 0.2 * rand(width, n)))
        s['skip'] = 1 + 0.1 * randn(width)
        step = torch.exp(rand(width) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))   # softplus(dt_bias)
        s['dt_bias'] = step + torch.log(-torch.expm1(-step))
        if op == 'scan_token' or case['carry']:
            s['state'] = randn(batch, width, n)
        if op == 'scan' and case['train']:
            s['dy'] = randn(*lead, width).to(t)
            if case['carry']:
                s['dlast'] = randn(batch, width, n)
    if op in ('conv', 'scan') and case['ragged']:
        s['lengths'] = torch.randint(max(0, case['length'] // 4), case['length'] + 1, (batch,), device=device,
                                     generator=g, dtype=torch.int32)
    return s


LEAVES = {'norm': ('x', 'weight', 'bias'), 'conv': ('x', 'weight', 'bias', 'state'),
          'scan': ('x', 'dt', 'a', 'b', 'c', 'skip', 'gate', 'dt_bias', 'state')}


def prepare(case, seed):
    s = _inputs(case, seed, 'cuda')
    if case.get('train'):
        for k in LEAVES[case['op']]:
            if k in s:
                s[k].requires_grad_(True)
    s['case'] = case
    return s


# -------------------------------------------------------------------------------------------------------- plain forms

def _silu(v):
    return v / (1 + torch.exp(-v))


def _dsilu(v):
    s = 1 / (1 + torch.exp(-v))
    return s * (1 + v * (1 - s))


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _live(s, length):
    """[B, L, 1]: whether a token is before its sequence's end; None where no lengths are given."""
    if 'lengths' not in s:
        return None
    return (torch.arange(length, device=s['x'].device)[None] < s['lengths'][:, None])[..., None]


def _mask(v, live):
    return v if live is None else torch.where(live, v, torch.zeros((), device=v.device))


def _norm(s):
    x = s['x'].float()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh = xc * rstd
    y = (xh * s['weight'] + s['bias']).to(s['x'].dtype)
    if 'dy' not in s:
        return {'y': y}
    dy = s['dy'].float()
    g = dy * s['weight']
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return {'y': y, 'dx': dx.to(y.dtype), 'dweight': (dy * xh).sum(0), 'dbias': dy.sum(0)}


def _last_rows(full, lengths, taps, length):
    """The taps - 1 rows before each sequence's end of [B, taps - 1 + L, D]."""
    if lengths is None:
        return full[:, length:]
    at = lengths.long()[:, None] + torch.arange(taps - 1, device=full.device)[None]
    return torch.gather(full, 1, at[..., None].expand(-1, -1, full.shape[2]))


def _conv(s):
    case, t = s['case'], s['x'].dtype
    taps, length = case['taps'], case['length']
    live = _live(s, length)
    x = _mask(s['x'].float(), live)
    before = s['state'].float() if 'state' in s else x.new_zeros(x.shape[0], taps - 1, x.shape[2])
    full = torch.cat([before, x], 1)
    w = s['weight']
    pre = s['bias'].expand_as(x)
    for k in range(taps):
        pre = pre + w[:, k] * full[:, k:k + length]
    out = {'y': _mask(_silu(pre), live).to(t)}
    if 'state' in s:
        out['last'] = _last_rows(full, s.get('lengths'), taps, length).to(t)
    if 'dy' not in s:
        return out
    g = _mask(s['dy'].float() * _dsilu(pre), live)
    dfull = torch.zeros_like(full)
    dw = []
    for k in range(taps):
        dfull[:, k:k + length] += w[:, k] * g
        dw.append((g * full[:, k:k + length]).sum((0, 1)))
    if 'dlast' in s:
        if 'lengths' in s:
            at = s['lengths'].long()[:, None] + torch.arange(taps - 1, device=x.device)[None]
            dfull.scatter_add_(1, at[..., None].expand(-1, -1, x.shape[2]), s['dlast'].float())
        else:
            dfull[:, length:] += s['dlast'].float()
    out |= {'dx': _mask(dfull[:, taps - 1:], live).to(t), 'dweight': torch.stack(dw, 1), 'dbias': g.sum((0, 1))}
    if 'state' in s:
        out['dstate'] = dfull[:, :taps - 1].to(t)
    return out


def _conv_token(s):
    full = torch.cat([s['state'], s['x'][:, None]], 1)
    pre = s['bias'] + (full.float() * s['weight'].t()).sum(1)
    s['state'].copy_(full[:, 1:])
    return {'y': _silu(pre).to(s['x'].dtype), 'state': s['state']}


def _running(decay, add):
    """h_t = decay_t h_{t-1} + add_t along axis 1, h before the first row 0, by doubling."""
    k, length = 1, add.shape[1]
    while k < length:
        add = torch.cat([add[:, :k], add[:, k:] + decay[:, k:] * add[:, :-k]], 1)
        decay = torch.cat([decay[:, :k], decay[:, k:] * decay[:, :-k]], 1)
        k *= 2
    return add


def _per_channel(v, width):
    """[..., G, N] -> [..., D, N]: each channel's group's row."""
    return v.float().repeat_interleave(width // v.shape[-2], -2)


def _scan(s):
    case, t = s['case'], s['x'].dtype
    width, length, groups = case['width'], case['length'], case['groups']
    live = _live(s, length)
    x, gate, a = _mask(s['x'].float(), live), s['gate'].float(), s['a']
    raw = s['dt'].float() + s['dt_bias']
    dt = _mask(_softplus(raw), live)
    b = _per_channel(s['b'], width)
    c = _per_channel(s['c'], width)
    decay = torch.exp(dt[..., None] * a)
    add = (dt * x)[..., None] * b
    if 'state' in s:
        add = torch.cat([add[:, :1] + decay[:, :1] * s['state'][:, None], add[:, 1:]], 1)
    h = _running(decay, add)
    del add
    core = (h * c).sum(-1) + s['skip'] * x
    out = {'y': _mask(core * _silu(gate), live).to(t)}
    if 'state' in s:
        out['last'] = h[:, -1].clone()
    if 'dy' not in s:
        return out
    dy = _mask(s['dy'].float(), live)
    dcore = dy * _silu(gate)
    dgate = dy * core * _dsilu(gate)
    dh = dcore[..., None] * c
    if 'dlast' in s:
        dh[:, -1] += s['dlast']
    # the adjoint runs the other way: G_t = dh_t + decay_{t+1} G_{t+1}
    later = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], 1).flip(1)
    G = _running(later, dh.flip(1)).flip(1)
    del later, dh
    before = torch.cat([s['state'][:, None] if 'state' in s else torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    through = G * before * decay
    del before
    dgroup = lambda v: v.reshape(*v.shape[:2], groups, width // groups, -1).sum(3)   # noqa: E731
    gb = (G * b).sum(-1)
    draw_ = _mask(((through * a).sum(-1) + x * gb) * (1 / (1 + torch.exp(-raw))), live)
    out |= {'dx': _mask(dt * gb + s['skip'] * dcore, live).to(t), 'ddt': draw_.to(t),
            'da': (through * dt[..., None]).sum((0, 1)), 'dskip': (dcore * x).sum((0, 1)),
            'ddt_bias': draw_.sum((0, 1)), 'dgate': _mask(dgate, live).to(t)}
    del through
    out['db'] = _mask(dgroup(G * (dt * x)[..., None]).flatten(2), live).unflatten(2, (groups, -1)).to(t)
    out['dc'] = _mask(dgroup(h * dcore[..., None]).flatten(2), live).unflatten(2, (groups, -1)).to(t)
    if 'state' in s:
        out['dstate'] = G[:, 0] * decay[:, 0]
    return out


def _scan_token(s):
    width = s['case']['width']
    x = s['x'].float()
    dt = _softplus(s['dt'].float() + s['dt_bias'])
    h = torch.exp(dt[..., None] * s['a']) * s['state'] + (dt * x)[..., None] * _per_channel(s['b'], width)
    s['state'].copy_(h)
    y = (h * _per_channel(s['c'], width)).sum(-1) + s['skip'] * x
    return {'y': (y * _silu(s['gate'].float())).to(s['x'].dtype), 'state': s['state']}


PLAIN = {'norm': _norm, 'conv': _conv, 'conv_token': _conv_token, 'scan': _scan, 'scan_token': _scan_token}


# ------------------------------------------------------------------------------------------------------------- a pass

def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return PLAIN[s['case']['op']](s)


def _own(s):
    from vqa_amd import sequence as S
    case = s['case']
    op = case['op']
    if op == 'conv_token':
        return {'y': S.causal_conv_step(s['x'], s['state'], s['weight'], s['bias']), 'state': s['state']}
    if op == 'scan_token':
        y = S.selective_scan_step(s['x'], s['state'], s['dt'], s['a'], s['b'], s['c'], s['skip'], s['gate'],
                                  s['dt_bias'])
        return {'y': y, 'state': s['state']}
    if op == 'norm':
        out = {'y': S.layer_norm(s['x'], s['weight'], s['bias'])}
    else:
        if op == 'conv':
            r = S.causal_conv(s['x'], s['weight'], s['bias'], state=s.get('state'), lengths=s.get('lengths'),
                              return_state=case['carry'])
        else:
            r = S.selective_scan(s['x'], s['dt'], s['a'], s['b'], s['c'], s['skip'], s['gate'], s['dt_bias'],
                                 state=s.get('state'), lengths=s.get('lengths'), return_state=case['carry'])
        out = {'y': r[0], 'last': r[1]} if case['carry'] else {'y': r}
    if 'dy' in s:
        names = [k for k in LEAVES[op] if k in s]
        ends = [(out['y'], s['dy'])] + ([(out['last'], s['dlast'])] if 'dlast' in s else [])
        grads = torch.autograd.grad([e for e, _ in ends], [s[k] for k in names], [g for _, g in ends])
        out = {k: v.detach() for k, v in out.items()}
        out |= {'d' + k: v for k, v in zip(names, grads)}
    return out


# ------------------------------------------------------------------------------------------------- bytes and operations

def work(case):
    e, op = 2 if case['dtype'] != 'f32' else 4, case['op']
    if op == 'norm':
        n = case['rows'] * case['width']
        if not case['train']:
            return {'bytes': 2 * n * e + 8 * case['width'], 'flops': 8 * n}
        return {'bytes': 4 * n * e + 16 * case['width'], 'flops': 22 * n}       # x, dy in; y, dx out
    batch, width = case['batch'], case['width']
    if op in ('conv', 'conv_token'):
        taps = case['taps']
        params = 4 * width * (taps + 1)
        rows = 2 * batch * (taps - 1) * width * e                               # the state in and out
        if op == 'conv_token':
            return {'bytes': 2 * batch * width * e + rows + params, 'flops': batch * width * (2 * taps + 6)}
        n = batch * case['length'] * width
        rows = rows if case['carry'] else 0
        if not case['train']:
            return {'bytes': 2 * n * e + rows + params, 'flops': n * (2 * taps + 6)}
        return {'bytes': 4 * n * e + 2 * rows + 2 * params, 'flops': n * (8 * taps + 18)}
    n, groups = case['state'], case['groups']
    params = 4 * width * (n + 2)
    states = 2 * batch * width * n * 4
    tokens = batch * (1 if op == 'scan_token' else case['length'])
    rows = tokens * width * e
    shared = 2 * tokens * groups * n * e
    if op == 'scan_token':
        return {'bytes': 4 * rows + shared + states + params, 'flops': tokens * width * (7 * n + 20)}
    states = states if case['carry'] else 0
    if not case['train']:
        return {'bytes': 4 * rows + shared + states + params, 'flops': tokens * width * (7 * n + 20)}
    # x, dt, gate, dy in; y and the three gradients out; b, c and theirs
    return {'bytes': 8 * rows + 2 * shared + 2 * states + 2 * params, 'flops': tokens * width * (24 * n + 50)}


# ---------------------------------------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    """The operators token by token in 64 bits; the gradients by differentiating that."""
    s = {k: v.double() if v.is_floating_point() else v for k, v in _inputs(case, seed, 'cuda').items()}
    op = case['op']
    names = [k for k in LEAVES.get(op, ()) if k in s] if case.get('train') else []
    for k in names:
        s[k] = s[k].requires_grad_(True)
    F = torch.nn.functional
    if op == 'norm':
        out = {'y': F.layer_norm(s['x'], (case['width'],), s['weight'], s['bias'], 1e-5)}
    elif op == 'conv_token':
        window = torch.cat([s['state'], s['x'].unsqueeze(1)], 1)
        out = {'y': F.silu(torch.einsum('bkd,dk->bd', window, s['weight']) + s['bias']), 'state': window[:, 1:]}
    elif op == 'scan_token':
        y, h = _exact_token(s, s['x'], s['dt'], s['b'], s['c'], s['gate'], s['state'])
        out = {'y': y, 'state': h}
    elif op == 'conv':
        out = _exact_conv(case, s)
    else:
        out = _exact_scan(case, s)
    if names:
        ends = [out['y']] + ([out['last']] if 'dlast' in s else [])
        grads = torch.autograd.grad(ends, [s[k] for k in names], [s['dy']] + ([s['dlast']] if 'dlast' in s else []))
        out |= {'d' + k: v for k, v in zip(names, grads)}
    return {k: v.detach() for k, v in out.items()}


def _exact_conv(case, s):
    taps, length, width = case['taps'], case['length'], case['width']
    start = s['state'] if 'state' in s else s['x'].new_zeros(case['batch'], taps - 1, width)
    rows = torch.cat([start, s['x']], 1)
    y = torch.nn.functional.conv1d(rows.transpose(1, 2), s['weight'].unsqueeze(1), s['bias'], groups=width)
    y = torch.nn.functional.silu(y).transpose(1, 2)
    if 'lengths' in s:
        y = y * (torch.arange(length, device=y.device) < s['lengths'][:, None])[..., None]
    out = {'y': y}
    if case['carry']:
        ends = s['lengths'].tolist() if 'lengths' in s else [length] * case['batch']
        out['last'] = torch.stack([rows[i, e:e + taps - 1] for i, e in enumerate(ends)])
    return out


def _exact_token(s, x, dt, b, c, gate, h, on=None):
    share = x.shape[-1] // b.shape[-2]                              # channels of one group
    step = torch.nn.functional.softplus(dt + s['dt_bias'], threshold=1e9)
    new = torch.exp(step.unsqueeze(-1) * s['a']) * h + (step * x).unsqueeze(-1) * b.repeat_interleave(share, -2)
    y = (new * c.repeat_interleave(share, -2)).sum(-1) + s['skip'] * x
    y = y * torch.nn.functional.silu(gate)
    if on is None:
        return y, new
    return torch.where(on[:, None], y, torch.zeros_like(y)), torch.where(on[:, None, None], new, h)


def _exact_scan(case, s):
    h = s['state'] if 'state' in s else s['x'].new_zeros(case['batch'], case['width'], case['state'])
    rows = [s[k].unbind(1) for k in ('x', 'dt', 'b', 'c', 'gate')]
    ys = []
    for t in range(case['length']):
        on = s['lengths'] > t if 'lengths' in s else None
        y, h = _exact_token(s, *(r[t] for r in rows), h, on)
        ys.append(y)
    return {'y': torch.stack(ys, 1)} | ({'last': h} if case['carry'] else {})
