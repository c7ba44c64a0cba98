"""GPU: the sequence operators (vqa_amd.sequence) against the same formulas token by token in 64 bits: outputs, gradients,
padded batches, carried states, single tokens, strides, types, streams, graphs, refusals.

Roundings counted in a tolerance (sequence_ref.close): layer norm and the convolution chain a few operations per value plus
their sums' partial chains (rows / 16 rows side by side); a scan's state takes 3 roundings a token and its decay's error is
that of dt (about 16: softplus by exponential, reciprocal and a series of 7 terms) times dt a e^{dt a} <= 1/e."""
# (softplus now takes a polynomial of degree 4 in place of the series: fewer roundings than the 16 that are counted)
import pytest
import torch

from tests import sequence_ref as R

pytestmark = pytest.mark.gpu

DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def S():
    from vqa_amd import sequence
    return sequence


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _leaf(t, dtype=torch.float32):
    """(GPU leaf in dtype, CPU float64 leaf of the same values)"""
    if t is None:
        return None, None
    t = t.to(dtype)
    return t.cuda().requires_grad_(True), t.double().requires_grad_(True)


def _grads(outs, seeds, leaves):
    names = [k for k, v in leaves.items() if v is not None]
    got = torch.autograd.grad([o for o in outs if o is not None], [leaves[k] for k in names],
                              [s for o, s in zip(outs, seeds) if o is not None])
    return dict(zip(names, got))


# ---------------------------------------------------------------------------------------------------------- layer norm

@pytest.mark.parametrize('rows,width,dtype', [
    (1, 1, 'f32'), (3, 2, 'bf16'), (14, 300, 'f32'), (5, 300, 'bf16'), (7, 513, 'f16'), (65, 1024, 'bf16'),
    (130, 64, 'f32'), (9, 1025, 'bf16'), (33, 2048, 'bf16'), (12, 2047, 'f32'), (6, 4096, 'f16'), (5, 4095, 'bf16'),
    (4, 8192, 'f32'), (3, 8191, 'bf16'), (2100, 40, 'bf16')])
def test_layer_norm(rows, width, dtype):
    g = _gen(rows * 10007 + width)
    x, xr = _leaf(torch.randn(rows, width, generator=g) * 2 + 0.5, DT[dtype])
    w, wr = _leaf(1 + 0.1 * torch.randn(width, generator=g))
    b, br = _leaf(0.1 * torch.randn(width, generator=g))
    dy = torch.randn(rows, width, generator=g).to(DT[dtype])
    y, yr = S().layer_norm(x, w, b), R.norm(xr, wr, br)
    assert y.dtype == x.dtype
    if width == 1:
        # a row of one value: x - mean is 0, rstd is 1 / sqrt(eps) = 316 and no gradient reaches x
        R.close('y', y, yr, 16)
        (dx,) = torch.autograd.grad(y, [x], dy.cuda())
        assert not dx.any()
        return
    R.close('y', y, yr, 32)
    got = _grads([y], [dy.cuda()], dict(x=x, w=w, b=b))
    want = _grads([yr], [dy.double()], dict(x=xr, w=wr, b=br))
    # dx = rstd (g - mean(g) - xh mean(g xh)), g = dy w: each of the three terms is at most rstd max|g| sqrt(width) and
    # rounded a few times, while their sum may cancel altogether (two values a row: xh = +-1, the sum is 0 but for eps),
    # so dx's rounding is counted at the terms' size.  max|xh| <= sqrt(width); mean(g xh) <= max|g|.
    rstd = float(1 / torch.sqrt(xr.detach().var(-1, unbiased=False) + 1e-5).max())
    xd = xr.detach()
    terms = rstd * float((dy.double() * wr.detach()).abs().max()) * float(
        ((xd - xd.mean(-1, keepdim=True)).abs().amax(-1) / xd.std(-1, unbiased=False)).max())
    R.close('dx', got['x'], want['x'], 64, scale=terms)
    R.close('dw', got['w'], want['w'], 64 + rows)
    R.close('db', got['b'], want['b'], 64 + rows)


@pytest.mark.parametrize('weight,bias', [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters_and_in_three_axes(weight, bias):
    g = _gen(3)
    x, xr = _leaf(torch.randn(4, 5, 72, generator=g), torch.bfloat16)
    w, wr = _leaf(torch.randn(72, generator=g)) if weight else (None, None)
    b, br = _leaf(torch.randn(72, generator=g)) if bias else (None, None)
    dy = torch.randn(4, 5, 72, generator=g).bfloat16()
    y, yr = S().layer_norm(x, w, b, eps=1e-3), R.norm(xr, wr, br, 1e-3)
    R.close('y', y, yr, 32)
    got, want = _grads([y], [dy.cuda()], dict(x=x, w=w, b=b)), _grads([yr], [dy.double()], dict(x=xr, w=wr, b=br))
    for k in got:
        R.close(k, got[k], want[k], 128)


@pytest.mark.parametrize('width,dtype', [(48, 'bf16'), (47, 'f32'), (2048, 'bf16')])
def test_layer_norm_of_strided_rows(width, dtype):
    """Rows of a wider matrix (aligned and not), every other row, a transposed matrix, a broadcast row, a broadcast dy."""
    g = _gen(5)
    base = torch.randn(10, 2 * width + 8, generator=g).to(DT[dtype])
    w = torch.randn(width, generator=g)
    dev = base.cuda()
    for name, f in {'aligned': lambda m: m[:, 8:8 + width], 'odd': lambda m: m[:, 3:3 + width],
                    'alternate': lambda m: m[::2, :width], 'transposed': lambda m: m[:, :10].t()[:, :7],
                    'broadcast': lambda m: m[:1, :width].expand(6, width)}.items():
        x, xr = f(dev), f(base).double()
        ww = w[:x.shape[1]]
        y = S().layer_norm(x, ww.cuda(), None)
        R.close(name, y, R.norm(xr, ww.double(), None), 32)
        assert y.is_contiguous()
    x, xr = _leaf(base[:, :width], DT[dtype])
    y, yr = S().layer_norm(x), R.norm(xr, None, None)
    y.sum().backward()                                       # dy with strides 0
    # xhat sums to 0 over a row, so the exact gradient of the sum is 0: what is left is rounding of terms of size rstd
    assert float(x.grad.abs().max()) <= 64 * 2.0 ** -24 * float(1 / xr.detach().std(1, unbiased=False).min())


def test_layer_norm_extremes():
    """A constant row (variance 0), a row far from 0, rows with NaN and infinity: each row by itself."""
    g = _gen(6)
    x = torch.randn(6, 384, generator=g)
    x[0] = 3.25
    x[1] += 4096
    x[2, 5] = float('nan')
    x[3, 7] = float('inf')
    y = S().layer_norm(x.cuda()).cpu()
    assert not y[0].any()
    # the mean of values near 4096 is off by a few of its half steps, 2^-12 each; y has the scale 1
    assert float((y[1].double() - R.norm(x[1:2].double(), None, None)[0]).abs().max()) <= 8 * 2.0 ** -12
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    R.close('rest', y[4:], R.norm(x[4:].double(), None, None), 32)
    w = torch.ones(384, device='cuda', requires_grad=True)
    assert S().layer_norm(torch.empty(0, 384, device='cuda'), w).shape == (0, 384)
    S().layer_norm(torch.empty(0, 384, device='cuda'), w).sum().backward()
    assert not w.grad.any()


# --------------------------------------------------------------------------------------------------- causal convolution

def _conv_case(B, T, D, taps, dtype, act, lengths, carry, seed=0, bias=True):
    g = _gen(seed + B * 1000 + T * 10 + D)
    t = DT[dtype]
    raw = torch.randn(B, T, D, generator=g)
    w = torch.randn(D, taps, generator=g) / taps ** 0.5
    lens = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    dy, dlast = torch.randn(B, T, D, generator=g).to(t), torch.randn(B, taps - 1, D, generator=g).to(t)
    leaves = dict(x=_leaf(raw, t), w=_leaf(w), b=_leaf(0.2 * torch.randn(D, generator=g)) if bias else (None, None),
                  state=_leaf(torch.randn(B, taps - 1, D, generator=g), t) if carry else (None, None))
    return leaves, lens, dy, dlast


@pytest.mark.parametrize('B,T,D,taps,dtype,act,lengths,carry', [
    (1, 1, 1, 4, 'f32', 'silu', None, False), (2, 1, 8, 3, 'bf16', 'silu', None, True),
    (3, 2, 7, 4, 'f32', None, None, True), (4, 14, 64, 4, 'bf16', 'silu', [14, 0, 1, 9], True),
    (2, 33, 300, 2, 'f16', 'silu', [2, 33], False), (3, 65, 96, 3, 'bf16', None, [64, 3, 70], True),
    (1, 200, 2048, 4, 'bf16', 'silu', None, True), (5, 71, 515, 4, 'f32', 'silu', [71, 70, -3, 2, 3], True),
    (70, 9, 24, 4, 'bf16', 'silu', None, False)])
def test_causal_conv(B, T, D, taps, dtype, act, lengths, carry):
    leaves, lens, dy, dlast = _conv_case(B, T, D, taps, dtype, act, lengths, carry)
    (x, xr), (w, wr), (b, br), (st, sr) = (leaves[k] for k in ('x', 'w', 'b', 'state'))
    dlen = lens.cuda() if lens is not None else None
    y, last = S().causal_conv(x, w, b, act, state=st, lengths=dlen, return_state=True)
    yr, lastr = R.conv(xr, wr, br, act, sr, lens)
    R.close('y', y, yr, 32)
    assert torch.equal(last.detach().cpu().double(), lastr.detach())          # copies of rows
    got = _grads([y, last], [dy.cuda(), dlast.cuda()], dict(x=x, w=w, b=b, state=st))
    want = _grads([yr, lastr], [dy.double(), dlast.double()], dict(x=xr, w=wr, b=br, state=sr))
    for k in got:
        R.close('d' + k, got[k], want[k], 64 if k in ('x', 'state') else 64 + B * T)
    if lens is not None:                                     # padding may hold anything, in x and in dy
        bad, bady = x.detach().clone(), dy.cuda()
        for i, n in enumerate(lengths):
            bad[i, max(0, n):], bady[i, max(0, n):] = float('nan'), float('inf')
        bad.requires_grad_(True)
        y2, last2 = S().causal_conv(bad, w, b, act, state=st, lengths=dlen, return_state=True)
        assert torch.equal(y2, y) and torch.equal(last2, last)
        again = _grads([y2, last2], [bady, dlast.cuda()], dict(x=bad, w=w, b=b, state=st))
        for k in again:
            assert torch.equal(again[k], got[k]), k


def test_causal_conv_parts_of_outputs():
    """Only y, only the state, no bias; a state that nothing needs."""
    leaves, _, dy, dlast = _conv_case(2, 6, 16, 4, 'f32', 'silu', None, True, bias=False)
    (x, xr), (w, wr), (st, sr) = (leaves[k] for k in ('x', 'w', 'state'))
    y = S().causal_conv(x, w, state=st)
    yr, lastr = R.conv(xr, wr, None, 'silu', sr, None)
    got, want = (_grads([o], [d], l) for o, d, l in ((y, dy.cuda(), dict(x=x, w=w, s=st)),
                                                     (yr, dy.double(), dict(x=xr, w=wr, s=sr))))
    for k in got:
        R.close(k, got[k], want[k], 128)
    _, last = S().causal_conv(x, w, state=st, return_state=True)
    gx, gw = torch.autograd.grad(last, [x, w], dlast.cuda())
    assert torch.equal(gx[:, 3:], dlast.cuda()) and not gx[:, :3].any() and not gw.any()
    y0, last0 = S().causal_conv(x[:, :0], w, state=st, return_state=True)
    assert y0.shape == (2, 0, 16) and torch.equal(last0, st)
    assert torch.autograd.grad(last0, st, dlast.cuda())[0].equal(dlast.cuda())


@pytest.mark.parametrize('dtype,D', [('bf16', 64), ('f32', 33)])
def test_causal_conv_strided_and_broadcast(dtype, D):
    """x as half of a projection's output, time-major x, one sequence broadcast over the batch (gradient summed)."""
    g = _gen(11)
    t = DT[dtype]
    w = torch.randn(D, 4, generator=g)
    wide = torch.randn(3, 10, 2 * D, generator=g).to(t)
    for f in (lambda m: m[..., :D], lambda m: m[..., D:], lambda m: m[..., 1:D + 1], lambda m: m.transpose(0, 1)[..., :D],
              lambda m: m[:, ::2, :D], lambda m: m[..., ::2]):
        x = f(wide.cuda())
        y = S().causal_conv(x, w.cuda())
        R.close('y', y, R.conv(f(wide).double(), w.double(), None, 'silu', None, None)[0], 32)
    one, oner = _leaf(wide[:1, :, :D], t)
    dy = torch.randn(4, 10, D, generator=g).to(t)
    (gx,) = torch.autograd.grad(S().causal_conv(one.expand(4, -1, -1), w.cuda()), one, dy.cuda())
    (want,) = torch.autograd.grad(R.conv(oner.expand(4, -1, -1), w.double(), None, 'silu', None, None)[0], oner, dy.double())
    # four rounded rows are summed by autograd in x's type: 4 half steps of the terms, 3 of the partial sums
    tol = 8 * torch.finfo(t).eps * float(want.abs().max())
    assert float((gx.cpu().double() - want).abs().max()) <= tol


@pytest.mark.parametrize('B,D,taps,dtype', [(1, 1, 2, 'f32'), (3, 64, 4, 'bf16'), (5, 301, 3, 'f16'), (300, 24, 4, 'bf16')])
def test_causal_conv_steps_continue_a_sequence(B, D, taps, dtype):
    """A padded prompt, then tokens one at a time = the whole sequence at once, bit for bit (one order of sums)."""
    g = _gen(12)
    t = DT[dtype]
    w, b = torch.randn(D, taps, generator=g).cuda(), torch.randn(D, generator=g).cuda()
    x = torch.randn(B, 9, D, generator=g).to(t).cuda()
    n = torch.randint(0, 6, (B,), generator=g, dtype=torch.int32)
    whole = S().causal_conv(x, w, b)
    _, state = S().causal_conv(x[:, :5], w, b, lengths=n.cuda(), return_state=True)
    pool = torch.full((B, taps - 1, 2 * D), 7.0, device='cuda', dtype=t)        # a state kept as part of something wider
    pool[..., :D] = state
    for k in range(3):
        at = (n.long() + k).cuda().clamp(max=8)
        tok = x[torch.arange(B, device='cuda'), at]
        y = S().causal_conv_step(tok, state, w, b)
        assert torch.equal(S().causal_conv_step(tok, pool[..., :D], w, b), y)
        assert torch.equal(y, whole[torch.arange(B, device='cuda'), at])
    assert torch.equal(pool[..., :D], state) and (pool[..., D:] == 7).all()


# ------------------------------------------------------------------------------------------------- selective state space

SCAN = ('x', 'dt', 'a', 'b', 'c', 'skip', 'gate', 'dt_bias', 'state')


def _scan_case(B, T, D, N, G, dtype, seed=0, carry=True, without=()):
    g = _gen(seed + B * 1000 + T * 10 + D + N)
    t = DT[dtype]
    rn = lambda *s: torch.randn(*s, generator=g)                                # noqa: E731
    v = dict(x=rn(B, T, D), dt=0.5 * rn(B, T, D), a=-(0.2 + 4 * torch.rand(D, N, generator=g)), b=rn(B, T, G, N),
             c=rn(B, T, G, N), skip=rn(D), gate=rn(B, T, D), dt_bias=rn(D) - 2, state=rn(B, D, N) if carry else None)
    leaves = {k: (None, None) if v[k] is None or k in without else
              _leaf(v[k], torch.float32 if k in ('a', 'skip', 'dt_bias', 'state') else t) for k in SCAN}
    return leaves, rn(B, T, D).to(t), rn(B, D, N)


def _scan_check(leaves, dy, dlast, lens, softplus=True):
    B, T, D = dy.shape
    G = {k: v[0] for k, v in leaves.items()}
    C = {k: v[1] for k, v in leaves.items()}
    dlen = lens.cuda() if lens is not None else None
    y, last = S().selective_scan(*(G[k] for k in SCAN[:8]), softplus=softplus, state=G['state'], lengths=dlen,
                                 return_state=True)
    yr, lastr = R.scan(*(C[k] for k in SCAN[:8]), softplus, C['state'], lens)
    n = 128 + 8 * T
    R.close('y', y, yr, n)
    R.close('last', last, lastr, n)
    got = _grads([y, last], [dy.cuda(), dlast.cuda()], G)
    want = _grads([yr, lastr], [dy.double(), dlast.double()], C)
    for k in got:
        # db, dc sum over the channels of a group; parameter gradients over all tokens
        R.close('d' + k, got[k], want[k], 2 * n + {'b': D, 'c': D}.get(k, B * T if k in ('a', 'skip', 'dt_bias') else 0))
    return G, y, last, got


@pytest.mark.parametrize('B,T,D,N,G,dtype,lengths', [
    (1, 1, 1, 1, 1, 'f32', None), (2, 3, 5, 3, 1, 'bf16', None), (1, 7, 64, 16, 1, 'bf16', None),
    (2, 8, 65, 16, 1, 'f32', None), (3, 9, 128, 16, 2, 'bf16', [9, 0, 5]), (2, 17, 48, 8, 1, 'f16', [1, 17]),
    (2, 14, 33, 17, 1, 'f32', None), (1, 23, 64, 32, 2, 'bf16', None), (2, 19, 40, 64, 1, 'bf16', [18, 30]),
    (2, 12, 36, 33, 4, 'f32', [-1, 12]), (9, 5, 16, 16, 1, 'f32', None)])
def test_selective_scan(B, T, D, N, G, dtype, lengths):
    lens = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    leaves, dy, dlast = _scan_case(B, T, D, N, G, dtype)
    ins, y, last, got = _scan_check(leaves, dy, dlast, lens)
    if lens is not None:                                     # padding may hold anything
        bad, bady = {k: v.detach().clone() for k, v in ins.items()}, dy.cuda()
        for i, n in enumerate(lengths):
            for j, k in enumerate(('x', 'dt', 'b', 'c', 'gate')):
                bad[k][i, max(0, n):] = (float('nan'), float('inf'), float('-inf'))[j % 3]
            bady[i, max(0, n):] = float('nan')
        bad = {k: v.requires_grad_(True) for k, v in bad.items()}
        y2, last2 = S().selective_scan(*(bad[k] for k in SCAN[:8]), state=bad['state'], lengths=lens.cuda(),
                                       return_state=True)
        assert torch.equal(y2, y) and torch.equal(last2, last)
        again = _grads([y2, last2], [bady, dlast.cuda()], bad)
        for k in again:
            assert torch.equal(again[k], got[k]), k


@pytest.mark.parametrize('B,T,D,N,G,dtype,lengths', [
    (1, 600, 32, 16, 1, 'f32', None), (2, 333, 72, 16, 1, 'bf16', [200, 333]), (1, 257, 24, 40, 2, 'f32', [256]),
    (2, 130, 17, 20, 1, 'bf16', [0, 64]),
    (1, 200, 70, 8, 1, 'bf16', None), (2, 150, 34, 5, 2, 'f32', [149, 3])])
def test_selective_scan_in_segments(B, T, D, N, G, dtype, lengths):
    """Few rows and a long axis: the tokens are cut into segments that are joined again."""
    lens = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    leaves, dy, dlast = _scan_case(B, T, D, N, G, dtype, seed=1)
    _scan_check(leaves, dy, dlast, lens)


@pytest.mark.parametrize('without,softplus,carry', [(('gate',), True, False), (('skip', 'dt_bias'), True, True),
                                                    (('gate', 'skip', 'dt_bias'), False, False)])
def test_selective_scan_options(without, softplus, carry):
    leaves, dy, dlast = _scan_case(2, 21, 40, 16, 1, 'f32', seed=2, carry=carry, without=without)
    if not softplus:                                         # dt as it is: positive, so that the states stay bounded
        dt = 0.1 * torch.rand(2, 21, 40, generator=_gen(9))
        leaves['dt'] = _leaf(dt)
    _scan_check(leaves, dy, dlast, None, softplus)


@pytest.mark.parametrize('N', [16, 8, 20])
def test_selective_scan_many_sequences_in_one_wave(N):
    """More batch rows than waves are wanted for: a wave takes several, its parameter sums run on; and fewer, where a wave
    takes half the channels: the same bits."""
    B, T, D = 300, 3, 1024
    leaves, dy, _ = _scan_case(B, T, D, N, 1, 'f32', seed=3, carry=False)
    G = {k: v[0] for k, v in leaves.items()}
    y = S().selective_scan(*(G[k] for k in SCAN[:8]))
    got = _grads([y], [dy.cuda()], G)
    half = {k: 0 for k in ('a', 'skip', 'dt_bias')}
    for lo in range(0, B, 100):                              # the same sums, from three calls that take one row a wave
        part = {k: (v.detach()[lo:lo + 100] if k in ('x', 'dt', 'b', 'c', 'gate') else v.detach()).requires_grad_(True)
                for k, v in G.items() if v is not None}
        p = S().selective_scan(*(part[k] for k in SCAN[:8]))
        assert torch.equal(p, y[lo:lo + 100])
        gp = _grads([p], [dy.cuda()[lo:lo + 100]], part)
        for k in ('x', 'dt', 'b', 'c', 'gate'):
            assert torch.equal(gp[k], got[k][lo:lo + 100]), k
        for k in half:
            half[k] = half[k] + gp[k].double()
    for k in half:
        R.close(k, got[k], half[k].cpu(), 2 * B * T)


@pytest.mark.parametrize('dtype,D', [('bf16', 64), ('f32', 20)])
def test_selective_scan_strided_and_shared(dtype, D):
    """Rows as slices of projections' outputs, b and c as one slice [B, L, N] each, one sequence's b broadcast."""
    g = _gen(14)
    t, N = DT[dtype], 16
    rn = lambda *s: torch.randn(*s, generator=g)                                # noqa: E731
    proj, small = rn(3, 11, 3 * D).to(t), rn(3, 11, 5 + 2 * N).to(t)
    a, bias = -(0.2 + 3 * torch.rand(D, N, generator=g)), rn(D) - 2
    args = lambda p, s: (p[..., :D], p[..., D:2 * D], s[..., 5:5 + N], s[..., 5 + N:], p[..., 2 * D:])  # noqa: E731
    x, dt, b, c, gate = args(proj.cuda(), small.cuda())
    y = S().selective_scan(x, dt, a.cuda(), b, c, None, gate, bias.cuda())
    x, dt, b, c, gate = args(proj.double(), small.double())
    yr, _ = R.scan(x, dt, a.double(), b[:, :, None], c[:, :, None], None, gate, bias.double(), True, None, None)
    R.close('y', y, yr, 256)
    p, s = proj.cuda(), small.cuda().requires_grad_(True)
    x, dt, b, c, gate = args(p, s)
    tm = [v.transpose(0, 1).contiguous().transpose(0, 1) for v in (x, dt, gate)]          # time-major rows
    y2 = S().selective_scan(tm[0], tm[1], a.cuda(), b, c, None, tm[2], bias.cuda())
    assert torch.equal(y2, y)
    one = b[:1].detach().requires_grad_(True)
    cc = c.detach()
    (gb,) = torch.autograd.grad(S().selective_scan(x, dt, a.cuda(), one.expand(3, -1, -1), cc, None, gate, bias.cuda()),
                                one, torch.ones_like(y))
    full = one.expand(3, -1, -1).detach().clone().requires_grad_(True)
    (gf,) = torch.autograd.grad(S().selective_scan(x, dt, a.cuda(), full, cc, None, gate, bias.cuda()), full,
                                torch.ones_like(y))
    assert float((gb.double() - gf.double().sum(0, keepdim=True)).abs().max()) <= 4 * torch.finfo(t).eps * float(
        gf.double().abs().sum(0).max())


def test_softplus_over_its_range():
    """dt alone: one token from the zero state with x = b = c = 1, so y = dt = softplus(raw), relative to its own value over
    the whole range of an f32 exponential (a chain of some 16 roundings)."""
    raw = torch.cat([torch.linspace(-80, 40, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 88.0, 200.0])])
    D = raw.numel()
    x, one = torch.ones(1, 1, D, device='cuda'), torch.ones(1, 1, 1, device='cuda')
    y = S().selective_scan(x, raw.cuda().view(1, 1, D), -torch.ones(D, 1, device='cuda'), one, one)
    want = torch.nn.functional.softplus(raw.double(), threshold=1e9)
    # exp(-|raw|) is off by raw's rounding times log2 e: |raw| 2^-24 relative on the small side
    tol = (16 + raw.double().abs().clamp(max=80) * 2) * 2.0 ** -24 * want
    assert ((y.cpu().view(-1).double() - want).abs() <= tol).all()


def test_selective_scan_of_nothing():
    leaves, _, dlast = _scan_case(2, 3, 16, 16, 1, 'f32')
    G = {k: v[0] for k, v in leaves.items()}
    cut = {k: v[:, :0] if k in ('x', 'dt', 'b', 'c', 'gate') else v for k, v in G.items()}
    y, last = S().selective_scan(*(cut[k] for k in SCAN[:8]), state=G['state'], return_state=True)
    assert y.shape == (2, 0, 16) and torch.equal(last, G['state'])
    gs, ga = torch.autograd.grad(last, [G['state'], G['a']], dlast.cuda())
    assert torch.equal(gs, dlast.cuda()) and not ga.any()


@pytest.mark.parametrize('B,D,N,G,dtype', [(1, 1, 1, 1, 'f32'), (3, 64, 16, 1, 'bf16'), (2, 40, 5, 2, 'f32'),
                                           (4, 48, 8, 1, 'f16'), (2, 24, 33, 1, 'bf16'), (3, 32, 64, 4, 'f32')])
def test_selective_scan_steps_continue_a_sequence(B, D, N, G, dtype):
    """A padded prompt, then tokens one at a time, against the whole sequences in 64 bits; the state in a wider pool."""
    T, steps = 6, 3
    leaves, _, _ = _scan_case(B, T + steps, D, N, G, dtype, seed=4, carry=False)
    g = {k: v[0].detach() if v[0] is not None else None for k, v in leaves.items()}
    n = torch.randint(0, T + 1, (B,), generator=_gen(5), dtype=torch.int32)
    _, state = S().selective_scan(*(g[k][:, :T] if k in ('x', 'dt', 'b', 'c', 'gate') else g[k] for k in SCAN[:8]),
                                  lengths=n.cuda(), return_state=True)
    pool = torch.full((B, 2, D, N), 5.0, device='cuda')
    pool[:, 1] = state
    rows = torch.arange(B, device='cuda')
    yr, hr = R.scan(*(leaves[k][1] for k in SCAN[:8]), True, None, n + steps)
    for k in range(steps):
        at = n.long().cuda() + k
        tok = {q: g[q][rows, at] for q in ('x', 'dt', 'b', 'c', 'gate')}
        args = (tok['dt'], g['a'], tok['b'], tok['c'], g['skip'], tok['gate'], g['dt_bias'])
        y = S().selective_scan_step(tok['x'], state, *args)
        assert torch.equal(S().selective_scan_step(tok['x'], pool[:, 1], *args), y)
        R.close('y', y, yr[torch.arange(B), n.long() + k], 128 + 8 * (T + steps))
    R.close('state', state, hr, 128 + 8 * (T + steps))
    assert torch.equal(pool[:, 1], state) and (pool[:, 0] == 5).all()


# ------------------------------------------------------------------------------------------------------------- together

def _block(P, x, lengths=None, states=None, keep=False):
    """One token-mixing block: norm, projection, convolution, projections of dt / b / c, scan, projection."""
    s = S()
    D, N = P['a'].shape
    h = s.layer_norm(x, P['nw'], P['nb'])
    xz = h @ P['win']
    u = s.causal_conv(xz[..., :D], P['wc'], P['bc'], state=states and states[0], lengths=lengths, return_state=True)
    dbc = u[0] @ P['wx']
    y = s.selective_scan(u[0], dbc[..., :D], P['a'], dbc[..., D:D + N], dbc[..., D + N:], P['skip'], xz[..., D:],
                         P['dtb'], state=states and states[1], lengths=lengths, return_state=True)
    out = x + y[0] @ P['wout']
    return (out, (u[1], y[1])) if keep else out


def _block_ref(P, x, lengths):
    D, N = P['a'].shape
    xz = R.norm(x, P['nw'], P['nb']) @ P['win']
    u, _ = R.conv(xz[..., :D], P['wc'], P['bc'], 'silu', None, lengths)
    dbc = u @ P['wx']
    y, _ = R.scan(u, dbc[..., :D], P['a'], dbc[..., None, D:D + N], dbc[..., None, D + N:], P['skip'], xz[..., D:],
                  P['dtb'], True, None, lengths)
    return x + y @ P['wout']


def _block_params(C, D, N):
    g = _gen(21)
    rn = lambda *s: torch.randn(*s, generator=g)                                # noqa: E731
    p = dict(nw=1 + 0.1 * rn(C), nb=0.1 * rn(C), win=rn(C, 2 * D) / C ** 0.5, wc=rn(D, 4) / 2, bc=0.1 * rn(D),
             wx=rn(D, D + 2 * N) / D ** 0.5, a=-(0.2 + 3 * torch.rand(D, N, generator=g)), skip=rn(D), dtb=rn(D) - 2,
             wout=rn(D, C) / D ** 0.5)
    return {k: v.cuda().requires_grad_(True) for k, v in p.items()}, {k: v.double().requires_grad_(True) for k, v in p.items()}


def test_block_trains():
    """All operators in one float32 block over a padded batch: the loss's gradient for every parameter and the input."""
    P, Pr = _block_params(24, 48, 16)
    x, xr = _leaf(torch.randn(3, 14, 24, generator=_gen(22)))
    lens = torch.tensor([14, 5, 9], dtype=torch.int32)
    out, ref = _block(P, x, lens.cuda()), _block_ref(Pr, xr, lens)
    dy = torch.randn(3, 14, 24, generator=_gen(23))
    # the chain of all operators: the scan's 128 + 8 T, the products' sums of at most 96 terms, amplified by each other
    R.close('out', out, ref, 2048)
    got, want = _grads([out], [dy.cuda()], dict(P, x=x)), _grads([ref], [dy.double()], dict(Pr, x=xr))
    for k in got:
        R.close('d' + k, got[k], want[k], 8192)


def test_block_reads_a_padded_prompt_and_then_single_tokens():
    P, Pr = _block_params(16, 32, 16)
    s = S()
    x = torch.randn(3, 9, 16, generator=_gen(24))
    n = torch.tensor([4, 1, 6], dtype=torch.int32)
    with torch.no_grad():
        _, (cs, hs) = _block(P, x[:, :6].cuda(), n.cuda(), keep=True)
        ref = _block_ref(Pr, x.double(), None)
        D, N = P['a'].shape
        for k in range(3):
            at = n.long() + k
            tok = x[torch.arange(3), at].cuda()
            xz = s.layer_norm(tok, P['nw'], P['nb']) @ P['win']
            u = s.causal_conv_step(xz[:, :D], cs, P['wc'], P['bc'])
            dbc = u @ P['wx']
            y = s.selective_scan_step(u, hs, dbc[:, :D], P['a'], dbc[:, D:D + N], dbc[:, D + N:], P['skip'], xz[:, D:],
                                      P['dtb'])
            R.close('token', tok + y @ P['wout'], ref[torch.arange(3), at], 2048)


def test_gradients_against_differences():
    """d/de of <out, dy> along a random direction, from the kernels' own forward at +-e (float32, so e = 2^-6: the
    difference is off by e^2 of a third derivative of the order of the value and by 2^-24 / e)."""
    P, _ = _block_params(16, 32, 16)
    x = torch.randn(2, 20, 16, generator=_gen(31)).cuda().requires_grad_(True)
    dy = torch.randn(2, 20, 16, generator=_gen(32)).cuda()
    leaves = dict(P, x=x)
    grads = _grads([_block(P, x)], [dy], leaves)
    g = _gen(33)
    for k, v in leaves.items():
        way = torch.randn(v.shape, generator=g).cuda()
        way = way / way.norm()
        vals = []
        with torch.no_grad():
            for e in (2.0 ** -6, -2.0 ** -6):
                Q = {q: w.detach() + (e * way if q == k else 0) for q, w in leaves.items()}
                vals.append((_block(Q, Q['x']).double() * dy.double()).sum())
        slope = float((vals[0] - vals[1]) * 32)
        want = float((grads[k].double() * way.double()).sum())
        assert abs(slope - want) <= 2e-3 * max(float(grads[k].double().norm()), 1e-3), k


# ---------------------------------------------------------------------------------------------- streams, graphs, devices

def test_same_bits_every_time_and_on_another_stream():
    P, _ = _block_params(64, 128, 16)
    x = torch.randn(4, 130, 64, generator=_gen(41)).cuda().requires_grad_(True)
    lens = torch.tensor([130, 64, 1, 100], dtype=torch.int32, device='cuda')
    dy = torch.randn(4, 130, 64, generator=_gen(42)).cuda()

    def once():
        out = _block(P, x, lens)
        return [out.detach()] + list(_grads([out], [dy], dict(P, x=x)).values())
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(first, second):
        assert torch.equal(u, v)


def test_two_streams_at_once():
    """Two calls in flight on two streams (states and workspaces of their own), several times over."""
    sets = []
    for k in (1, 2):
        leaves, dy, _ = _scan_case(2, 300, 96, 16, 1, 'bf16', seed=70 + k)
        ins = {q: v[0].detach() for q, v in leaves.items()}
        sets.append((ins, S().selective_scan(*(ins[q] for q in SCAN[:8]), state=ins['state'], return_state=True)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                ins = sets[i][0]
                outs[i].append(S().selective_scan(*(ins[q] for q in SCAN[:8]), state=ins['state'], return_state=True))
    torch.cuda.synchronize()
    for i in (0, 1):
        for y, last in outs[i]:
            assert torch.equal(y, sets[i][1][0]) and torch.equal(last, sets[i][1][1])


def test_strides_past_32_bits():
    """Sequences 2^31 and more elements apart, rows 2^26 apart: the same as contiguous copies of them."""
    s = S()
    far = (1 << 31) + 24
    buf = torch.zeros(far + 8192, device='cuda', dtype=torch.bfloat16)
    x = buf.as_strided((2, 20, 64), (far, 64, 1), 16)
    x.copy_(torch.randn(2, 20, 64, generator=_gen(80)))
    near = x.contiguous()
    w = torch.randn(64, 4, generator=_gen(81)).cuda()
    assert torch.equal(s.layer_norm(x[:, 3]), s.layer_norm(near[:, 3]))
    assert torch.equal(s.causal_conv(x, w), s.causal_conv(near, w))
    a, b = -torch.rand(64, 8, device='cuda'), torch.randn(2, 20, 8, generator=_gen(82)).cuda().bfloat16()
    assert torch.equal(s.selective_scan(x, x, a, b, b, gate=x), s.selective_scan(near, near, a, b, b, gate=near))
    cs = buf.as_strided((2, 3, 64), (far, 64, 1), 4096)
    cs.copy_(near[:, :3])
    c2 = cs.contiguous()
    assert torch.equal(s.causal_conv_step(x[:, 4], cs, w), s.causal_conv_step(near[:, 4], c2, w)) and torch.equal(cs, c2)
    hbuf = buf.view(torch.float32)
    h = hbuf.as_strided((2, 64, 8), ((1 << 30) + 8, 8, 1), 64)
    h2 = h.contiguous()
    assert torch.equal(s.selective_scan_step(x[:, 4], h, x[:, 5], a, b[:, 0], b[:, 1]),
                       s.selective_scan_step(near[:, 4], h2, near[:, 5], a, b[:, 0], b[:, 1])) and torch.equal(h, h2)
    rows = buf.as_strided((1, 9, 64), (64, 1 << 26, 1), 8)
    assert torch.equal(s.selective_scan(rows, rows, a, b[:1, :9], b[:1, :9]),
                       s.selective_scan(rows.contiguous(), rows.contiguous(), a, b[:1, :9], b[:1, :9]))


def test_captured_graphs_replay():
    """Forward and backward captured (two graphs of different sizes, replayed in turn with eager work between), every
    replay against the eager result on the inputs of that replay."""
    s = S()

    def make(B, T, D, N):
        leaves, dy, _ = _scan_case(B, T, D, N, 1, 'bf16', seed=B)
        ins = {k: v[0] for k, v in leaves.items()}
        w = torch.randn(D, 4, generator=_gen(1)).cuda().requires_grad_(True)
        nw = torch.randn(D, generator=_gen(2)).cuda().requires_grad_(True)

        def step(ins, w, nw, dy):
            u = s.causal_conv(s.layer_norm(ins['x'], nw), w)
            y, last = s.selective_scan(u, *(ins[k] for k in SCAN[1:8]), state=ins['state'], return_state=True)
            return [y, last] + list(torch.autograd.grad(y, [*ins.values(), w, nw], dy))
        return ins, w, nw, dy.cuda(), step

    graphs = []
    for shape in ((2, 9, 64, 16), (1, 200, 40, 16)):
        ins, w, nw, dy, step = make(*shape)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(ins, w, nw, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(ins, w, nw, dy)
        graphs.append((graph, ins, w, nw, dy, step, outs))
    for k in range(3):
        for graph, ins, w, nw, dy, step, outs in graphs:
            with torch.no_grad():
                ins['x'].copy_(torch.randn(ins['x'].shape, generator=_gen(50 + k)))
                dy.copy_(torch.randn(dy.shape, generator=_gen(60 + k)))
            graph.replay()
            fresh = {q: v.detach().clone().requires_grad_(True) for q, v in ins.items()}
            want = step(fresh, w.detach().clone().requires_grad_(True), nw.detach().clone().requires_grad_(True), dy)
            torch.cuda.synchronize()
            for u, v in zip(outs, want):
                assert torch.equal(u, v)


def test_captured_steps_replay():
    """Serving: one token's two steps captured, the states living outside the graph."""
    s = S()
    B, D, N = 4, 64, 16
    leaves, _, _ = _scan_case(B, 8, D, N, 1, 'bf16', seed=7, carry=False)
    g = {k: v[0].detach() if v[0] is not None else None for k, v in leaves.items()}
    w = torch.randn(D, 4, generator=_gen(3)).cuda()
    tok = {k: torch.zeros_like(g[k][:, 0]) for k in ('x', 'dt', 'b', 'c', 'gate')}
    cs, hs = torch.zeros(B, 3, D, device='cuda', dtype=torch.bfloat16), torch.zeros(B, D, N, device='cuda')

    def step():
        u = s.causal_conv_step(tok['x'], cs, w)
        return s.selective_scan_step(u, hs, tok['dt'], g['a'], tok['b'], tok['c'], g['skip'], tok['gate'], g['dt_bias'])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    cs.zero_(), hs.zero_()
    want = s.selective_scan(s.causal_conv(g['x'], w), *(g[k] for k in SCAN[1:8]))
    for k in range(8):
        for q in tok:
            tok[q].copy_(g[q][:, k])
        graph.replay()
        torch.cuda.synchronize()
        R.close('y', out, want[:, k].double().cpu(), 256 + 2.0 ** 17)           # (both sides are rounded to bf16)


def test_versions_and_second_derivatives():
    s = S()
    x = torch.randn(2, 8, device='cuda')
    state = torch.zeros(2, 3, 8, device='cuda')
    w = torch.randn(8, 4, device='cuda', requires_grad=True)
    y = s.causal_conv(x[:, None], w, state=state)
    with torch.no_grad():
        s.causal_conv_step(x, state, w)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    z = torch.randn(3, 8, device='cuda', requires_grad=True)
    (g,) = torch.autograd.grad(s.layer_norm(z).square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        g.sum().backward()


def test_inference_mode():
    s = S()
    with torch.inference_mode():
        x = torch.randn(2, 5, 16, device='cuda')
        w = torch.randn(16, 4, device='cuda')
        y, state = s.causal_conv(x[:, :4], w, return_state=True)
        assert torch.equal(s.causal_conv_step(x[:, 4], state, w), s.causal_conv(x, w)[:, 4])
        a, b = -torch.rand(16, 8, device='cuda'), torch.randn(2, 5, 8, device='cuda')
        y, h = s.selective_scan(x[:, :4], x[:, :4], a, b[:, :4], b[:, :4], return_state=True)
        z = s.selective_scan_step(x[:, 4], h, x[:, 4], a, b[:, 4], b[:, 4])
        assert z.shape == (2, 16) and s.layer_norm(x).shape == x.shape


def test_one_row_at_any_stride():
    """A sequence of one token whose row stride says nothing: torch calls it contiguous at any stride."""
    s = S()
    buf = torch.randn(2, 64, generator=_gen(90)).cuda().bfloat16()
    far = lambda t: t.as_strided((2, 1, t.shape[1]), (t.shape[1], 1 << 40, 1))       # noqa: E731
    near = lambda t: t.clone().view(2, 1, -1)      # noqa: E731
    w, a, g = torch.randn(64, 4, generator=_gen(91)).cuda(), -torch.rand(64, 8, device='cuda'), buf[:, :8].contiguous()
    got, want = [], []
    for view, out in ((far, got), (near, want)):
        x = buf.clone().requires_grad_(True)
        b = g.clone().requires_grad_(True)
        u = view(x) if view is far else x.view(2, 1, 64)
        v = view(b) if view is far else b.view(2, 1, 8)
        y = s.selective_scan(u, u, a, v, v, gate=u)
        out += [y, s.causal_conv(u, w), s.layer_norm(u)]
        dy = view(torch.ones(2, 64, device='cuda', dtype=torch.bfloat16))
        out += torch.autograd.grad(y, [x, b], dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_layer_norm_of_more_rows_than_a_launch_takes():
    """Rows past 2^22 and (one wave a row) past 2^32 threads: each as it is by itself."""
    s = S()
    rows = (1 << 26) + 5
    x = torch.empty(rows, 2, device='cuda', dtype=torch.bfloat16).normal_(generator=torch.Generator('cuda').manual_seed(92))
    w, b = torch.tensor([0.5, -2.0], device='cuda'), torch.tensor([0.25, 1.0], device='cuda')
    y = s.layer_norm(x, w, b)
    for r in (0, (1 << 22) - 3, 5 * (1 << 22) - 7, rows - 9):
        assert torch.equal(y[r:r + 9], s.layer_norm(x[r:r + 9].clone(), w, b))
    x = x[:(1 << 22) + 7].clone().requires_grad_(True)
    dy = torch.ones_like(x)
    dy[:, 1] = 0.5
    dx, = torch.autograd.grad(s.layer_norm(x, w, b), x, dy)
    part = x.detach()[-20:].clone().requires_grad_(True)
    want, = torch.autograd.grad(s.layer_norm(part, w, b), part, dy[-20:].clone())
    assert torch.equal(dx[-20:], want)


def test_selective_scan_gradients_of_many_shared_rows():
    """More values of db and dc than one pass of the grid that joins them: sequences as they are in halves of the batch
    (neither is cut into segments)."""
    s = S()
    B, T, D, N = 2048, 72, 2, 64
    x = torch.randn(B, T, D, generator=_gen(93)).cuda()
    a = -torch.rand(D, N, generator=_gen(94)).cuda()
    b, c = (torch.randn(B, T, N, generator=_gen(95 + i)).cuda() for i in range(2))
    lens = torch.randint(0, T + 1, (B,), generator=_gen(97), dtype=torch.int32).cuda()

    def grads(lo, hi):
        bb, cc = b[lo:hi].clone().requires_grad_(True), c[lo:hi].clone().requires_grad_(True)
        y = s.selective_scan(x[lo:hi], x[lo:hi], a, bb, cc, lengths=lens[lo:hi])
        return torch.autograd.grad(y, [bb, cc], torch.ones_like(y))
    whole, first, second = grads(0, B), grads(0, B // 2), grads(B // 2, B)
    for t in range(2):
        assert torch.equal(whole[t][:B // 2], first[t]) and torch.equal(whole[t][B // 2:], second[t])


def test_refusals():
    s = S()
    from vqa_amd._lib import VqaHipError
    x = torch.zeros(2, 4, 8, device='cuda')
    w = torch.zeros(8, 4, device='cuda')
    state = torch.zeros(2, 3, 8, device='cuda')
    a = -torch.ones(8, 16, device='cuda')
    b = torch.zeros(2, 4, 16, device='cuda')
    h = torch.zeros(2, 8, 16, device='cuda')
    lens = torch.tensor([4, 2], dtype=torch.int32, device='cuda')
    bad = [
        lambda: s.layer_norm(x.cpu()), lambda: s.layer_norm(x.double()), lambda: s.layer_norm(x, torch.ones(7, device='cuda')),
        lambda: s.layer_norm(x, torch.ones(8, device='cuda').bfloat16()), lambda: s.layer_norm(x, torch.ones(8)),
        lambda: s.layer_norm(torch.zeros(2, 8193, device='cuda')), lambda: s.layer_norm(torch.zeros((), device='cuda')),
        lambda: s.causal_conv(x[0], w), lambda: s.causal_conv(x, w[:, :1]), lambda: s.causal_conv(x, w[:7]),
        lambda: s.causal_conv(x, torch.zeros(8, 5, device='cuda')), lambda: s.causal_conv(x, w, activation='relu'),
        lambda: s.causal_conv(x, w, state=state[:, :2]), lambda: s.causal_conv(x, w, state=state.bfloat16()),
        lambda: s.causal_conv(x, w, lengths=lens.long()), lambda: s.causal_conv(x, w, lengths=lens.cpu()),
        lambda: s.causal_conv(x, w, lengths=lens[:1]),
        lambda: s.causal_conv_step(x, state, w), lambda: s.causal_conv_step(x[:, 0], state[:1].expand(2, 3, 8), w),
        lambda: s.causal_conv_step(x[:, 0], state[:, :1].expand(2, 3, 8), w),
        lambda: s.causal_conv_step(x[:, 0], state.transpose(1, 2).contiguous().transpose(1, 2), w),
        lambda: s.causal_conv_step(x[:, 0], state, w.clone().requires_grad_(True)),
        lambda: s.selective_scan(x, x[:, :3], a, b, b), lambda: s.selective_scan(x, x.bfloat16(), a, b, b),
        lambda: s.selective_scan(x, x, a[:, :8], b, b), lambda: s.selective_scan(x, x, a.bfloat16(), b, b),
        lambda: s.selective_scan(x, x, a, b, b[..., :8]), lambda: s.selective_scan(x, x, a, b[:1], b[:1]),
        lambda: s.selective_scan(x, x, a, b[:, :, None].expand(2, 4, 3, 16), b[:, :, None].expand(2, 4, 3, 16)),
        lambda: s.selective_scan(x, x, torch.zeros(8, 65, device='cuda'), *(torch.zeros(2, 4, 65, device='cuda'),) * 2),
        lambda: s.selective_scan(x, x, a, b, b, gate=x[..., :4]), lambda: s.selective_scan(x, x, a, b, b, state=h[:1]),
        lambda: s.selective_scan(x, x, a, b, b, lengths=lens.float()),
        lambda: s.selective_scan_step(x[:, 0], h[:1].expand(2, 8, 16), x[:, 0], a, b[:, 0], b[:, 0]),
        lambda: s.selective_scan_step(x[:, 0], h.transpose(1, 2).contiguous().transpose(1, 2), x[:, 0], a, b[:, 0], b[:, 0]),
        lambda: s.selective_scan_step(x[:, 0], h.bfloat16(), x[:, 0], a, b[:, 0], b[:, 0]),
        lambda: s.selective_scan_step(x[:, 0], h, x[:, 0], a.clone().requires_grad_(True), b[:, 0], b[:, 0]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(VqaHipError):
            f()
            pytest.fail(f'call {i} was not refused')


def test_selective_scan_without_channels():
    s = S()
    b, c = (torch.randn(2, 3, 4, device='cuda', requires_grad=True) for _ in range(2))
    x, a, h = torch.zeros(2, 3, 0, device='cuda'), torch.zeros(0, 4, device='cuda'), torch.zeros(2, 0, 4, device='cuda')
    y, last = s.selective_scan(x, x, a, b, c, state=h, return_state=True)
    assert y.shape == (2, 3, 0) and last.shape == (2, 0, 4)
    junk = [torch.full((2, 3, 1, 4), float('nan'), device='cuda') for _ in range(8)]
    del junk
    db, dc = torch.autograd.grad(y, [b, c], torch.zeros_like(y))
    assert not db.any() and not dc.any()


def test_tangents_and_recorders_are_refused():
    """Nothing that follows or records operators one by one gets an answer that it could not see."""
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    from vqa_amd._lib import VqaHipError
    s = S()
    x, w, wc = (torch.randn(*n, device='cuda') for n in ((2, 4, 8), (8,), (8, 4)))
    a, b, h, cs = -torch.ones(8, 4, device='cuda'), torch.randn(2, 4, 4, device='cuda'), torch.zeros(2, 8, 4, device='cuda'), \
        torch.zeros(2, 3, 8, device='cuda')
    calls = [lambda x: s.layer_norm(x, w), lambda x: s.causal_conv(x, wc), lambda x: s.selective_scan(x, x, a, b, b),
             lambda x: s.causal_conv_step(x[:, 0], cs, wc), lambda x: s.selective_scan_step(x[:, 0], h, x[:, 0], a, b[:, 0], b[:, 1])]
    for f in calls:
        want = f(x)
        with fw.dual_level():
            with pytest.raises(VqaHipError, match='tangent'):
                f(fw.make_dual(x, torch.ones_like(x)))
        with pytest.raises(VqaHipError, match='recorded'):
            torch.jit.trace(f, (x,))
        with pytest.raises(VqaHipError, match='recorded'):
            make_fx(f)(x)
        cs.zero_(), h.zero_()
        with fw.dual_level():
            assert torch.equal(f(x), want)                 # (no tangent among the inputs)
        cs.zero_(), h.zero_()
    for f in calls[:3]:
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x[None])
    z = x.clone().requires_grad_(True)
    y = s.layer_norm(z)
    with fw.dual_level():
        with pytest.raises(VqaHipError, match='tangent'):
            torch.autograd.grad(y, z, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_compiled_callers(backend):
    """torch.compile around a caller: the same bits, values and gradients."""
    s = S()
    x, w, wc = (torch.randn(*n, device='cuda') for n in ((2, 4, 8), (8,), (8, 4)))
    a, b, h, cs = -torch.ones(8, 4, device='cuda'), torch.randn(2, 4, 4, device='cuda'), torch.zeros(2, 8, 4, device='cuda'), \
        torch.zeros(2, 3, 8, device='cuda')
    calls = [lambda x: 2 * s.layer_norm(x, w), lambda x: 2 * s.causal_conv(x, wc), lambda x: 2 * s.selective_scan(x, x, a, b, b),
             lambda x: 2 * s.causal_conv_step(x[:, 0], cs, wc),
             lambda x: 2 * s.selective_scan_step(x[:, 0], h, x[:, 0], a, b[:, 0], b[:, 1])]
    for i, f in enumerate(calls):
        outs = []
        for g in (f, torch.compile(f, backend=backend)):
            cs.zero_(), h.zero_()
            outs.append([g(x), cs.clone(), h.clone()])
            if i < 3:
                leaf = x.clone().requires_grad_(True)
                outs[-1] += torch.autograd.grad(g(leaf), leaf, x)
        torch._dynamo.reset()
        for p, q in zip(*outs):
            assert torch.equal(p, q), i


def test_scalar_arguments():
    """Numbers and truth values of numpy as Python's; an eps in a tensor is refused, not taken by its address."""
    import numpy as np
    from vqa_amd._lib import VqaHipError
    s = S()
    x, w = torch.randn(3, 8, device='cuda'), torch.ones(8, device='cuda')
    with pytest.raises(VqaHipError, match='eps'):
        s.layer_norm(x, w, eps=torch.tensor(1e-5, device='cuda'))
    assert torch.equal(s.layer_norm(x, w, eps=np.float32(0.5)), s.layer_norm(x, w, eps=0.5))
    assert torch.equal(s.layer_norm(x, w, eps=1), s.layer_norm(x, w, eps=1.0))
    a, b = -torch.ones(8, 4, device='cuda'), torch.randn(3, 4, device='cuda')
    for flag in (True, False):
        h = [torch.ones(3, 8, 4, device='cuda') for _ in range(2)]
        assert torch.equal(s.selective_scan_step(x, h[0], x, a, b, b, softplus=np.bool_(flag)),
                           s.selective_scan_step(x, h[1], x, a, b, b, softplus=flag)) and torch.equal(*h)


def test_axes_past_31_bits_are_refused():
    """(one value, expanded: no memory behind it)"""
    from vqa_amd._lib import VqaHipError
    s, far = S(), (1 << 32) + 1
    one = torch.ones(1, device='cuda', dtype=torch.bfloat16)
    w, a = torch.ones(1, 4, device='cuda'), -torch.ones(1, 1, device='cuda')
    for shape in ((far, 1, 1), (1, far, 1)):
        x = one.expand(shape)
        for f in (lambda: s.layer_norm(x), lambda: s.causal_conv(x, w), lambda: s.selective_scan(x, x, a, x, x)):
            with pytest.raises(VqaHipError):
                f()
    x = one.expand(far, 1)
    h = torch.zeros(1, 1, 1, device='cuda')
    for f in (lambda: s.causal_conv_step(x, one.expand(far, 3, 1), w),
              lambda: s.selective_scan_step(x, h.expand(far, 1, 1), x, a, x, x)):
        with pytest.raises(VqaHipError):
            f()


def _same_kind(name, got, want, roundings):
    """Where the definition (64 bits) gives a number, got is near it; where it gives an infinity, that infinity; where it
    gives no number, anything."""
    g, w = got.detach().double().cpu(), want.detach()
    inf = w.isinf()
    assert torch.equal(g[inf], w[inf]), f'{name}: {g[inf][:8]} for {w[inf][:8]}'
    ok = w.isfinite()
    assert ok.any(), name
    R.close(name, got.detach().cpu()[ok], w[ok], roundings)


@pytest.mark.parametrize('B,T,D,N,dtype', [(2, 19, 40, 5, 'f32'), (2, 19, 40, 16, 'f32'), (1, 21, 65, 12, 'bf16'),
                                           (2, 300, 40, 20, 'f32'), (1, 300, 72, 33, 'f32'), (1, 2100, 8, 3, 'f32'),
                                           (70, 17, 2048, 12, 'bf16')])
def test_selective_scan_of_infinite_values(B, T, D, N, dtype):
    """One infinite x, where the states' terms have one sign: an infinite state and y from there on, and nothing else; one
    infinite dy: an infinite gradient of what came before."""
    leaves, dy, dlast = _scan_case(B, T, D, N, 1, dtype, seed=40)
    at, ch, late = (0, T // 3, 3), 5, 2 * T // 3
    for k in ('x', 'b', 'c', 'skip', 'state'):
        for v in leaves[k]:
            v.data.abs_().clamp_(min=0.125)
    dy, dlast = dy.abs() + 0.125, dlast.abs() + 0.125
    n = 128 + 8 * T
    if B == 70:                                            # (many sequences: the first is compared)
        leaves = {k: (g, c[:1] if k in ('x', 'dt', 'b', 'c', 'gate', 'state') else c) for k, (g, c) in leaves.items()}
    G, C = ({k: v[i].detach().clone() for k, v in leaves.items()} for i in (0, 1))

    def go(x_inf, dy_inf):
        outs = []
        for v, f, d, dl in ((G, None, dy.cuda(), dlast.cuda()), (C, R.scan, dy.double(), dlast.double())):
            v = {k: t.clone() for k, t in v.items()}
            d = d[:len(v['x'])].clone()
            if x_inf:
                v['x'][at] = float('inf')
            if dy_inf:
                d[0, late, ch] = float('inf')
                v['gate'][0, late, ch] = 1.0
            v = {k: t.requires_grad_(True) for k, t in v.items()}
            if f is None:
                y, last = S().selective_scan(*(v[k] for k in SCAN[:8]), state=v['state'], return_state=True)
            else:
                y, last = R.scan(*(v[k] for k in SCAN[:8]), True, v['state'], None)
            outs.append((y, last, _grads([y, last], [d, dl[:len(d)]], v)))
        return outs
    (y, last, _), (yr, lastr, _) = go(True, False)
    assert yr[0, T // 3:, 3].isinf().all() and lastr[0, 3].isinf().all()
    _same_kind('y', y[:len(yr)], yr, n)
    _same_kind('last', last[:len(yr)], lastr, n)
    (_, _, g), (_, _, w) = go(False, True)
    assert w['x'][0, :late + 1, ch].isinf().all()
    for k in ('x', 'dt', 'gate', 'state', 'b'):
        _same_kind('d' + k, g[k][:len(yr)], w[k], 2 * n + (D if k == 'b' else 0))
    if B < 70:
        _same_kind('da', g['a'], w['a'], 2 * n + B * T)


@pytest.mark.parametrize('N', [3, 5, 12, 16, 33])
def test_selective_scan_step_of_infinite_values(N):
    g = _gen(41)
    B, D = 2, 24
    rn = lambda *s: torch.rand(*s, generator=g) + 0.125                          # noqa: E731
    x, dt, gate, b, c, h, a, skip = rn(B, D), rn(B, D), rn(B, D), rn(B, 1, N), rn(B, 1, N), rn(B, D, N), -rn(D, N), rn(D)
    x[1, 7], dt[0, 2] = float('inf'), float('inf')
    state = h.cuda()
    y = S().selective_scan_step(*(v.cuda() if v is not state else v for v in (x, state, dt, a, b, c, skip, gate)))
    yr, hr = R.scan(*(v.double()[:, None] for v in (x, dt)), a.double(), b.double()[:, None], c.double()[:, None],
                    skip.double(), gate.double()[:, None], None, True, h.double(), None)
    assert yr[1, 0, 7].isinf() and yr[0, 0, 2].isinf()
    _same_kind('y', y, yr[:, 0], 256)
    _same_kind('state', state, hr, 256)


@pytest.mark.parametrize('N', [16, 5])
def test_selective_scan_infinite_states_pass_segments(N):
    """A segment's decay underflows to 0 where no token's does: an infinite state, and an infinite adjoint, pass it as they
    pass its tokens, and finite ones are forgotten."""
    g = _gen(42)
    B, T, D = 1, 400, 24
    rn = lambda *s: torch.rand(*s, generator=g) + 0.125                          # noqa: E731
    v = dict(x=rn(B, T, D), dt=rn(B, T, D), a=-10 * rn(D, N), b=rn(B, T, 1, N), c=rn(B, T, 1, N), skip=rn(D))
    v['x'][0, 20, 3] = float('inf')
    dy = rn(B, T, D)
    dy[0, 390, 5] = float('inf')
    dev = {k: t.cuda().requires_grad_(True) for k, t in v.items()}
    ref = {k: t.double().requires_grad_(True) for k, t in v.items()}
    y, last = S().selective_scan(*(dev[k] for k in SCAN[:6]), return_state=True)
    yr, lastr = R.scan(*(ref[k] for k in SCAN[:6]), None, None, True, None, None)
    assert yr[0, 20:, 3].isinf().all() and lastr[0, 3].isinf().all()
    _same_kind('y', y, yr, 128 + 8 * T)
    _same_kind('last', last, lastr, 128 + 8 * T)
    (dx,), (dxr,) = torch.autograd.grad(y, [dev['x']], dy.cuda()), torch.autograd.grad(yr, [ref['x']], dy.double())
    assert dxr[0, :391, 5].isinf().all()
    _same_kind('dx', dx, dxr, 2 * (128 + 8 * T))


@pytest.mark.parametrize('N,D', [(16, 64), (5, 33)])
def test_absent_parameters_meet_no_infinity(N, D):
    """skip=None is no skip, not a skip of 0: an infinite x or dy keeps its sign."""
    g = _gen(43)
    B, T = 2, 19
    rn = lambda *s: torch.rand(*s, generator=g) + 0.125                          # noqa: E731
    v = dict(x=rn(B, T, D), dt=rn(B, T, D), a=-rn(D, N), b=rn(B, T, 1, N), c=rn(B, T, 1, N), gate=rn(B, T, D))
    dy = rn(B, T, D)
    dy[1, 9, 2], v['gate'][1, 9, 2] = float('inf'), 1.0
    dev = {k: t.cuda().requires_grad_(True) for k, t in v.items()}
    ref = {k: t.double().requires_grad_(True) for k, t in v.items()}
    y, _ = S().selective_scan(*(dev[k] for k in SCAN[:5]), gate=dev['gate'], return_state=True)
    yr, _ = R.scan(*(ref[k] for k in SCAN[:5]), None, ref['gate'], None, True, None, None)
    got, want = _grads([y], [dy.cuda()], dev), _grads([yr], [dy.double()], ref)
    assert want['x'][1, :10, 2].isinf().all()
    for k in ('x', 'gate', 'dt'):
        _same_kind('d' + k, got[k], want[k], 2 * (128 + 8 * T))
    x = v['x'].clone()
    x[0, 4, 1] = float('inf')
    args = {k: v[k] for k in SCAN[1:5]}
    y = S().selective_scan(x.cuda(), *(t.cuda() for t in args.values()), gate=v['gate'].cuda())
    yr, _ = R.scan(x.double(), *(t.double() for t in args.values()), None, v['gate'].double(), None, True, None, None)
    assert yr[0, 4:, 1].isinf().all()
    _same_kind('y', y, yr, 128 + 8 * T)
    h = torch.zeros(B, D, N, device='cuda')
    one = S().selective_scan_step(x[:, 4].cuda(), h, *(args[k][:, 4].cuda() if k != 'a' else args[k].cuda() for k in args),
                                  gate=v['gate'][:, 4].cuda())
    yr, _ = R.scan(*(t.double()[:, 4:5] if k != 'a' else t.double() for k, t in dict(x=x, **args).items()), None,
                   v['gate'].double()[:, 4:5], None, True, None, None)
    _same_kind('step', one, yr[:, 0], 256)


@pytest.mark.parametrize('B,T,D,N,lengths', [(2, 5, 24, 16, None), (3, 19, 40, 5, [19, 3, 0]), (2, 300, 24, 16, [300, 17]),
                                             (1, 8, 16, 8, None)])
def test_selective_scan_of_states_that_are_forgotten(B, T, D, N, lengths):
    """a = -inf: every token forgets such a state; tokens that a sequence does not have leave it.  Against a = -1e30, where
    64 bits have the products that 0 times -inf has not."""
    lens = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    leaves, dy, dlast = _scan_case(B, T, D, N, 1, 'f32', seed=44)
    leaves['a'][0].data[:, 1], leaves['a'][1].data[:, 1] = float('-inf'), -1e30
    _scan_check(leaves, dy, dlast, lens)


@pytest.mark.parametrize('width,dtype', [(3, 'f32'), (47, 'f32'), (300, 'bf16'), (512, 'f16'), (1051, 'bf16'), (1600, 'f32'),
                                         (2048, 'bf16'), (5000, 'f16'), (8191, 'bf16')])
def test_layer_norm_of_infinite_gradients(width, dtype):
    """One infinite dy, in the first and in the last column: dx by the formula in 64 bits, and no other row touched."""
    g = _gen(45)
    x = torch.randn(5, width, generator=g).to(DT[dtype])
    w = torch.rand(width, generator=g) + 0.5
    dy = torch.randn(5, width, generator=g).to(DT[dtype])
    dy[1, -1] = dy[3, 0] = float('inf')
    leaf = x.cuda().requires_grad_(True)
    dx, = torch.autograd.grad(S().layer_norm(leaf, w.cuda()), leaf, dy.cuda())
    xd, gd = x.double(), dy.double() * w.double()
    rstd = 1 / torch.sqrt(xd.var(-1, unbiased=False, keepdim=True) + 1e-5)
    xh = (xd - xd.mean(-1, keepdim=True)) * rstd
    want = rstd * (gd - gd.mean(-1, keepdim=True) - xh * (gd * xh).mean(-1, keepdim=True))
    assert want[1].isinf().any() or want[3].isinf().any()
    _same_kind('dx', dx, want, 1024)


@pytest.mark.parametrize('B,T,D,N,G,dtype,lengths', [
    (2, 100, 64, 16, 4, 'f32', [100, 41]), (2, 20, 30, 5, 10, 'bf16', None), (1, 200, 12, 12, 12, 'f32', [199]),
    (3, 64, 24, 33, 8, 'f32', None), (2, 50, 40, 8, 8, 'f16', [50, 3]), (300, 9, 62, 16, 2, 'f32', None)])
def test_selective_scan_narrow_groups(B, T, D, N, G, dtype, lengths):
    """Groups of a few channels, whose states lie close together in the workspaces; whole and in segments."""
    lens = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    leaves, dy, dlast = _scan_case(B, T, D, N, G, dtype, seed=46)
    _scan_check(leaves, dy, dlast, lens)


@pytest.mark.parametrize('T,N,lengths', [(13, 16, None), (21, 5, [17]), (300, 16, None), (40, 33, [33])])
def test_selective_scan_infinite_last_state(T, N, lengths):
    """The last token's x is infinite: no token follows, so a's gradient has no infinite state in it."""
    g = _gen(47)
    B, D = 1, 24
    rn = lambda *s: torch.rand(*s, generator=g) + 0.125                          # noqa: E731
    v = dict(x=rn(B, T, D), dt=rn(B, T, D), a=-rn(D, N), b=rn(B, T, 1, N), c=rn(B, T, 1, N), skip=rn(D))
    end = T if lengths is None else lengths[0]
    v['x'][0, end - 1, 3] = float('inf')
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    dy, dlast = rn(B, T, D), rn(B, D, N)
    dev = {k: t.cuda().requires_grad_(True) for k, t in v.items()}
    ref = {k: t.double().requires_grad_(True) for k, t in v.items()}
    y, last = S().selective_scan(*(dev[k] for k in SCAN[:6]), lengths=None if lens is None else lens.cuda(), return_state=True)
    yr, lastr = R.scan(*(ref[k] for k in SCAN[:6]), None, None, True, None, lens)
    for ends in (1, 2):
        got = _grads([y, last][:ends], [dy.cuda(), dlast.cuda()], dev)
        want = torch.autograd.grad([yr, lastr][:ends], list(ref.values()), [dy.double(), dlast.double()][:ends], retain_graph=True)
        want = dict(zip(ref, want))
        assert want['a'].isfinite().all()
        for k in ('a', 'x', 'dt'):
            _same_kind('d' + k, got[k], want[k], 2 * (128 + 8 * T) + (B * T if k == 'a' else 0))
        y, last = S().selective_scan(*(dev[k] for k in SCAN[:6]), lengths=None if lens is None else lens.cuda(), return_state=True)
