"""Sequence operators beside the GRU and BatchNorm, HIP-backed: layer norm over the last axis, the short causal convolution
and the selective state space scan over tokens - whole sequences with their gradients, and one token at a time against a
state that the caller keeps.

    h = layer_norm(x, w, b)                                          # [..., C]
    u, conv_state = causal_conv(h, wc, bc, return_state=True)        # [B, L, D]
    y, state = selective_scan(u, dt, a, b, c, skip, gate, dt_bias, return_state=True)
    ... the next token:  u = causal_conv_step(h1, conv_state, wc, bc);  y = selective_scan_step(u, state, dt1, a, b1, c1, ...)

Rows (x, dt, b, c, gate, the convolution's state) are float32, bfloat16 or float16, all of one type; parameters (weight,
bias, a, skip, dt_bias) and the scan's state are float32, as are all sums.  The last axis of a row must be contiguous (it
is copied otherwise), the other axes may have any stride.  `lengths` (int32 [B], on the GPU) marks a padded batch: tokens at
or past lengths[b] give zero rows and zero gradients, take no part in any sum or state, and may hold anything; values are
taken between 0 and L.  `state` continues a sequence and `return_state` returns what its continuation needs; gradients pass
through both.  Everything runs on torch's current stream of the tensors' device; workspaces are torch allocations of the
call, so captured graphs share nothing.  A backward that is to be captured into a graph needs leaves that no live eager
graph uses (torch ties a leaf's gradient accumulation to the stream of its first use); the *_step functions are forward
only, and the state they update shares no memory with their other arguments.  There are no forward-mode derivatives, and
torch.jit.trace, make_fx and torch.export cannot record these calls.  Errors of use raise VqaHipError (a
RuntimeError) before anything is launched.
"""
import ctypes
from functools import lru_cache

import torch
import torch.fx._symbolic_trace as _fx
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib as L

_ROW_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_F32 = torch.float32


_device, _stream_of = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_grad_enabled, _tracing = torch.is_grad_enabled, torch._C._is_tracing


def _elsewhere(x):
    """Whether x's device is not the current one (the kernels go to the current device's stream; autograd makes a
    backward's device the current one by itself)."""
    return _device() != x.get_device()


def _fail(what):
    raise L.VqaHipError(what)


def _followed(*tensors):
    """The kernels run behind torch's back: what follows or records a computation operator by operator (forward-mode
    derivatives, torch.jit.trace, make_fx and torch.export) would see an empty allocation in place of a result.  Refused -
    called only where one of them is at work (a call looks for that and at its arguments' types in 0.3 us).  torch.compile
    leaves its graph for a call of the library."""
    if not torch.compiler.is_dynamo_compiling() and (
            _tracing() or torch._C._dispatch_tls_is_dispatch_key_included(torch._C.DispatchKey.PreDispatch)
            or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None):
        _fail('the sequence operators cannot be recorded by torch.jit.trace, make_fx or torch.export')
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                _fail('an input carries a tangent: the sequence operators have no forward-mode derivative')


_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}


def _stored(*args):
    """Every argument of another class is a tensor with memory of its own: a wrapper's address is 0, which an entry point
    takes for an argument that was left out."""
    for t in args:
        if type(t) not in _PLAIN:
            if not isinstance(t, torch.Tensor):
                _fail(f'a {type(t).__name__} was given where a tensor is wanted')
            if t.layout is not torch.strided or t.numel() and not t.data_ptr():
                _fail(f'a {type(t).__name__} has no storage that a kernel could read')


def _first(x, dims, what, *others):
    """The tensor that sets the type and the device: rows on the GPU, of a row type, with this many axes (None: any).
    others: the call's other tensors, or None."""
    if forward_ad._current_level >= 0 or _fx._is_fx_tracing_flag or _tracing():
        _followed(x, *others)
    if type(x) not in _PLAIN or not _PLAIN.issuperset(map(type, others)):
        _stored(x, *others)
    if not x.is_cuda:
        _fail('x must be on the GPU (there is no CPU fallback)')
    if x.dtype not in _ROW_TYPES:
        _fail(f'x must be float32, bfloat16 or float16, not {x.dtype}')
    if dims is not None and x.dim() != dims:
        _fail(f'x has shape {tuple(x.shape)}: {what} is wanted')
    if x.numel() > 0x7fffffff and max(x.shape) > 0x7fffffff:   # (the entry points take sizes of 32 bits)
        _fail(f'x has shape {tuple(x.shape)}: axes below 2^31 are wanted')


def _rows(name, t, shape, x):
    """A row tensor of x's type and device and (shape not None) of this shape."""
    if t.dtype is not x.dtype or t.get_device() != x.get_device():
        _fail(f'{name} is {t.dtype} on {t.device}: {x.dtype} on {x.device} is wanted')
    if shape is not None and t.shape != shape:
        _fail(f'{name} has shape {tuple(t.shape)}: {tuple(shape)} is wanted')


def _param(name, p, shape, x):
    """A float32 parameter or state of this shape on x's device, contiguous; None stays None."""
    if p is None:
        return None
    if p.dtype is not _F32 or p.get_device() != x.get_device():
        _fail(f'{name} is {p.dtype} on {p.device}: float32 on {x.device} is wanted')
    if p.shape != shape:
        _fail(f'{name} has shape {tuple(p.shape)}: {tuple(shape)} is wanted')
    return p if p.is_contiguous() else p.contiguous()


def _number(name, v):
    """A Python number (a tensor would go to the library as its address)"""
    if isinstance(v, torch.Tensor):
        _fail(f'{name} is a tensor: a number is wanted')
    try:
        return float(v)
    except (TypeError, ValueError):
        _fail(f'{name} is {v!r}: a number is wanted')


def _lengths(lengths, x):
    if lengths is None:
        return None
    if lengths.dtype != torch.int32 or lengths.device != x.device or lengths.shape != x.shape[:1]:
        _fail(f'lengths must be int32 [{x.shape[0]}] on {x.device}')
    return lengths.contiguous()


def _unit(x):
    """x with a contiguous last axis"""
    return x if x.stride(-1) == 1 else x.contiguous()


def _like(x):
    """A contiguous tensor of x's kind for a result"""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _near(x):
    """... and rows whose distance the scan's kernels can take (8 rows within 2 GiB)"""
    if x.dim() == 2 or x.stride(1) < 1 << 26:
        return _unit(x)
    return x.clone(memory_format=torch.contiguous_format)      # (contiguous() keeps the stride of an axis of one row)


def _touched(state):
    """A kernel wrote into `state`: autograd's version of it moves on."""
    if not state.is_inference():
        increment_version(state)


def _tracked(*tensors):
    if _grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tracking(what, *tensors):
    if _grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail(f'{what} has no gradient: call it under torch.no_grad()')


def _backward(f):
    """The backward of these operators, which has no derivative of its own: asked for one (create_graph) its results are
    marked so.  (once_differentiable alone costs every ordinary backward a few microseconds.)"""
    marked = once_differentiable(f)

    def backward(ctx, *grads):
        if forward_ad._current_level >= 0 or _fx._is_fx_tracing_flag or _tracing():
            _followed(*grads)
        return marked(ctx, *grads) if _grad_enabled() else f(ctx, *grads)
    return staticmethod(backward)


# ---------------------------------------------------------------------------------------------------------- layer norm

def _as_matrix(x):
    """[..., C] -> [rows, C] with a contiguous last axis and one row stride; a view where the strides allow it"""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 else x.contiguous()


def _norm_fwd(x, weight, bias, eps, stats):
    x2 = _as_matrix(x)
    rows, width = x2.shape
    y = _like(x)
    st = torch.empty(2, rows, device=x.device, dtype=_F32) if stats else None
    if rows:
        L.call('vqa_layer_norm_fwd', L.dt(x), x2, x2.stride(0), weight, bias, rows, width, eps, y, st)
    return y, st


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, st = _norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, st)
        ctx.has_bias = bias is not None
        return y

    @_backward
    def backward(ctx, dy):
        x, weight, st = ctx.saved_tensors
        x2, dy2 = _as_matrix(x), _as_matrix(dy)
        rows, width = x2.shape
        dev = x.device
        dx = torch.empty(x.shape, device=dev, dtype=x.dtype)
        dw = torch.empty(width, device=dev, dtype=_F32) if weight is not None else None
        db = torch.empty(width, device=dev, dtype=_F32) if ctx.has_bias else None
        if rows:
            part = torch.empty(_norm_parts(rows, width), 2, width, device=dev, dtype=_F32)
            L.call('vqa_layer_norm_bwd', L.dt(x), dy2, dy2.stride(0), x2, x2.stride(0), weight, st, rows, width,
                   dx, dw, db, part)
        else:
            for g in (dw, db):
                if g is not None:
                    g.zero_()
        return dx, dw, db, None


@lru_cache(maxsize=1024)
def _norm_parts(rows, width):
    return L.lib().vqa_layer_norm_bwd_part(rows, width)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (biased variance), statistics in float32.
    x [..., C] with C <= 8192; weight, bias float32 [C] or None."""
    if type(eps) is not float:
        eps = _number('eps', eps)
    _first(x, None, '', weight, bias)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return layer_norm(x, weight, bias, eps)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        _fail(f'x has shape {tuple(x.shape)}: a last axis of 1 to 8192 is wanted')
    width = (x.shape[-1],)
    weight, bias = _param('weight', weight, width, x), _param('bias', bias, width, x)
    if _tracked(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_fwd(x, weight, bias, eps, False)[0]


# --------------------------------------------------------------------------------------------------- causal convolution

def _silu_flag(activation):
    if activation == 'silu':
        return 1
    if activation is not None:
        _fail(f"activation is {activation!r}: 'silu' or None is wanted")
    return 0


def _taps(weight, D):
    if weight.dim() != 2 or weight.shape[0] != D or not 2 <= weight.shape[1] <= 4:
        _fail(f'weight has shape {tuple(weight.shape)}: [{D}, 2 to 4] is wanted')
    return weight.shape[1]


def _conv_fwd(x, weight, bias, silu, state, lengths, want_last):
    B, T, D = x.shape
    taps = weight.shape[1]
    y = _like(x)
    last = torch.empty(B, taps - 1, D, device=x.device, dtype=x.dtype) if want_last else None
    if y.numel():
        L.call('vqa_causal_conv_fwd', L.dt(x), x, x.stride(0), x.stride(1), weight, bias, state, lengths, B, T, D, taps,
               silu, y, last)
    elif want_last and last.numel():
        last.zero_() if state is None else last.copy_(state)
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, state, lengths, want_last):
        y, last = _conv_fwd(x, weight, bias, silu, state, lengths, want_last)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, last

    @_backward
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        B, T, D = x.shape
        taps, dev = weight.shape[1], x.device
        dy = torch.zeros(B, T, D, device=dev, dtype=x.dtype) if dy is None else _unit(dy)
        dlast = None if dlast is None else dlast.contiguous()
        dx = torch.empty(B, T, D, device=dev, dtype=x.dtype)
        dw = torch.empty(D, taps, device=dev, dtype=_F32)
        db = torch.empty(D, device=dev, dtype=_F32) if bias is not None else None
        dstate = torch.empty(B, taps - 1, D, device=dev, dtype=x.dtype) if state is not None else None
        if dx.numel():
            part = torch.empty(_conv_parts(B, T, D), taps + 1, D, device=dev, dtype=_F32)
            L.call('vqa_causal_conv_bwd', L.dt(x), dy, dy.stride(0), dy.stride(1), dlast, x, x.stride(0),
                   x.stride(1), weight, bias, state, lengths, B, T, D, taps, ctx.silu, dx, dw, db, dstate, part)
        else:
            dw.zero_()
            if db is not None:
                db.zero_()
            if dstate is not None:
                dstate.zero_() if dlast is None else dstate.copy_(dlast)
        return dx, dw, db, None, dstate, None, None


@lru_cache(maxsize=1024)
def _conv_parts(B, T, D):
    return L.lib().vqa_causal_conv_bwd_part(B, T, D)


def causal_conv(x, weight, bias=None, activation='silu', state=None, lengths=None, return_state=False):
    """One filter of 2 to 4 taps per channel over the tokens of x [B, L, D], each token seeing itself and those before it:
    y_t = act(bias + sum_k weight[:, k] x_{t - taps + 1 + k}), act = silu or (activation=None) nothing; weight float32
    [D, taps], bias float32 [D].  state [B, taps - 1, D] (x's type): the rows before the first (None: zeros).  Returns y,
    or with return_state (y, state after each sequence's last token)."""
    _first(x, 3, '[B, L, D]', weight, bias, state, lengths)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return causal_conv(x, weight, bias, activation, state, lengths, return_state)
    B, T, D = x.shape
    taps = _taps(weight, D)
    weight, bias = _param('weight', weight, (D, taps), x), _param('bias', bias, (D,), x)
    silu = _silu_flag(activation)
    if state is not None:
        _rows('state', state, (B, taps - 1, D), x)
        state = state.contiguous()
    lengths = _lengths(lengths, x)
    x = _unit(x)
    if _tracked(x, weight, bias, state):
        y, last = _CausalConv.apply(x, weight, bias, silu, state, lengths, return_state)
    else:
        y, last = _conv_fwd(x, weight, bias, silu, state, lengths, return_state)
    return (y, last) if return_state else y


def causal_conv_step(x, state, weight, bias=None, activation='silu'):
    """causal_conv for ONE new token per sequence: x [B, D]; state [B, taps - 1, D] (x's type; rows may be strided) is
    shifted in place.  Returns y [B, D].  Forward only."""
    _first(x, 2, '[B, D]', state, weight, bias)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return causal_conv_step(x, state, weight, bias, activation)
    B, D = x.shape
    taps = _taps(weight, D)
    weight, bias = _param('weight', weight, (D, taps), x), _param('bias', bias, (D,), x)
    silu = _silu_flag(activation)
    _rows('state', state, (B, taps - 1, D), x)
    _no_tracking('causal_conv_step', x, state, weight, bias)
    y = torch.empty(B, D, device=x.device, dtype=x.dtype)
    if not y.numel():
        return y
    s0, s1, s2 = state.stride()
    if (s2 != 1 and D > 1) or not (s1 >= D or taps == 2) or not (
            B == 1 or s0 >= (taps - 2) * s1 + D or (s0 >= D and s1 >= (B - 1) * s0 + D)):
        _fail(f'state has strides {state.stride()}: it is updated in place, so rows must be contiguous and apart')
    x = _unit(x)
    if L._PROFILE is None and L._REC is None:
        rc = L.lib().vqa_causal_conv_token(
            _stream_of(x.get_device()), L.dt(x), x.data_ptr(), x.stride(0), state.data_ptr(), s0, s1, weight.data_ptr(),
            None if bias is None else bias.data_ptr(), B, D, taps, silu, y.data_ptr())
        if rc:
            L.check(rc, 'vqa_causal_conv_token')
    else:
        L.call('vqa_causal_conv_token', L.dt(x), x, x.stride(0), state, s0, s1, weight, bias, B, D, taps, silu, y)
    _touched(state)
    return y


# ------------------------------------------------------------------------------------------------- selective state space

@lru_cache(maxsize=1024)
def _scan_bytes(dtype, B, T, D, N, G):
    sizes = (ctypes.c_long * 3)()
    if L.lib().vqa_scan_ws_bytes(dtype, B, T, D, N, G, ctypes.addressof(sizes)) != 0:
        _fail(f'selective_scan: batch {B}, length {T}, width {D}, {N} states in {G} groups is out of range')
    return tuple(sizes)


def _floats(nbytes, dev):
    return torch.empty(nbytes // 4, device=dev, dtype=_F32) if nbytes else None


def _strides(x):
    """batch and row stride of a row tensor, zeros for None"""
    return (0, 0) if x is None else (x.stride(0), x.stride(1))


def _scan_fwd(x, dt, a, b, c, skip, gate, dt_bias, softplus, state, lengths, want_last, want_keep):
    B, T, D = x.shape
    G, N, dev, code = b.shape[2], b.shape[3], x.device, L.dt(x)
    y = _like(x)
    last = torch.empty(B, D, N, device=dev, dtype=_F32) if want_last else None
    if not y.numel():
        if want_last and last.numel():
            last.zero_() if state is None else last.copy_(state)
        return y, last, None
    fwd, keep_bytes, _ = _scan_bytes(code, B, T, D, N, G)
    ws = _floats(fwd, dev)
    keep = _floats(keep_bytes, dev) if want_keep else None
    L.call('vqa_scan_fwd', code, x, x.stride(0), x.stride(1), dt, dt.stride(0), dt.stride(1), gate,
           *_strides(gate), a, b, b.stride(0), b.stride(1), c, c.stride(0), c.stride(1), skip, dt_bias, softplus,
           state, lengths, B, T, D, N, G, y, last, keep, ws)
    return y, last, keep


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, a, b, c, skip, gate, dt_bias, softplus, state, lengths, want_last):
        y, last, keep = _scan_fwd(x, dt, a, b, c, skip, gate, dt_bias, softplus, state, lengths, want_last, True)
        ctx.save_for_backward(x, dt, a, b, c, skip, gate, dt_bias, state, lengths, keep)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, last

    @_backward
    def backward(ctx, dy, dlast):
        x, dt, a, b, c, skip, gate, dt_bias, state, lengths, keep = ctx.saved_tensors
        B, T, D = x.shape
        G, N, dev, code = b.shape[2], b.shape[3], x.device, L.dt(x)
        f32 = lambda *s: torch.empty(*s, device=dev, dtype=_F32)       # noqa: E731
        rows = lambda *s: torch.empty(*s, device=dev, dtype=x.dtype)            # noqa: E731
        dlast = None if dlast is None else dlast.contiguous()
        dx, ddt, dgate = rows(B, T, D), rows(B, T, D), rows(B, T, D) if gate is not None else None
        db, dc, da = rows(B, T, G, N), rows(B, T, G, N), f32(D, N)
        dskip, dbias = f32(D) if skip is not None else None, f32(D) if dt_bias is not None else None
        dstate = f32(B, D, N) if state is not None else None
        if not dx.numel():
            for g in (da, db, dc, dskip, dbias):           # (without channels, db and dc still have values)
                if g is not None:
                    g.zero_()
            if dstate is not None:
                dstate.zero_() if dlast is None else dstate.copy_(dlast)
        else:
            dy = torch.zeros(B, T, D, device=dev, dtype=x.dtype) if dy is None else _near(dy)
            ws = _floats(_scan_bytes(code, B, T, D, N, G)[2], dev)
            L.call('vqa_scan_bwd', code, dy, dy.stride(0), dy.stride(1), dlast, x, x.stride(0), x.stride(1), dt,
                   dt.stride(0), dt.stride(1), gate, *_strides(gate), a, b, b.stride(0), b.stride(1), c,
                   c.stride(0), c.stride(1), skip, dt_bias, ctx.softplus, state, lengths, B, T, D, N, G, keep, dx, ddt,
                   dgate, da, db, dc, dskip, dbias, dstate, ws)
        return dx, ddt, da, db, dc, dskip, dgate, dbias, None, dstate, None, None


def _shared(name, b, lead, x):
    """b or c as [*lead, G, N] with contiguous groups"""
    _rows(name, b, None, x)
    k = len(lead)
    if b.dim() not in (k + 1, k + 2) or b.shape[:k] != lead:
        _fail(f'{name} has shape {tuple(b.shape)}: [{", ".join(map(str, lead))}, N] or [.., G, N] is wanted')
    if b.dim() == k + 1:
        b = b.unsqueeze(k)
    G, N = b.shape[k:]
    if k == 2 and b.stride(1) >= 1 << 26:
        return b.clone(memory_format=torch.contiguous_format)  # (as in _near)
    return b if b.stride(-1) == 1 and (G == 1 or b.stride(-2) == N) else b.contiguous()


def _scan_args(x, dt, a, b, c, skip, gate, dt_bias):
    lead, D = x.shape[:-1], x.shape[-1]
    _rows('dt', dt, x.shape, x)
    if gate is not None:
        _rows('gate', gate, x.shape, x)
        gate = _near(gate)
    b, c = _shared('b', b, lead, x), _shared('c', c, lead, x)
    G, N = b.shape[-2:]
    if c.shape != b.shape:
        _fail(f'b and c have shapes {tuple(b.shape)} and {tuple(c.shape)}: the same is wanted')
    if not 1 <= N <= 64 or G < 1 or D % G:
        _fail(f'{N} states in {G} groups over {D} channels: 1 to 64 states and a whole number of channels a group')
    return (_near(x), _near(dt), _param('a', a, (D, N), x), b, c, _param('skip', skip, (D,), x), gate,
            _param('dt_bias', dt_bias, (D,), x))


def selective_scan(x, dt, a, b, c, skip=None, gate=None, dt_bias=None, softplus=True, state=None, lengths=None,
                   return_state=False):
    """The selective state space recurrence over x [B, L, D], token by token, per channel and its N <= 64 states:
        dt_t = softplus(dt_t + dt_bias)                   (softplus=False: dt_t + dt_bias)
        h_t = exp(dt_t a) h_{t-1} + (dt_t x_t) b_t,       y_t = (sum_n c_t h_t + skip x_t) * silu(gate_t)
    dt, gate [B, L, D]; b, c [B, L, N], or [B, L, G, N] where each of G groups of D / G channels has its own; a float32
    [D, N]; skip, dt_bias float32 [D]; state float32 [B, D, N] (None: zeros).  gate, skip, dt_bias may be None.
    Returns y, or with return_state (y, state after each sequence's last token)."""
    _first(x, 3, '[B, L, D]', dt, a, b, c, skip, gate, dt_bias, state, lengths)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return selective_scan(x, dt, a, b, c, skip, gate, dt_bias, softplus, state, lengths, return_state)
    args = x, dt, a, b, c, skip, gate, dt_bias = _scan_args(x, dt, a, b, c, skip, gate, dt_bias)
    state = _param('state', state, (x.shape[0], *a.shape), x)
    lengths = _lengths(lengths, x)
    if _tracked(*args, state):
        y, last = _SelectiveScan.apply(*args, int(softplus), state, lengths, return_state)
    else:
        y, last, _ = _scan_fwd(*args, int(softplus), state, lengths, return_state, False)
    return (y, last) if return_state else y


def _ready(x, dt, a, b, c, skip, gate, dt_bias):
    """(G, N) where every argument of a step is already as its kernel takes it - the usual case, found by a third of
    _scan_args' host time.  None: _scan_args says what is wrong, or makes copies."""
    t, g, rows, shared = x.dtype, x.get_device(), x.shape, b.shape
    k = len(shared)
    N = shared[-1] if k else 0
    G = shared[1] if k == 3 else 1
    D = rows[1]
    if (k == 2 or k == 3) and shared[0] == rows[0] and 1 <= N <= 64 and G > 0 and D % G == 0 \
            and dt.dtype is t and dt.get_device() == g and dt.shape == rows and dt.stride(1) == 1 and x.stride(1) == 1 \
            and b.dtype is t and b.get_device() == g and b.stride(-1) == 1 and (G == 1 or b.stride(1) == N) \
            and c.dtype is t and c.get_device() == g and c.shape == shared and c.stride(-1) == 1 \
            and (G == 1 or c.stride(1) == N) and a.dtype is _F32 and a.get_device() == g and a.shape == (D, N) \
            and a.is_contiguous() \
            and (gate is None or (gate.dtype is t and gate.get_device() == g and gate.shape == rows
                                  and gate.stride(1) == 1)):
        for p in (skip, dt_bias):
            if p is not None and not (p.dtype is _F32 and p.get_device() == g and p.shape == (D,) and p.is_contiguous()):
                return None
        return G, N
    return None


def selective_scan_step(x, state, dt, a, b, c, skip=None, gate=None, dt_bias=None, softplus=True):
    """selective_scan for ONE new token per sequence: x, dt, gate [B, D]; b, c [B, N] or [B, G, N]; state float32
    [B, D, N] is updated in place (its batch axis may be strided).  Returns y [B, D].  Forward only."""
    _first(x, 2, '[B, D]', state, dt, a, b, c, skip, gate, dt_bias)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return selective_scan_step(x, state, dt, a, b, c, skip, gate, dt_bias, softplus)
    B, D = x.shape
    ready = _ready(x, dt, a, b, c, skip, gate, dt_bias)
    if ready is None:
        x, dt, a, b, c, skip, gate, dt_bias = _scan_args(x, dt, a, b, c, skip, gate, dt_bias)
        ready = b.shape[1:]
    G, N = ready
    if state.dtype is not _F32 or state.get_device() != x.get_device() or state.shape != (B, D, N):
        _fail(f'state is {state.dtype} {tuple(state.shape)} on {state.device}: float32 {(B, D, N)} on {x.device} is wanted')
    _no_tracking('selective_scan_step', x, state, dt, a, b, c, skip, gate, dt_bias)
    y = torch.empty(B, D, device=x.device, dtype=x.dtype)
    if not y.numel():
        return y
    s0, s1, s2 = state.stride()
    if (s2 != 1 and N > 1) or (s1 != N and D > 1) or (B > 1 and s0 < D * N):
        _fail(f'state has strides {state.stride()}: it is updated in place, so [D, N] must be contiguous and apart')
    sg, softplus = 0 if gate is None else gate.stride(0), int(softplus)
    if L._PROFILE is None and L._REC is None:
        # (one token's latency is host time: pointers are taken here, 3 us less than by L.call)
        rc = L.lib().vqa_scan_token(
            _stream_of(x.get_device()), L.dt(x), x.data_ptr(), x.stride(0), state.data_ptr(), s0, dt.data_ptr(),
            dt.stride(0), None if gate is None else gate.data_ptr(), sg, a.data_ptr(), b.data_ptr(), b.stride(0),
            c.data_ptr(), c.stride(0), None if skip is None else skip.data_ptr(),
            None if dt_bias is None else dt_bias.data_ptr(), softplus, B, D, N, G, y.data_ptr())
        if rc:
            L.check(rc, 'vqa_scan_token')
    else:
        L.call('vqa_scan_token', L.dt(x), x, x.stride(0), state, s0, dt, dt.stride(0), gate, sg, a, b,
               b.stride(0), c, c.stride(0), skip, dt_bias, softplus, B, D, N, G, y)
    _touched(state)
    return y
