"""CPU: the sequence operators' entry points refuse what their kernels do not take before anything is launched, and size
their workspaces consistently."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    from vqa_amd import sequence as S
    from vqa_amd._lib import VqaHipError
    x = torch.zeros(2, 3, 8)
    for f in (lambda: S.layer_norm(x), lambda: S.causal_conv(x, torch.zeros(8, 4)),
              lambda: S.causal_conv_step(x[:, 0], x, torch.zeros(8, 4)),
              lambda: S.selective_scan(x, x, torch.zeros(8, 4), x[..., :4], x[..., :4]),
              lambda: S.selective_scan_step(x[:, 0], torch.zeros(2, 8, 4), x[:, 0], torch.zeros(8, 4), x[:, 0, :4], x[:, 0, :4])):
        with pytest.raises(VqaHipError, match='GPU'):
            f()


P = ctypes.c_void_p(64)          # never dereferenced: every call below is refused by the host code


def test_entry_points_refuse_bad_arguments():
    from vqa_amd import _lib as L
    lib = L.lib()
    norm = lambda dtype=0, x=P, rows=4, width=8, y=P: lib.vqa_layer_norm_fwd(      # noqa: E731
        None, dtype, x, width, None, None, rows, width, 1e-5, y, None)
    assert all(rc == 1 for rc in (norm(dtype=3), norm(x=None), norm(rows=0), norm(width=0), norm(width=8193),
                                  norm(y=None), norm(rows=1 << 31)))
    assert lib.vqa_layer_norm_bwd(None, 0, P, 8, P, 8, None, P, 4, 8, P, None, None, None) == 1
    assert lib.vqa_layer_norm_bwd(None, 0, P, 8, P, 8, None, None, 4, 8, P, None, None, P) == 1
    assert lib.vqa_layer_norm_bwd_part(0, 8) == 0 and lib.vqa_layer_norm_bwd_part(4, 9000) == 0
    conv = lambda dtype=0, B=1, T=4, D=8, taps=4, w=P: lib.vqa_causal_conv_fwd(                    # noqa: E731
        None, dtype, P, T * D, D, w, None, None, None, B, T, D, taps, 1, P, None)
    assert all(rc == 1 for rc in (conv(dtype=-1), conv(B=0), conv(T=0), conv(D=0), conv(taps=1), conv(taps=5),
                                  conv(w=None), conv(B=1 << 20, T=1 << 20)))
    assert lib.vqa_causal_conv_bwd_part(0, 4, 8) == 0
    assert lib.vqa_causal_conv_token(None, 0, P, 8, None, 24, 8, P, None, 1, 8, 4, 1, P) == 1
    sizes = (ctypes.c_long * 3)()
    at = ctypes.addressof(sizes)
    for args in ((0, 0, 4, 8, 16, 1), (0, 1, 0, 8, 16, 1), (0, 1, 4, 8, 65, 1), (0, 1, 4, 8, 0, 1), (0, 1, 4, 9, 16, 2),
                 (5, 1, 4, 8, 16, 1), (0, 1, 1 << 30, 8, 16, 1), (0, 1, 4, 8, 16, 0)):
        assert lib.vqa_scan_ws_bytes(*args, at) == 1, args
    assert lib.vqa_scan_ws_bytes(0, 1, 4, 8, 16, 1, None) == 1

    def scan(B=1, T=1024, D=8, N=16, G=1, ws=P, keep=None, y=P):
        return lib.vqa_scan_fwd(None, 0, P, T * D, D, P, T * D, D, None, 0, 0, P, P, T * N, N, P, T * N, N, None, None, 1,
                                None, None, B, T, D, N, G, y, None, keep, ws)
    assert all(rc == 1 for rc in (scan(ws=None), scan(ws=ctypes.c_void_p(68)), scan(keep=ctypes.c_void_p(72)), scan(N=65),
                                  scan(G=3), scan(y=None), scan(B=0)))


def test_entry_points_refuse_grids_past_32_bits():
    """Shapes whose launch would have 2^32 threads or more, within every other limit: refused, nothing is launched."""
    from vqa_amd import _lib as L
    lib = L.lib()
    conv = lambda B, T, D: lib.vqa_causal_conv_fwd(None, 0, P, T * D, D, P, None, None, None, B, T, D, 4, 1, P, None)   # noqa: E731
    assert conv(1000000000, 1, 20) == 1 and conv(1, 1, 25000001) == 1
    assert lib.vqa_causal_conv_token(None, 0, P, 7, P, 21, 7, P, None, 700000000, 7, 4, 1, P) == 1
    token = lambda B, D, N: lib.vqa_scan_token(None, 0, P, D, P, D * N, P, D, None, 0, P, P, N, P, N, None, None, 1,    # noqa: E731
                                               B, D, N, 1, P)
    assert token(13000000, 17, 64) == 1
    sizes = (ctypes.c_long * 3)()
    assert lib.vqa_scan_ws_bytes(0, 1, 1, 5000000, 64, 1, ctypes.addressof(sizes)) == 1
    assert lib.vqa_scan_ws_bytes(0, 1, 1, 5000000, 16, 1, ctypes.addressof(sizes)) == 0


def test_scan_workspaces_hold_what_the_kernels_write():
    """The forward's segments, the kept states and the backward's partial sums, from the sizes alone."""
    from vqa_amd import _lib as L
    lib = L.lib()
    for B, T, D, N, G in ((1, 1, 1, 1, 1), (256, 14, 2048, 16, 1), (1, 16383, 2048, 16, 1), (3, 577, 600, 16, 2),
                          (4, 2048, 2048, 16, 1), (2, 100, 64, 64, 4), (7, 700, 33, 20, 1)):
        sizes = (ctypes.c_long * 3)()
        assert lib.vqa_scan_ws_bytes(1, B, T, D, N, G, ctypes.addressof(sizes)) == 0
        fwd, keep, bwd = sizes
        padded, states = G * -(-(D // G) // (128 if N <= 16 else 64)) * (128 if N <= 16 else 64), 8 if N <= 8 else 16 if N <= 16 else 32 if N <= 32 else 64
        assert keep == 4 * B * (-(-T // 8) - 1) * padded * states      # (before every tile but the first)
        assert bwd >= fwd + 4 * B * T * G * 2 * N + 4 * padded * (states + 2)
        assert all(s % 16 == 0 for s in (fwd, keep)) and fwd >= 0
        if fwd:
            segments = fwd // (4 * B * padded * (states + 1))
            assert fwd == 4 * B * padded * (states + 1) * segments and 1 < segments <= max(1, T // 16)


def test_selective_scan_gradients_without_channels():
    """No channel, so nothing is launched; b and c still have values, and their gradients are 0 (memory is handed out here
    that held other values before)."""
    from vqa_amd.sequence import _SelectiveScan
    for _ in range(4):
        b, c = (torch.randn(2, 3, 2, 4, requires_grad=True) for _ in range(2))
        x, a = torch.zeros(2, 3, 0), torch.zeros(0, 4, requires_grad=True)
        y, _ = _SelectiveScan.apply(x, x, a, b, c, None, None, None, 1, None, None, False)
        junk = [torch.full((2, 3, 2, 4), float('nan')) for _ in range(4)]
        del junk
        db, dc, da = torch.autograd.grad(y, [b, c, a], torch.zeros_like(y))
        assert not db.any() and not dc.any() and da.shape == (0, 4)


def _calls(x, w, wc, state, a, b, h, b1):
    """Every entry point, on x [2, 3, 8]."""
    from vqa_amd import sequence as S
    return [lambda x=x, w=w: S.layer_norm(x, w), lambda x=x, wc=wc: S.causal_conv(x, wc),
            lambda x=x, wc=wc: S.causal_conv_step(x[:, 0], state, wc),
            lambda x=x, a=a: S.selective_scan(x, x, a, b, b), lambda x=x, a=a: S.selective_scan_step(x[:, 0], h, x[:, 0], a, b1, b1)]


def _operands():
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*s, generator=g) for s in ((2, 3, 8), (8,), (8, 4), (2, 3, 8), (8, 4), (2, 3, 4), (2, 8, 4), (2, 4))]


@pytest.mark.parametrize('which', range(8))
def test_inputs_with_a_tangent_are_refused(which):
    """A tangent that a call would drop: in each argument, also where nothing requires a gradient."""
    import torch.autograd.forward_ad as fw
    from vqa_amd._lib import VqaHipError
    args = _operands()
    takers = {0: range(5), 1: (0,), 2: (1, 2), 3: (2,), 4: (3, 4), 5: (3,), 6: (4,), 7: (4,)}[which]
    with fw.dual_level():
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        for i in takers:
            with pytest.raises(VqaHipError, match='tangent'):
                _calls(*args)[i]()
        with fw._set_fwd_grad_enabled(False):              # (nothing is followed: refused for another reason)
            for f in _calls(*args):
                with pytest.raises(VqaHipError, match='GPU'):
                    f()
    with fw.dual_level():                                  # (a level alone is no tangent)
        for f in _calls(*_operands()):
            with pytest.raises(VqaHipError, match='GPU'):
                f()


def test_gradients_with_a_tangent_are_refused():
    """... and in the gradient that comes into a backward, as in a forward derivative of a backward pass."""
    import torch.autograd.forward_ad as fw
    from vqa_amd import sequence as S
    from vqa_amd._lib import VqaHipError
    x = torch.zeros(0, 8, requires_grad=True)              # (no row: nothing is launched)
    y = S._LayerNorm.apply(x, None, None, 1e-5)
    assert torch.autograd.grad(y, x, torch.zeros(0, 8), retain_graph=True)[0].shape == (0, 8)
    with fw.dual_level():
        with pytest.raises(VqaHipError, match='tangent'):
            torch.autograd.grad(y, x, fw.make_dual(torch.zeros(0, 8), torch.zeros(0, 8)))


@pytest.mark.parametrize('how', ['jit', 'make_fx', 'pre_dispatch', 'fake', 'export'])
def test_recording_is_refused(how):
    """A recorded program would hold an allocation that nothing fills; with and without a gradient."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from vqa_amd._lib import VqaHipError
    args = _operands()

    def one(i, grad):
        def f(x):
            with torch.set_grad_enabled(grad):
                return _calls(x, *args[1:])[i]()

        class Call(torch.nn.Module):
            def forward(self, x):
                return f(x)
        x = args[0].clone().requires_grad_(grad)
        with pytest.raises(VqaHipError, match='recorded'):
            {'jit': lambda: torch.jit.trace(f, (x,)), 'make_fx': lambda: make_fx(f)(x),
             'pre_dispatch': lambda: make_fx(f, pre_dispatch=True)(x),
             'fake': lambda: make_fx(f, tracing_mode='fake')(x),
             'export': lambda: torch.export.export(Call(), (x,), strict=False)}[how]()
    for i in range(5):
        one(i, False)
        one(i, True)


def test_compiled_callers_reach_the_checks():
    """torch.compile leaves its graph at these calls: on the CPU it ends at the same refusal as without it."""
    from vqa_amd._lib import VqaHipError
    args = _operands()
    for i in range(5):
        def f(x, i=i):
            return _calls(x, *args[1:])[i]()
        torch._dynamo.reset()
        with pytest.raises(VqaHipError, match='GPU'):
            torch.compile(f, backend='eager')(args[0])


class _Wrapper(torch.Tensor):
    """A tensor of another class without memory of its own, as distributed and quantized tensors are."""
    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device, strides=inner.stride())

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        raise NotImplementedError(str(f))


def test_tensors_without_storage_are_refused():
    """The address of such a tensor is 0, which the entry points take for an argument that was left out."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from vqa_amd import sequence as S
    from vqa_amd._lib import VqaHipError
    x, w, wc, state, a, b, h, b1 = _operands()
    t = x[:, 0]

    class Kept(torch.Tensor):                              # a class with ordinary memory is taken
        pass
    for make in (_Wrapper, FakeTensorMode().from_tensor):
        for f in (lambda: S.layer_norm(make(x)), lambda: S.layer_norm(x, make(w)), lambda: S.layer_norm(x, None, make(w)),
                  lambda: S.causal_conv(x, wc, make(w)), lambda: S.causal_conv(x, wc, state=make(state)),
                  lambda: S.causal_conv(x, wc, lengths=make(torch.ones(2, dtype=torch.int32))),
                  lambda: S.causal_conv_step(t, state, wc, make(w)),
                  lambda: S.selective_scan(x, x, a, b, b, make(w)), lambda: S.selective_scan(x, x, a, b, b, gate=make(x)),
                  lambda: S.selective_scan(x, x, a, b, b, state=make(h)),
                  lambda: S.selective_scan_step(t, h, t, a, b1, b1, gate=make(t)),
                  lambda: S.selective_scan_step(t, h, t, a, b1, b1, dt_bias=make(w))):
            with pytest.raises(VqaHipError, match='no storage'):
                f()
    with pytest.raises(VqaHipError, match='list was given'):
        S.causal_conv(x, wc, lengths=[1, 2])
    with pytest.raises(VqaHipError, match='GPU'):
        S.layer_norm(x.as_subclass(Kept), torch.nn.Parameter(w))


def test_eps_is_a_number():
    """A tensor would go to the library as its address; other numbers are converted."""
    import numpy as np
    from vqa_amd import sequence as S
    from vqa_amd._lib import VqaHipError
    x = torch.zeros(2, 8)
    for eps in (torch.tensor(1e-5), torch.tensor(1e-5, requires_grad=True), None, 'small', [1e-5]):
        with pytest.raises(VqaHipError, match='eps'):
            S.layer_norm(x, eps=eps)
    for eps in (1e-5, 0, 1, np.float32(1e-5), np.float64(1e-5)):
        with pytest.raises(VqaHipError, match='GPU'):
            S.layer_norm(x, eps=eps)


def test_axes_past_31_bits_are_refused():
    """A size of 2^32 + 1 would reach the library as 1: the first row would be answered, the others left as allocated."""
    from vqa_amd import sequence as S
    from vqa_amd._lib import VqaHipError

    class Said(torch.Tensor):                              # a CPU tensor that says it is on the GPU
        is_cuda = True

    def rows(*shape):
        return torch.zeros(1, dtype=torch.bfloat16).expand(shape).as_subclass(Said)
    far = (1 << 32) + 1
    for shape in ((far, 1, 1), (1, far, 1), (1, 1, far), (1 << 31, 2, 1)):
        with pytest.raises(VqaHipError, match='below 2'):
            S._first(rows(*shape), 3, '[B, L, D]')
    for shape in ((1 << 20, 1 << 12, 1), (far, 0, 1), ((1 << 31) - 1, 2, 1)):
        S._first(rows(*shape), 3, '[B, L, D]')


def test_scan_refuses_grids_past_32_bits():
    """64 threads for every 64, 32 or 16 channels of a group (up to 16, 32, 64 states), within every other limit."""
    from vqa_amd import _lib as L
    lib = L.lib()
    sizes = (ctypes.c_long * 3)()
    ok = lambda B, D, N, G=1: lib.vqa_scan_ws_bytes(1, B, 1, D, N, G, ctypes.addressof(sizes)) == 0      # noqa: E731
    for B, D, N, G in ((7751937, 129, 64, 1), (6896551, 145, 64, 1), (3448275, 290, 64, 2), (6211180, 161, 33, 1)):
        assert B * G * -(-(D // G) // 16) * 64 >= 1 << 32 and not ok(B, D, N, G)
        rc = lib.vqa_scan_fwd(None, 1, P, D, D, P, D, D, None, 0, 0, P, P, G * N, G * N, P, G * N, G * N, None, None, 1, None,
                              None, B, 1, D, N, G, P, None, None, P)
        assert rc == 1
    # the same widths with fewer rows, and more channels a wave, stay
    assert ok(7000000, 129, 64) and ok(7751937, 129, 32) and ok(7751937, 129, 16)


def test_scan_workspaces_of_narrow_groups():
    """Groups that fill less than a quarter of a workgroup's channels are held as they are."""
    from vqa_amd import _lib as L
    sizes = (ctypes.c_long * 3)()
    for B, T, D, N, G, states in ((64, 4096, 64, 16, 4, 16), (4, 2048, 2048, 16, 2048, 16), (2, 100, 30, 5, 10, 8), (3, 65, 24, 33, 8, 64)):
        assert L.lib().vqa_scan_ws_bytes(1, B, T, D, N, G, ctypes.addressof(sizes)) == 0
        fwd, keep, bwd = sizes
        assert keep == 4 * B * (-(-T // 8) - 1) * D * states
        assert fwd % 16 == 0 and keep % 16 == 0 and bwd % 4 == 0
        assert bwd < 2 * (fwd + 4 * B * T * G * 2 * N) + 4 * 2048 * D * (states + 2)


def _scan_plan(B, T, D, N, G, backward):
    """What the scan's launches write, counted again: (padded states, channels a group takes in a workspace, segments, tokens
    of one, channel blocks and batch groups of the backward)."""
    per, states = D // G, 8 if N <= 8 else 16 if N <= 16 else 32 if N <= 32 else 64
    wave, block = {8: 64, 16: 64, 32: 32, 64: 16}[states], 128 if N <= 16 else 64
    waves, blocks = B * G * -(-per // wave), -(-per // block)
    held = per if G > 1 and 4 * per < blocks * block else blocks * block
    cut = max(min(4096 // waves, T // 64), min(1024 // waves, T // 16), 1) if waves < (640 if backward else 400) else 1
    tokens = -(-(-(-T // cut)) // 8) * 8
    segments = -(-T // tokens)
    return states, held, segments, tokens, blocks, max(1, min(B, 1024 // (G * blocks * segments)))


@pytest.mark.parametrize('B,T,D,N,G', [
    (1, 1, 1, 1, 1), (256, 14, 2048, 16, 1), (1, 16383, 2048, 16, 1), (3, 577, 600, 16, 2), (4, 2048, 2048, 16, 1),
    (2, 100, 64, 64, 4), (7, 700, 33, 20, 1), (16, 512, 2048, 16, 1), (500, 64, 64, 16, 1), (639, 33, 30, 8, 1),
    (400, 40, 16, 33, 1), (64, 4096, 64, 16, 4), (4, 333, 30, 5, 10), (2, 100, 31, 64, 31), (640, 200, 64, 12, 1)])
def test_scan_workspace_sizes(B, T, D, N, G):
    """Exactly what the kernels write: the segments' states and sums of dt, h before every tile but the first, and the
    backward's shares of db / dc by channel block and of the parameters' gradients by (batch group, segment)."""
    from vqa_amd import _lib as L
    sizes = (ctypes.c_long * 3)()
    assert L.lib().vqa_scan_ws_bytes(1, B, T, D, N, G, ctypes.addressof(sizes)) == 0
    whole = lambda floats: -(-floats // 4) * 16                                 # noqa: E731
    ends = []
    for backward in (False, True):
        states, held, segments, tokens, blocks, groups = _scan_plan(B, T, D, N, G, backward)
        assert tokens % 8 == 0 and (segments - 1) * tokens < T <= segments * tokens
        ends.append(whole(B * segments * G * held * (states + 1)) if segments > 1 else 0)
    assert sizes[0] == ends[0]
    assert sizes[1] == 4 * B * (-(-T // 8) - 1) * G * held * states
    assert sizes[2] == ends[1] + whole(groups * segments * G * held * (states + 2)) + 4 * blocks * B * T * G * 2 * N
    if (B, T) in ((500, 64), (400, 40)):                   # (between the two thresholds: only the backward is cut)
        assert sizes[0] == 0 and ends[1] > 0
