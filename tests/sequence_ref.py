"""The sequence operators token by token in 64 bits on the CPU, and the tolerance that kernel outputs are held to."""
import torch


def norm(x, w, b, eps=1e-5):
    m = x.mean(-1, keepdim=True)
    v = ((x - m) ** 2).mean(-1, keepdim=True)
    y = (x - m) / torch.sqrt(v + eps)
    if w is not None:
        y = y * w
    return y if b is None else y + b


def silu(v):
    return v * torch.sigmoid(v)


def conv(x, w, b, act, state, lengths):
    B, T, D = x.shape
    K = w.shape[1]
    ys, lasts = [], []
    for i in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[i])))
        before = state[i] if state is not None else x.new_zeros(K - 1, D)
        full = torch.cat([before, x[i, :n]])
        rows = []
        for t in range(T):
            if t >= n:
                rows.append(x.new_zeros(D))
                continue
            p = (full[t:t + K] * w.t()).sum(0)
            p = p if b is None else p + b
            rows.append(silu(p) if act == 'silu' else p)
        ys.append(torch.stack(rows))
        lasts.append(full[n:n + K - 1])
    return torch.stack(ys), torch.stack(lasts)


def scan(x, dt, a, b, c, skip, gate, dt_bias, softplus, state, lengths):
    """b, c [B, L, G, N]"""
    B, T, D = x.shape
    per = D // b.shape[2]
    ys, hs = [], []
    for i in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[i])))
        h = state[i] if state is not None else x.new_zeros(D, a.shape[1])
        rows = []
        for t in range(T):
            if t >= n:
                rows.append(x.new_zeros(D))
                continue
            s = dt[i, t] if dt_bias is None else dt[i, t] + dt_bias
            s = torch.nn.functional.softplus(s, threshold=1e9) if softplus else s
            bt, ct = b[i, t].repeat_interleave(per, 0), c[i, t].repeat_interleave(per, 0)
            h = torch.exp(s[:, None] * a) * h + (s * x[i, t])[:, None] * bt
            y = (ct * h).sum(1)
            y = y if skip is None else y + skip * x[i, t]
            rows.append(y if gate is None else y * silu(gate[i, t]))
        ys.append(torch.stack(rows))
        hs.append(h)
    return torch.stack(ys), torch.stack(hs)


def close(name, got, want, roundings, scale=None):
    """|got - want| <= half a step of got's type at want + `roundings` half steps of float32 at the largest |want|: the
    kernels compute in float32 - `roundings` bounds the chain of them - and round once to their type.  scale: the largest
    term, in place of the largest |want|, where the terms cancel."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    f = torch.finfo(got.dtype)
    g, w = got.detach().double().cpu(), want.detach().double()
    assert torch.isfinite(w).all(), name
    assert torch.isfinite(g).all(), name
    tol = f.eps / 2 * w.abs() + f.tiny * f.eps + roundings * 2.0 ** -24 * (
        scale if scale is not None else w.abs().max() if w.numel() else 0.0)
    worst = ((g - w).abs() / tol.clamp(min=1e-300)).max() if w.numel() else 0.0
    assert worst <= 1.0, f'{name}: {float(worst):.3g} times its tolerance'
