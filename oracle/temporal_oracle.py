"""The sequence operators of gast_hip/temporal.py from their definitions, in 64 bits on the host (test infrastructure only).

Every formula is a sum of products with positive coefficients, apart from the two of layer norm that subtract a mean: the same function of
the absolute values bounds the sum of the absolute terms, which is what a rounding error is relative to."""
import torch


def rotary(x, positions, freqs, interleaved, scale=1.0, back=False):
    """x (B, T, J, H, D) float64, positions (B, T)"""
    R = 2 * freqs.numel()
    angle = positions.double()[..., None] * freqs.double() * (-1.0 if back else 1.0)
    cos, sin = (f(angle)[:, :, None, None] * scale for f in (torch.cos, torch.sin))
    y = x.double().clone()
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * cos - b * sin, a * sin + b * cos
    return y


def decay(q, k, v, log_decay, state=None, lengths=None, scale=1.0):
    """token by token: (o, state); q, k (B, T, J, H, Dk), v (B, T, J, H, Dv), all float64; differentiable"""
    B, T, J, H, Dk = q.shape
    lam = torch.exp(log_decay.double()).view(1, 1, H, 1, 1)
    S = torch.zeros(B, J, H, Dk, v.shape[4], dtype=torch.float64) if state is None else state
    n = torch.full((B,), T) if lengths is None else lengths.clamp(0, T)
    out = []
    for t in range(T):
        on = (t < n).view(B, 1, 1, 1, 1)
        # (a product with a zero mask would keep NaN: what is not there is replaced)
        qt, kt, vt = (torch.where(on, x[:, t].unsqueeze(-1), torch.zeros((), dtype=torch.float64)).squeeze(-1) for x in (q, k, v))
        new = lam * S + kt.unsqueeze(-1) * vt.unsqueeze(-2)
        S = torch.where(on, new, S)
        out.append((qt.unsqueeze(-1) * new).sum(-2) * scale)
    o = torch.stack(out, 1) if T else torch.zeros(B, 0, J, H, v.shape[4], dtype=torch.float64)
    return o, S


def decay_grads(q, k, v, log_decay, state, lengths, scale, do, dstate):
    """outputs and gradients: dict of o, state, dq, dk, dv, dstate0"""
    q, k, v = (x.double().detach().requires_grad_(True) for x in (q, k, v))
    s0 = None if state is None else state.double().detach().requires_grad_(True)
    with torch.enable_grad():
        o, new = decay(q, k, v, log_decay, s0, lengths, scale)
        loss = 0.0
        if do is not None:
            n = torch.full((q.shape[0],), q.shape[1]) if lengths is None else lengths.clamp(0, q.shape[1])
            on = (torch.arange(q.shape[1]) < n[:, None])[..., None, None, None]
            loss = loss + (o * torch.where(on, do.double(), torch.zeros((), dtype=torch.float64))).sum()
        if dstate is not None:
            loss = loss + (new * dstate.double()).sum()
        leaves = [q, k, v] + ([] if s0 is None else [s0])
        g = torch.autograd.grad(loss, leaves, allow_unused=True)
    g = [torch.zeros_like(x) if d is None else d for x, d in zip(leaves, g)]
    out = dict(o=o.detach(), state=new.detach(), dq=g[0], dk=g[1], dv=g[2])
    if s0 is not None:
        out['dstate0'] = g[3]
    return out


def drop_keep(seed, thresh, n, salt=0):
    """multipliers 0 / 1 of the library's dropout stream for elements 0 .. n - 1 of tensor `salt`"""
    m = 0xffffffff
    key = (int(seed) * 0x9E3779B9 + salt * 0x85EBCA6B) & m
    e = torch.arange(n, dtype=torch.int64)
    x = ((e >> 1) ^ key) & m
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & m
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & m
    x = x ^ (x >> 16)
    return torch.where(e % 2 == 1, x >> 16, x & 0xffff) >= thresh


def layer_norm(s, weight, bias, eps):
    """float64 in, (y, xhat, rstd)"""
    mean = s.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    xhat = (s - mean) * rstd
    y = xhat if weight is None else xhat * weight.double()
    return y if bias is None else y + bias.double(), xhat, rstd


def layer_norm_grads(xhat, rstd, weight, dy):
    """(ds of the norm, dweight, dbias)"""
    g = dy if weight is None else dy * weight.double()
    ds = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    lead = tuple(range(dy.dim() - 1))
    return ds, (dy * xhat).sum(lead), dy.sum(lead)
